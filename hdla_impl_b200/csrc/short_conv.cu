// Depthwise causal convolution over W taps with its activation:
//     p_t = bias + sum_{k<W} w[W-1-k] x_{t-k},   y_t = act(p_t)
// forward, backward and the step of single tokens.  A handful of operations an element: bound by HBM (x in, y out; backward x
// and dy in, dx out).  A thread owns PW neighbouring channels (one 16-byte access of x forward, 8 bytes of bf16 backward, where
// the taps' sums need the registers) and walks over a strip of tokens with the last W - 1 inputs in registers, so that a row
// is read once, plus W - 1 rows at each strip's edge, which the neighbouring strip has just brought to L2.
#include "ssm.cuh"

namespace hdla {
namespace {

struct ConvP {
    HdlaConvArgs a;
    int strip;                // tokens a thread walks over
    int strips, col_blocks;   // blocks of strips per sequence row, blocks of channels
    bool wide_w;              // the taps of a thread's channels can be read as 16-byte words
    float* part;              // backward: [B * strips][W + 1][D]
};

template <int DT>
__device__ __forceinline__ constexpr int pack_width() { return DT == HDLA_F32 ? 4 : 8; }

// w[k][c]: the weight of lag k for channel c of the thread's PW
template <int PW, int WT, bool Vec>
__device__ __forceinline__ void load_taps(const ConvP& p, int ch, int valid, float (&w)[WT][PW], float (&bias)[PW]) {
    const int W = WT == 8 ? p.a.W : WT;
    bool done = false;
    if constexpr (Vec && WT != 8) {
        if (p.wide_w && valid > 0) {
            if (p.a.w_dtype == HDLA_BF16) {
                if constexpr (PW * WT % 8 == 0) {
                    Pack<HDLA_BF16, PW * WT> r = ld_pack<HDLA_BF16, PW * WT, true>(p.a.weight, (long long)ch * WT, 1);
                    float f[PW * WT];
                    unpack<HDLA_BF16, PW * WT>(r, f);
#pragma unroll
                    for (int c = 0; c < PW; ++c)
#pragma unroll
                        for (int k = 0; k < WT; ++k) w[k][c] = f[c * WT + WT - 1 - k];
                    done = true;
                }
            } else if constexpr (PW * WT % 4 == 0) {
                Pack<HDLA_F32, PW * WT> r = ld_pack<HDLA_F32, PW * WT, true>(p.a.weight, (long long)ch * WT, 1);
#pragma unroll
                for (int c = 0; c < PW; ++c)
#pragma unroll
                    for (int k = 0; k < WT; ++k) w[k][c] = __uint_as_float(r.w[c * WT + WT - 1 - k]);
                done = true;
            }
        }
    }
#pragma unroll
    for (int c = 0; c < PW; ++c) {
        if (!done)
#pragma unroll
            for (int k = 0; k < WT; ++k)
                w[k][c] = c < valid && k < W ? ld_elem(p.a.weight, (size_t)(ch + c) * W + (W - 1 - k), p.a.w_dtype) : 0.f;
        bias[c] = p.a.bias && c < valid ? ld_elem(p.a.bias, ch + c, p.a.w_dtype) : 0.f;
    }
}

// Taps beyond W (only with WT == 8) are left out, not multiplied by zero: what they would read may be infinite.
template <int PW, int WT>
__device__ __forceinline__ void taps(const float (&w)[WT][PW], const float (&bias)[PW], const float* x, const float (&hist)[WT - 1][PW],
                                     int W, float* out) {
#pragma unroll
    for (int c = 0; c < PW; ++c) {
        float s = fmaf(w[0][c], x[c], bias[c]);
#pragma unroll
        for (int k = 1; k < WT; ++k)
            if (WT != 8 || k < W) s = fmaf(w[k][c], hist[k - 1][c], s);
        out[c] = s;
    }
}
template <int PW, int N>
__device__ __forceinline__ void shift(float (&hist)[N][PW], const float* x) {
#pragma unroll
    for (int k = N - 1; k > 0; --k)
#pragma unroll
        for (int c = 0; c < PW; ++c) hist[k][c] = hist[k - 1][c];
#pragma unroll
    for (int c = 0; c < PW; ++c) hist[0][c] = x[c];
}

// The inputs of the W - 1 tokens before token t of a sequence that starts at `start`: its initial state's rows before that.
template <int DT, int PW, int WT, bool Vec>
__device__ __forceinline__ void load_hist(const ConvP& p, long long xrow, long long state, int start, int t, int ch, int valid,
                                          float (&hist)[WT - 1][PW]) {
    const int W = WT == 8 ? p.a.W : WT;
#pragma unroll
    for (int k = 0; k < WT - 1; ++k) {
        const int tt = t - 1 - k;
        Pack<DT, PW> r = {};
        if (k < W - 1) {
            if (tt >= start) r = ld_pack<DT, PW, Vec>(p.a.x, xrow + tt * p.a.x_token + ch, valid);
            else if (p.a.h0) r = ld_pack<DT, PW, Vec>(p.a.h0, (state * (W - 1) + (W - 1 + tt - start)) * p.a.D + ch, valid);
        }
        unpack<DT, PW>(r, hist[k]);
    }
}
template <int DT, int PW, int WT, bool Vec>
__device__ __forceinline__ void store_state(const ConvP& p, void* to, long long state, int ch, int valid, const float (&hist)[WT - 1][PW]) {
    const int W = WT == 8 ? p.a.W : WT;
#pragma unroll
    for (int k = 0; k < WT - 1; ++k)
        if (k < W - 1) st_pack<DT, PW, Vec>(to, (state * (W - 1) + (W - 2 - k)) * p.a.D + ch, valid, hist[k]);
}

constexpr int kFwdWarps = 4, kBwdWarps = 8;

template <int DT, int WT, bool Vec>
__global__ void __launch_bounds__(32 * kFwdWarps) conv_fwd_kernel(const __grid_constant__ ConvP p) {
    constexpr int PW = pack_width<DT>(), U = 8;
    const int T = p.a.T, D = p.a.D, W = WT == 8 ? p.a.W : WT;
    const int cb = blockIdx.x % p.col_blocks, sb = blockIdx.x / p.col_blocks % p.strips, b = blockIdx.x / p.col_blocks / p.strips;
    const int ch = (cb * 32 + (threadIdx.x & 31)) * PW, valid = min(PW, D - ch);
    const long long first = ((long long)sb * kFwdWarps + (threadIdx.x >> 5)) * p.strip;
    if (valid <= 0 || first >= T) return;
    const int t0 = static_cast<int>(first), t1 = min(T, t0 + p.strip);
    const Seqs q{p.a.cu_seqlens, p.a.cu_seqlens ? p.a.n_seqs : 1, T};
    const long long xrow = b * p.a.x_batch, yrow = (long long)b * T;
    float w[WT][PW], bias[PW], hist[WT - 1][PW];
    load_taps<PW, WT, Vec>(p, ch, valid, w, bias);
    int s = q.ends_behind(t0);
    if (t0 == 0 && p.a.ht)
        for (int i = 0; i < s; ++i) {                          // empty sequences at the front
            load_hist<DT, PW, WT, Vec>(p, xrow, b + i, 0, 0, ch, valid, hist);
            store_state<DT, PW, WT, Vec>(p, p.a.ht, b + i, ch, valid, hist);
        }
    int end = s < q.n ? q.off(s + 1) : 0x7fffffff;
    if (s < q.n) load_hist<DT, PW, WT, Vec>(p, xrow, b + s, min(q.off(s), t0), t0, ch, valid, hist);
    for (int t = t0; t < t1; t += U) {
        Pack<DT, PW> in[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t + u < t1) in[u] = ld_pack<DT, PW, Vec>(p.a.x, xrow + (t + u) * p.a.x_token + ch, valid);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t + u >= t1) break;
            float x[PW], out[PW];
            unpack<DT, PW>(in[u], x);
            taps<PW, WT>(w, bias, x, hist, W, out);
#pragma unroll
            for (int c = 0; c < PW; ++c) {
                if (p.a.activation == HDLA_ACT_SILU) out[c] *= sigmoid_of(out[c]);
                if (s >= q.n) out[c] = 0.f;
            }
            st_pack<DT, PW, Vec>(p.a.y, (yrow + t + u) * D + ch, valid, out);
            shift<PW, WT - 1>(hist, x);
            while (end <= t + u + 1) {                         // this token was a sequence's last (and empty ones follow)
                if (p.a.ht) store_state<DT, PW, WT, Vec>(p, p.a.ht, b + s, ch, valid, hist);
                if (++s < q.n) {
                    load_hist<DT, PW, WT, Vec>(p, xrow, b + s, t + u + 1, t + u + 1, ch, valid, hist);
                    end = q.off(s + 1);
                } else {
                    end = 0x7fffffff;
                }
            }
        }
    }
}

// One token: the state is the history, and moves on by one row in place (a thread owns its channels' rows).
template <int DT, int WT, bool Vec>
__global__ void __launch_bounds__(128) conv_step_kernel(const __grid_constant__ ConvP p) {
    constexpr int PW = pack_width<DT>();
    const int D = p.a.D, W = WT == 8 ? p.a.W : WT;
    const int cb = blockIdx.x % p.col_blocks;
    const long long b = (long long)(blockIdx.x / p.col_blocks) * 4 + (threadIdx.x >> 5);
    const int ch = (cb * 32 + (threadIdx.x & 31)) * PW, valid = min(PW, D - ch);
    if (valid <= 0 || b >= p.a.B) return;
    float w[WT][PW], bias[PW], hist[WT - 1][PW], x[PW], out[PW];
    const Pack<DT, PW> in = ld_pack<DT, PW, Vec>(p.a.x, b * p.a.x_batch + ch, valid);
    load_hist<DT, PW, WT, Vec>(p, 0, b, 0, 0, ch, valid, hist);
    load_taps<PW, WT, Vec>(p, ch, valid, w, bias);
    unpack<DT, PW>(in, x);
    taps<PW, WT>(w, bias, x, hist, W, out);
    if (p.a.activation == HDLA_ACT_SILU)
#pragma unroll
        for (int c = 0; c < PW; ++c) out[c] *= sigmoid_of(out[c]);
    st_pack<DT, PW, Vec>(p.a.y, b * D + ch, valid, out);
    shift<PW, WT - 1>(hist, x);
    store_state<DT, PW, WT, Vec>(p, p.a.ht, b, ch, valid, hist);
}

// Backward: p_t is computed again; dp_t = dy_t act'(p_t);  dx_t = sum_k w_k dp_{t+k};  dw_k = sum_t dp_t x_{t-k}.
// Walking forward, the row that a token completes is the one W - 1 before it, so the gradient of the initial state comes out
// as the rows before a sequence's start, and the final state's gradient joins the last W - 1 rows, which W - 1 more steps
// with dp = 0 complete.  A strip also walks over the W - 1 tokens behind it, for its own last rows.
template <int DT, int WT, bool Vec>
__global__ void __launch_bounds__(32 * kBwdWarps) conv_bwd_kernel(const __grid_constant__ ConvP p) {
    constexpr int PW = 4, U = 4;
    __shared__ float red[kBwdWarps][WT + 1][32 * PW];
    const int T = p.a.T, D = p.a.D, W = WT == 8 ? p.a.W : WT;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cb = blockIdx.x % p.col_blocks, sb = blockIdx.x / p.col_blocks % p.strips, b = blockIdx.x / p.col_blocks / p.strips;
    const int ch = (cb * 32 + lane) * PW, valid = min(PW, D - ch);
    const long long first = ((long long)sb * kBwdWarps + warp) * p.strip;
    const Seqs q{p.a.cu_seqlens, p.a.cu_seqlens ? p.a.n_seqs : 1, T};
    const long long xrow = b * p.a.x_batch, yrow = (long long)b * T;
    float w[WT][PW], bias[PW], dw[WT][PW] = {}, db[PW] = {}, xh[WT - 1][PW], dph[WT - 1][PW];
    const float none[PW] = {};
    if (valid > 0 && first < T) {
        load_taps<PW, WT, Vec>(p, ch, valid, w, bias);
        const int t0 = static_cast<int>(first), t1 = min(T, t0 + p.strip);
        int s = q.ends_behind(t0), start = 0, end = 0, from = 0;
        // token t's dp (0 behind the sequence's end) completes row t - (W - 1)
        auto emit = [&](int t, const float* dp) {
            const int row = t - (W - 1);
            float v[PW];
#pragma unroll
            for (int c = 0; c < PW; ++c) {
                v[c] = 0.f;
#pragma unroll
                for (int k = 0; k < WT; ++k) {
                    if (WT != 8) v[c] = fmaf(w[k][c], k == W - 1 ? dp[c] : dph[WT - 2 - k < 0 ? 0 : WT - 2 - k][c], v[c]);
                    else if (k < W) {
                        float d = dp[c];
#pragma unroll
                        for (int i = 0; i < WT - 1; ++i)
                            if (i == W - 2 - k) d = dph[i][c];
                        v[c] = fmaf(w[k][c], d, v[c]);
                    }
                }
            }
            if (t >= end && p.a.dht) {
                float d[PW];
                unpack<DT, PW>(ld_pack<DT, PW, Vec>(p.a.dht, ((long long)(b + s) * (W - 1) + (t - end)) * D + ch, valid), d);
#pragma unroll
                for (int c = 0; c < PW; ++c) v[c] += d[c];
            }
            if (row >= from) {
                if (row < t1) st_pack<DT, PW, Vec>(p.a.dx, (yrow + row) * D + ch, valid, v);
            } else if (from == start && p.a.dh0) {
                st_pack<DT, PW, Vec>(p.a.dh0, ((long long)(b + s) * (W - 1) + (row - start + W - 1)) * D + ch, valid, v);
            }
            shift<PW, WT - 1>(dph, dp);
        };
        auto clear = [&] {
#pragma unroll
            for (int k = 0; k < WT - 1; ++k)
#pragma unroll
                for (int c = 0; c < PW; ++c) dph[k][c] = 0.f;
        };
        auto empty = [&](int i, int at) {                      // an empty sequence at token `at`: dh0 = dht
            if (!p.a.dh0) return;
            const int keep = s;
            s = i; start = end = from = at;
            clear();
            for (int f = 0; f < W - 1; ++f) {                  // its rows lie before `at`: nothing of dx is written
                emit(at + f, none);
            }
            s = keep;
        };
        if (t0 == 0)
            for (int i = 0; i < s; ++i) empty(i, 0);
        int t = t0;
        while (t < t1) {
            if (s >= q.n) {
                for (; t < t1; ++t) st_pack<DT, PW, Vec>(p.a.dx, (yrow + t) * D + ch, valid, none);
                break;
            }
            start = min(q.off(s), t); end = max(q.off(s + 1), t); from = t;      // (offsets that decrease stay harmless)
            const int stop = min(end, t1 + W - 1);
            load_hist<DT, PW, WT, Vec>(p, xrow, b + s, start, t, ch, valid, xh);
            clear();
            for (int tt = t; tt < stop; tt += U) {
                Pack<DT, PW> xin[U], yin[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (tt + u < stop) {
                        xin[u] = ld_pack<DT, PW, Vec>(p.a.x, xrow + (tt + u) * p.a.x_token + ch, valid);
                        if (p.a.dy) yin[u] = ld_pack<DT, PW, Vec>(p.a.dy, (yrow + tt + u) * D + ch, valid);
                        else yin[u] = {};
                    }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (tt + u >= stop) break;
                    float x[PW], dp[PW], pre[PW];
                    unpack<DT, PW>(xin[u], x);
                    unpack<DT, PW>(yin[u], dp);
                    if (p.a.activation == HDLA_ACT_SILU) {
                        taps<PW, WT>(w, bias, x, xh, W, pre);
#pragma unroll
                        for (int c = 0; c < PW; ++c) dp[c] *= act_grad(pre[c], HDLA_ACT_SILU);
                    }
                    if (tt + u < t1) {
#pragma unroll
                        for (int c = 0; c < PW; ++c) {
                            db[c] += dp[c];
                            dw[0][c] = fmaf(dp[c], x[c], dw[0][c]);
#pragma unroll
                            for (int k = 1; k < WT; ++k)
                                if (WT != 8 || k < W) dw[k][c] = fmaf(dp[c], xh[k - 1][c], dw[k][c]);
                        }
                    }
                    emit(tt + u, dp);
                    shift<PW, WT - 1>(xh, x);
                }
            }
            if (stop == end)
                for (int f = 0; f < W - 1; ++f) emit(end + f, none);
            t = min(end, t1);
            if (end <= t1) {
                ++s;
                while (s < q.n && q.off(s + 1) <= t) { empty(s, t); ++s; }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < WT; ++k)
#pragma unroll
        for (int c = 0; c < PW; ++c) red[warp][k][lane * PW + c] = dw[k][c];
#pragma unroll
    for (int c = 0; c < PW; ++c) red[warp][WT][lane * PW + c] = db[c];
    __syncthreads();
    float* part = p.part + (long long)(b * p.strips + sb) * (W + 1) * D;
    for (int i = threadIdx.x; i < (W + 1) * 32 * PW; i += 32 * kBwdWarps) {
        const int row = i / (32 * PW), c = i % (32 * PW), k = row < W ? W - 1 - row : WT;      // row r of the taps is lag W - 1 - r
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < kBwdWarps; ++j) v += red[j][k][c];
        if (cb * 32 * PW + c < D) part[(long long)row * D + cb * 32 * PW + c] = v;
    }
}

// Strips of 16 (forward) or 32 tokens (backward: also W - 1 tokens behind the strip) unless too few threads would be left to
// keep the memory busy (about 512 an SM), then shorter ones.
int strip_of(const HdlaConvArgs& a, int pw, int longest) {
    int strip = longest;
    while (strip > 4 && (long long)a.B * ((a.T + strip - 1) / strip) * ((a.D + pw - 1) / pw) < 512LL * sm_count()) strip /= 2;
    return strip;
}
ConvP plan(const HdlaConvArgs& a, int pw, int longest, int warps) {
    ConvP p{};
    p.a = a;
    p.strip = strip_of(a, pw, longest);
    p.strips = static_cast<int>(((long long)a.T + (long long)p.strip * warps - 1) / ((long long)p.strip * warps));
    p.col_blocks = (a.D + 32 * pw - 1) / (32 * pw);
    p.wide_w = aligned16(a.weight);
    return p;
}
bool conv_vec(const HdlaConvArgs& a, int pw, int size) {
    const int bytes = pw * size;
    auto ok = [&](const void* q) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; };
    return a.D % pw == 0 && a.x_batch % pw == 0 && a.x_token % pw == 0 && ok(a.x) && ok(a.h0) && ok(a.y) && ok(a.ht) && ok(a.dy) &&
           ok(a.dht) && ok(a.dx) && ok(a.dh0);
}

template <int DT, bool Vec, typename F>
void with_taps(int W, F f) {
    if (W == 2) f(std::integral_constant<int, 2>());
    else if (W == 3) f(std::integral_constant<int, 3>());
    else if (W == 4) f(std::integral_constant<int, 4>());
    else f(std::integral_constant<int, 8>());
}

}  // namespace

int short_conv_fwd(const HdlaConvArgs& a, bool step, cudaStream_t st) {
    const int size = a.dtype == HDLA_F32 ? 4 : 2, pw = 16 / size;
    const bool vec = conv_vec(a, pw, size);
    const ConvP p = plan(a, pw, 16, kFwdWarps);
    const long long grid = step ? (long long)p.col_blocks * ((a.B + 3) / 4) : (long long)p.col_blocks * p.strips * a.B;
    if (grid > 0x7fffffffLL) return fail(HDLA_ERR_UNSUPPORTED, "short_conv: %lld blocks", grid);
    auto go = [&](auto dt, auto v) {
        with_taps<dt, v>(a.W, [&](auto wt) {
            if (step) conv_step_kernel<dt, wt, v><<<(unsigned)grid, 128, 0, st>>>(p);
            else conv_fwd_kernel<dt, wt, v><<<(unsigned)grid, 32 * kFwdWarps, 0, st>>>(p);
        });
    };
    using F32 = std::integral_constant<int, HDLA_F32>;
    using BF16 = std::integral_constant<int, HDLA_BF16>;
    if (a.dtype == HDLA_F32) vec ? go(F32(), std::true_type()) : go(F32(), std::false_type());
    else vec ? go(BF16(), std::true_type()) : go(BF16(), std::false_type());
    HDLA_CHECK_LAUNCH(step ? "conv_step_kernel" : "conv_fwd_kernel");
    return HDLA_OK;
}

size_t short_conv_bwd_workspace(const HdlaConvArgs& a) {
    const ConvP p = plan(a, 4, 32, kBwdWarps);
    return up256((size_t)a.B * p.strips * (a.W + 1) * a.D * sizeof(float));
}

int short_conv_bwd(const HdlaConvArgs& a, float* part, cudaStream_t st) {
    const int size = a.dtype == HDLA_F32 ? 4 : 2, pw = 4;
    const bool vec = conv_vec(a, pw, size);
    ConvP p = plan(a, pw, 32, kBwdWarps);
    p.part = part;
    const long long grid = (long long)p.col_blocks * p.strips * a.B;
    if (grid > 0x7fffffffLL) return fail(HDLA_ERR_UNSUPPORTED, "short_conv: %lld blocks", grid);
    auto go = [&](auto dt, auto v) {
        with_taps<dt, v>(a.W, [&](auto wt) { conv_bwd_kernel<dt, wt, v><<<(unsigned)grid, 32 * kBwdWarps, 0, st>>>(p); });
    };
    using F32 = std::integral_constant<int, HDLA_F32>;
    using BF16 = std::integral_constant<int, HDLA_BF16>;
    if (a.dtype == HDLA_F32) vec ? go(F32(), std::true_type()) : go(F32(), std::false_type());
    else vec ? go(BF16(), std::true_type()) : go(BF16(), std::false_type());
    HDLA_CHECK_LAUNCH("conv_bwd_kernel");
    ColJobs js{};
    js.n = 1;
    js.j[0] = ColJob{part, {a.dweight, a.dbias, nullptr}, (long long)(a.W + 1) * a.D, a.B * p.strips, a.W + 1, a.D, a.D, a.w_dtype, 1, 0, 0};
    return column_sum_launch(js, st);
}

}  // namespace hdla
