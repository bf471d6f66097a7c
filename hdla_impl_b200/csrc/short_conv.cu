// Depthwise causal convolution over W taps with its activation:
//     p_t = bias + sum_{k<W} w[W-1-k] x_{t-k},   y_t = act(p_t)
// forward, backward and the step of single tokens.  A handful of operations an element: bound by HBM (x in, y out; backward x
// and dy in, dx out).  A thread owns four neighbouring channels, as two packed pairs, and walks over a strip of tokens with the
// last W - 1 inputs in registers, so that a row is read once, plus W - 1 rows at each strip's edge, which the neighbouring strip
// has just brought to L2.  Several tokens are requested at a time, and forward the next ones before these are worked on.  Four
// channels a thread and not eight (16 bytes of bf16): the taps, their sums and the histories are what fills the registers, and
// with half of them twice the warps hide the latency (forward 100 -> 61 us, backward 262 -> 148 us at 32768 x 2048, W = 4).
// There forward now takes 55 us = 4.9 TB/s (0.76 of the measured copy), backward 106 us = 3.8 TB/s (0.59) and its sums 10 us;
// 16384 x 2048 in fp32: 49 us = 5.5 TB/s (0.85) and 101 us = 4.0 TB/s (0.62).
#include "ssm.cuh"

namespace hdla {
namespace {

constexpr int PW = 4;
constexpr int kFwdWarps = 4, kBwdWarps = 8;
struct Quad { f2 v[2]; };                                        // four channels
template <int WT> constexpr int kHist = WT > 1 ? WT - 1 : 1;     // rows of history (one, of no use, with a single tap)

struct ConvP {
    HdlaConvArgs a;
    int strip;                // tokens a thread walks over
    int strips, col_blocks;   // blocks of strips per sequence row, blocks of channels
    bool wide_w;              // the taps of a thread's channels can be read as 16-byte words
    float* part;              // backward: [B * strips][W + 1][D]
};

template <int DT>
__device__ __forceinline__ Quad quad_of(const Pack<DT, PW>& r) {
    float f[PW];
    unpack<DT, PW>(r, f);
    return Quad{{f2_pack(f[0], f[1]), f2_pack(f[2], f[3])}};
}
template <int DT, bool Vec>
__device__ __forceinline__ void st_quad(void* base, long long i, int valid, const Quad& q) {
    float f[PW];
    f2_unpack(q.v[0], f[0], f[1]);
    f2_unpack(q.v[1], f[2], f[3]);
    st_pack<DT, PW, Vec>(base, i, valid, f);
}
// w[k]: the weights of lag k for the thread's channels
template <int WT, bool Vec>
__device__ __forceinline__ void load_taps(const ConvP& p, int ch, int valid, Quad (&w)[WT], Quad& bias) {
    float f[PW][WT], b[PW];
    bool done = false;
    if constexpr (Vec && PW * WT % 8 == 0) {
        if (p.wide_w) {
            if (p.a.w_dtype == HDLA_BF16)
                unpack<HDLA_BF16, PW * WT>(ld_pack<HDLA_BF16, PW * WT, true>(p.a.weight, (long long)ch * WT, 1), &f[0][0]);
            else
                unpack<HDLA_F32, PW * WT>(ld_pack<HDLA_F32, PW * WT, true>(p.a.weight, (long long)ch * WT, 1), &f[0][0]);
            done = true;
        }
    }
#pragma unroll
    for (int c = 0; c < PW; ++c) {
        if (!done)
#pragma unroll
            for (int j = 0; j < WT; ++j) f[c][j] = c < valid ? ld_elem(p.a.weight, (size_t)(ch + c) * WT + j, p.a.w_dtype) : 0.f;
        b[c] = p.a.bias && c < valid ? ld_elem(p.a.bias, ch + c, p.a.w_dtype) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < WT; ++k) {
        const int j = WT - 1 - k;
        w[k] = Quad{{f2_pack(f[0][j], f[1][j]), f2_pack(f[2][j], f[3][j])}};
    }
    bias = Quad{{f2_pack(b[0], b[1]), f2_pack(b[2], b[3])}};
}

template <int WT>
__device__ __forceinline__ Quad taps(const Quad (&w)[WT], const Quad& bias, const Quad& x, const Quad (&hist)[kHist<WT>]) {
    Quad out;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        f2 s = f2_fma(w[0].v[c], x.v[c], bias.v[c]);
#pragma unroll
        for (int k = 1; k < WT; ++k) s = f2_fma(w[k].v[c], hist[k - 1].v[c], s);
        out.v[c] = s;
    }
    return out;
}
template <int N>
__device__ __forceinline__ void shift(Quad (&hist)[N], const Quad& x) {
#pragma unroll
    for (int k = N - 1; k > 0; --k) hist[k] = hist[k - 1];
    hist[0] = x;
}

// The inputs of the W - 1 tokens before token t of a sequence that starts at `start`: its initial state's rows before that.
template <int DT, int WT, bool Vec>
__device__ __forceinline__ void load_hist(const ConvP& p, long long xrow, long long state, int start, int t, int ch, int valid, Quad (&hist)[kHist<WT>]) {
    constexpr int W = WT;
    hist[0] = Quad{{0, 0}};
#pragma unroll
    for (int k = 0; k < WT - 1; ++k) {
        const int tt = t - 1 - k;
        Pack<DT, PW> r = {};
        if (tt >= start) r = ld_pack<DT, PW, Vec>(p.a.x, xrow + tt * p.a.x_token + ch, valid);
        else if (p.a.h0) r = ld_pack<DT, PW, Vec>(p.a.h0, (state * (W - 1) + (W - 1 + tt - start)) * p.a.D + ch, valid);
        hist[k] = quad_of<DT>(r);
    }
}
template <int DT, int WT, bool Vec>
__device__ __forceinline__ void store_state(const ConvP& p, long long state, int ch, int valid, const Quad (&hist)[kHist<WT>]) {
    constexpr int W = WT;
#pragma unroll
    for (int k = 0; k < WT - 1; ++k) st_quad<DT, Vec>(p.a.ht, (state * (W - 1) + (W - 2 - k)) * p.a.D + ch, valid, hist[k]);
}

template <int DT, int WT, bool Vec>
__global__ void __launch_bounds__(32 * kFwdWarps) conv_fwd_kernel(const __grid_constant__ ConvP p) {
    constexpr int U = 8;                                       // tokens requested ahead (four: 60 us instead of 55 at 32768 x 2048)
    const int T = p.a.T, D = p.a.D;
    const int cb = blockIdx.x % p.col_blocks, sb = blockIdx.x / p.col_blocks % p.strips, b = blockIdx.x / p.col_blocks / p.strips;
    const int ch = (cb * 32 + (threadIdx.x & 31)) * PW, valid = min(PW, D - ch);
    const long long first = ((long long)sb * kFwdWarps + (threadIdx.x >> 5)) * p.strip;
    if (valid <= 0 || first >= T) return;
    const int t0 = static_cast<int>(first), t1 = min(T, t0 + p.strip);
    const Seqs q{p.a.cu_seqlens, p.a.cu_seqlens ? p.a.n_seqs : 1, T};
    const long long xrow = b * p.a.x_batch;
    constexpr int size = DT == HDLA_F32 ? 4 : 2;
    const char* from = static_cast<const char*>(p.a.x) + (xrow + t0 * p.a.x_token + ch) * size;
    char* to = static_cast<char*>(p.a.y) + (((long long)b * T + t0) * D + ch) * size;
    const long long from_step = p.a.x_token * size, to_step = (long long)D * size;
    Pack<DT, PW> in[U], next[U];
    auto request = [&](int tokens) {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = ld_pack<DT, PW, Vec, true>(from + u * from_step, 0, u < tokens ? valid : 0);
        from += U * from_step;
    };
    request(t1 - t0);
    Quad w[WT], bias, hist[kHist<WT>];
    load_taps<WT, Vec>(p, ch, valid, w, bias);
    int s = q.ends_behind(t0);
    if (t0 == 0 && p.a.ht)
        for (int i = 0; i < s; ++i) {                          // empty sequences at the front
            load_hist<DT, WT, Vec>(p, xrow, b + i, 0, 0, ch, valid, hist);
            store_state<DT, WT, Vec>(p, b + i, ch, valid, hist);
        }
    int end = s < q.n ? q.off(s + 1) : 0x7fffffff;
    load_hist<DT, WT, Vec>(p, xrow, b + min(s, q.n - 1), s < q.n ? min(q.off(s), t0) : t0, t0, ch, valid, hist);
    for (int t = t0; t < t1; t += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) in[u] = next[u];
        if (t + U < t1) request(t1 - t - U);
        auto one = [&](int u) {
            const Quad x = quad_of<DT>(in[u]);
            Quad out = taps<WT>(w, bias, x, hist);
            if (p.a.activation == HDLA_ACT_SILU)
#pragma unroll
                for (int c = 0; c < 2; ++c) out.v[c] = f2_mul(out.v[c], sigmoid_pair(out.v[c]));
            shift(hist, x);
            return out;
        };
        if (t + U <= t1 && end > t + U && s < q.n) {
#pragma unroll
            for (int u = 0; u < U; ++u) st_quad<DT, Vec>(to + u * to_step, 0, valid, one(u));
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t + u >= t1) break;
                Quad out = one(u);
                if (s >= q.n) out = Quad{{0, 0}};              // a token of no sequence
                st_quad<DT, Vec>(to + u * to_step, 0, valid, out);
                while (end <= t + u + 1) {                     // this token was a sequence's last (and empty ones follow)
                    if (p.a.ht) store_state<DT, WT, Vec>(p, b + s, ch, valid, hist);
                    if (++s < q.n) {
                        load_hist<DT, WT, Vec>(p, xrow, b + s, t + u + 1, t + u + 1, ch, valid, hist);
                        end = q.off(s + 1);
                    } else {
                        end = 0x7fffffff;
                    }
                }
            }
        }
        to += U * to_step;
    }
}

// One token: the state is the history, and moves on by one row in place (a thread owns its channels' rows).
template <int DT, int WT, bool Vec>
__global__ void __launch_bounds__(128) conv_step_kernel(const __grid_constant__ ConvP p) {
    const int D = p.a.D;
    const int cb = blockIdx.x % p.col_blocks;
    const long long b = (long long)(blockIdx.x / p.col_blocks) * 4 + (threadIdx.x >> 5);
    const int ch = (cb * 32 + (threadIdx.x & 31)) * PW, valid = min(PW, D - ch);
    if (valid <= 0 || b >= p.a.B) return;
    Quad w[WT], bias, hist[kHist<WT>];
    const Pack<DT, PW> in = ld_pack<DT, PW, Vec>(p.a.x, b * p.a.x_batch + ch, valid);
    load_hist<DT, WT, Vec>(p, 0, b, 0, 0, ch, valid, hist);
    load_taps<WT, Vec>(p, ch, valid, w, bias);
    const Quad x = quad_of<DT>(in);
    Quad out = taps<WT>(w, bias, x, hist);
    if (p.a.activation == HDLA_ACT_SILU)
#pragma unroll
        for (int c = 0; c < 2; ++c) out.v[c] = f2_mul(out.v[c], sigmoid_pair(out.v[c]));
    st_quad<DT, Vec>(p.a.y, b * D + ch, valid, out);
    shift(hist, x);
    store_state<DT, WT, Vec>(p, b, ch, valid, hist);
}

// Backward: p_t is computed again; dp_t = dy_t act'(p_t);  dx_t = sum_k w_k dp_{t+k};  dw_k = sum_t dp_t x_{t-k}.
// Walking forward, the row that a token completes is the one W - 1 before it, so the gradient of the initial state comes out
// as the rows before a sequence's start, and the final state's gradient joins the last W - 1 rows, which W - 1 more steps
// with dp = 0 complete.  A strip also walks over the W - 1 tokens behind it, for its own last rows.
// Two blocks an SM where the registers of that many taps allow it (16384 x 2048, W = 4, bf16: 64 us, with one block 80 us; fp32
// spills with two, 165 us, with one 100 us).
template <int DT, int WT, bool Vec>
__global__ void __launch_bounds__(32 * kBwdWarps, WT <= (DT == HDLA_F32 ? 2 : 4) ? 2 : 1) conv_bwd_kernel(const __grid_constant__ ConvP p) {
    constexpr int U = 4, W = WT;
    __shared__ __align__(16) float red[kBwdWarps][WT + 1][32 * PW];
    const int T = p.a.T, D = p.a.D;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cb = blockIdx.x % p.col_blocks, sb = blockIdx.x / p.col_blocks % p.strips, b = blockIdx.x / p.col_blocks / p.strips;
    const int ch = (cb * 32 + lane) * PW, valid = min(PW, D - ch);
    const long long first = ((long long)sb * kBwdWarps + warp) * p.strip;
    const Seqs q{p.a.cu_seqlens, p.a.cu_seqlens ? p.a.n_seqs : 1, T};
    const long long xrow = b * p.a.x_batch, yrow = (long long)b * T;
    const bool silu = p.a.activation == HDLA_ACT_SILU;
    constexpr int size = DT == HDLA_F32 ? 4 : 2;
    const long long x_step = p.a.x_token * size, y_step = (long long)D * size;
    Quad dw[WT], db = {{0, 0}};
#pragma unroll
    for (int k = 0; k < WT; ++k) dw[k] = Quad{{0, 0}};
    if (valid > 0 && first < T) {
        Quad w[WT], bias, xh[kHist<WT>], dph[kHist<WT>];
        load_taps<WT, Vec>(p, ch, valid, w, bias);
        const int t0 = static_cast<int>(first), t1 = min(T, t0 + p.strip);
        int s = q.ends_behind(t0), start = 0, end = 0, from = 0;
        // what a token's dp (0 behind the sequence's end) completes: row t - (W - 1)
        auto complete = [&](const Quad& dp) {
            Quad v;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                f2 r = 0;
#pragma unroll
                for (int k = 0; k < WT; ++k) r = f2_fma(w[k].v[c], k == WT - 1 ? dp.v[c] : dph[WT - 2 - k < 0 ? 0 : WT - 2 - k].v[c], r);
                v.v[c] = r;
            }
            shift(dph, dp);
            return v;
        };
        auto emit = [&](int t, const Quad& dp) {
            const int row = t - (W - 1);
            Quad v = complete(dp);
            if (t >= end && p.a.dht) {
                const Quad d = quad_of<DT>(ld_pack<DT, PW, Vec>(p.a.dht, ((long long)(b + s) * (W - 1) + (t - end)) * D + ch, valid));
                v.v[0] = f2_add(v.v[0], d.v[0]);
                v.v[1] = f2_add(v.v[1], d.v[1]);
            }
            if (row >= from) {
                if (row < t1) st_quad<DT, Vec>(p.a.dx, (yrow + row) * D + ch, valid, v);
            } else if (from == start && p.a.dh0) {
                st_quad<DT, Vec>(p.a.dh0, ((long long)(b + s) * (W - 1) + (row - start + W - 1)) * D + ch, valid, v);
            }
        };
        // dp of a token, and its share of the weights' gradients where it is the strip's own
        auto gradient = [&](const Pack<DT, PW>& xin, const Pack<DT, PW>& yin, bool mine) {
            const Quad x = quad_of<DT>(xin);
            Quad dp = quad_of<DT>(yin);
            if (silu) {
                const Quad pre = taps<WT>(w, bias, x, xh);
#pragma unroll
                for (int c = 0; c < 2; ++c) {                  // silu' = s + p s (1 - s)
                    const f2 sg = sigmoid_pair(pre.v[c]), ps = f2_mul(pre.v[c], sg);
                    dp.v[c] = f2_mul(dp.v[c], f2_fma(ps, f2_fma(sg, f2_dup(-1.f), f2_dup(1.f)), sg));
                }
            }
            if (mine)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    db.v[c] = f2_add(db.v[c], dp.v[c]);
                    dw[0].v[c] = f2_fma(dp.v[c], x.v[c], dw[0].v[c]);
#pragma unroll
                    for (int k = 1; k < WT; ++k) dw[k].v[c] = f2_fma(dp.v[c], xh[k - 1].v[c], dw[k].v[c]);
                }
            shift(xh, x);
            return dp;
        };
        auto clear = [&] {
#pragma unroll
            for (int k = 0; k < kHist<WT>; ++k) dph[k] = Quad{{0, 0}};
        };
        const Quad none = {{0, 0}};
        auto empty = [&](int i, int at) {                      // an empty sequence at token `at`: dh0 = dht
            if (!p.a.dh0) return;
            const int keep = s;
            s = i; start = end = from = at;
            clear();
            for (int f = 0; f < W - 1; ++f) emit(at + f, none);      // its rows lie before `at`: nothing of dx is written
            s = keep;
        };
        if (t0 == 0)
            for (int i = 0; i < s; ++i) empty(i, 0);
        int t = t0;
        while (t < t1) {
            if (s >= q.n) {
                for (; t < t1; ++t) st_quad<DT, Vec>(p.a.dx, (yrow + t) * D + ch, valid, none);
                break;
            }
            start = min(q.off(s), t); end = max(q.off(s + 1), t); from = t;      // (offsets that decrease stay harmless)
            const int stop = min(end, t1 + W - 1);
            load_hist<DT, WT, Vec>(p, xrow, b + s, start, t, ch, valid, xh);
            clear();
            const char* fx = static_cast<const char*>(p.a.x) + (xrow + t * p.a.x_token + ch) * size;
            const char* fy = static_cast<const char*>(p.a.dy) + ((yrow + t) * D + ch) * size;
            char* to = static_cast<char*>(p.a.dx) + ((yrow + t - (W - 1)) * D + ch) * size;
            Pack<DT, PW> xn[U], yn[U];
            auto request = [&](int tokens) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int ok = u < tokens ? valid : 0;
                    xn[u] = ld_pack<DT, PW, Vec>(fx + u * x_step, 0, ok);
                    yn[u] = ld_pack<DT, PW, Vec>(fy + u * y_step, 0, p.a.dy ? ok : 0);
                }
                fx += U * x_step;
                fy += U * y_step;
            };
            request(stop - t);
            for (int tt = t; tt < stop; tt += U) {
                Pack<DT, PW> xin[U], yin[U];
#pragma unroll
                for (int u = 0; u < U; ++u) { xin[u] = xn[u]; yin[u] = yn[u]; }
                if (tt + U < stop) request(stop - tt - U);
                if (tt - (W - 1) >= from && tt + U <= min(stop, t1)) {       // rows and tokens of this strip and sequence
#pragma unroll
                    for (int u = 0; u < U; ++u) st_quad<DT, Vec>(to + u * y_step, 0, valid, complete(gradient(xin[u], yin[u], true)));
                } else {
#pragma unroll 1
                    for (int u = 0; u < min(U, stop - tt); ++u) {
                        emit(tt + u, gradient(xin[0], yin[0], tt + u < t1));
#pragma unroll
                        for (int i = 0; i < U - 1; ++i) { xin[i] = xin[i + 1]; yin[i] = yin[i + 1]; }
                    }
                }
                to += U * y_step;
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
    for (int k = 0; k < WT; ++k) *reinterpret_cast<ulonglong2*>(&red[warp][k][lane * PW]) = make_ulonglong2(dw[k].v[0], dw[k].v[1]);
    *reinterpret_cast<ulonglong2*>(&red[warp][WT][lane * PW]) = make_ulonglong2(db.v[0], db.v[1]);
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

// Strips of 128 tokens unless too few threads would be left to keep the memory busy (about 1024 an SM), then shorter ones:
// backward a strip's first and last tokens take a slower way, and it walks over W - 1 tokens behind itself.
ConvP plan(const HdlaConvArgs& a, int warps) {
    ConvP p{};
    p.a = a;
    p.strip = 128;
    while (p.strip > 4 && (long long)a.B * ((a.T + p.strip - 1) / p.strip) * ((a.D + PW - 1) / PW) < 1024LL * sm_count()) p.strip /= 2;
    p.strips = static_cast<int>(((long long)a.T + (long long)p.strip * warps - 1) / ((long long)p.strip * warps));
    p.col_blocks = (a.D + 32 * PW - 1) / (32 * PW);
    p.wide_w = aligned16(a.weight);
    return p;
}
bool conv_vec(const HdlaConvArgs& a) {
    const int bytes = a.dtype == HDLA_F32 ? 16 : 8;
    auto ok = [&](const void* q) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; };
    return a.D % PW == 0 && a.x_batch % PW == 0 && a.x_token % PW == 0 && ok(a.x) && ok(a.h0) && ok(a.y) && ok(a.ht) && ok(a.dy) &&
           ok(a.dht) && ok(a.dx) && ok(a.dh0);
}

template <typename F>
void with_taps(int W, F f) {
    switch (W) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        case 4: return f(std::integral_constant<int, 4>());
        case 5: return f(std::integral_constant<int, 5>());
        case 6: return f(std::integral_constant<int, 6>());
        case 7: return f(std::integral_constant<int, 7>());
        default: return f(std::integral_constant<int, 8>());
    }
}
template <typename F>
void with_type(int dtype, bool vec, F f) {
    using F32 = std::integral_constant<int, HDLA_F32>;
    using BF16 = std::integral_constant<int, HDLA_BF16>;
    if (dtype == HDLA_F32) vec ? f(F32(), std::true_type()) : f(F32(), std::false_type());
    else vec ? f(BF16(), std::true_type()) : f(BF16(), std::false_type());
}

}  // namespace

int short_conv_fwd(const HdlaConvArgs& a, bool step, cudaStream_t st) {
    const ConvP p = plan(a, kFwdWarps);
    const long long grid = step ? (long long)p.col_blocks * ((a.B + 3) / 4) : (long long)p.col_blocks * p.strips * a.B;
    if (grid > 0x7fffffffLL) return fail(HDLA_ERR_UNSUPPORTED, "short_conv: %lld blocks", grid);
    with_type(a.dtype, conv_vec(a), [&](auto dt, auto v) {
        with_taps(a.W, [&](auto wt) {
            if (step) conv_step_kernel<dt, wt, v><<<(unsigned)grid, 128, 0, st>>>(p);
            else conv_fwd_kernel<dt, wt, v><<<(unsigned)grid, 32 * kFwdWarps, 0, st>>>(p);
        });
    });
    HDLA_CHECK_LAUNCH(step ? "conv_step_kernel" : "conv_fwd_kernel");
    return HDLA_OK;
}

size_t short_conv_bwd_workspace(const HdlaConvArgs& a) {
    return up256((size_t)a.B * plan(a, kBwdWarps).strips * (a.W + 1) * a.D * sizeof(float));
}

int short_conv_bwd(const HdlaConvArgs& a, float* part, cudaStream_t st) {
    ConvP p = plan(a, kBwdWarps);
    p.part = part;
    const long long grid = (long long)p.col_blocks * p.strips * a.B;
    if (grid > 0x7fffffffLL) return fail(HDLA_ERR_UNSUPPORTED, "short_conv: %lld blocks", grid);
    with_type(a.dtype, conv_vec(a), [&](auto dt, auto v) {
        with_taps(a.W, [&](auto wt) { conv_bwd_kernel<dt, wt, v><<<(unsigned)grid, 32 * kBwdWarps, 0, st>>>(p); });
    });
    HDLA_CHECK_LAUNCH("conv_bwd_kernel");
    ColJobs js{};
    js.n = 1;
    js.j[0] = ColJob{part, {a.dweight, a.dbias, nullptr}, (long long)(a.W + 1) * a.D, a.B * p.strips, a.W + 1, a.D, a.D, a.w_dtype, 1, 0, 0};
    return column_sum_launch(js, st);
}

}  // namespace hdla
