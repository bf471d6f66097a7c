// Selective state space scan, backward (the layout of the work is in selective_scan.cuh).
//
// With g = dy silu(z) and dh carried from the right, dh_t = C_t g_t + exp(d_{t+1} A) dh_{t+1}, and
//     dx = d sum_n dh B + skip g,   d(d) = x sum_n dh B + sum_n A dh e^{dA} h_{t-1},   dB = sum_c dh d x,   dC = sum_c g h,
//     dA = sum_t d dh e^{dA} h_{t-1},   dz = dy (y before the gate) silu'(z)
// The states are computed again, eight tokens at a time, from checkpoints that forward left every eight tokens (states cannot
// be run backwards: the decays underflow), and stay in registers for the eight steps back.  y before the gate and the sums for
// dC come out of the way there, the rest out of the way back.  Sums over channels (dB, dC) and over states go through shared
// memory as partial sums, which the block's threads add; the blocks' shares of dB and dC are written per tile of channels and
// added up in a fixed order by a last kernel, as are those of the weights.
//
// What bounds it: shared-memory cycles (62 % of their peak over the whole kernel, phases between barriers included), the issue
// of 24 instructions per (token, channel, state) (45 %) and two exponentials (38 %), none of which overlaps the others fully
// with the three warps a scheduler that the registers leave room for.  8 x 4096 x 2048, N = 16, bf16: 1485 us, the maps of 8
// segments 365 us, the last kernel's sums 38 us.
#include "selective_scan.cuh"

namespace hdla {
namespace {

// Walks over the segment's tokens from the last to the first.  Maps: only dh, from zero behind the segment (or from the final
// state's gradient of a sequence that ends inside it); what leaves at the segment's first token, with the sum of d, is the
// segment's map.
template <int DT, bool Vec, int NL, int CT, bool Maps>
__global__ void __launch_bounds__(kScanThreads, Maps ? 5 : 3) scan_bwd_kernel(const __grid_constant__ ScanP p) {
    using TileT = Tile<NL, CT>;
    constexpr int NP = TileT::NP, CH = TileT::CH, LC = TileT::LC, Pitch = TileT::Pitch, PW = 4, TB = kCheckpoint;
    constexpr int Groups = CH / PW, Items = TB * Groups, IT = (Items + kScanThreads - 1) / kScanThreads;
    constexpr int Rows = kScanWarps * LC;                        // partial sums over channels: one per warp and channel lane
    static_assert(CH % PW == 0 && kScanThreads % Groups == 0, "a thread's pieces are of one group of channels");
    __shared__ __align__(16) float s_d[TB][CH], s_g[TB][CH], s_u[Maps ? 1 : TB][CH], s_B[TB][NP], s_C[TB][NP];
    __shared__ __align__(16) float s_1[Maps ? 1 : TB * NL][Pitch], s_2[Maps ? 1 : TB * NL][Pitch];      // sums over n: y, then dh B; A dh e^{dA} h
    __shared__ __align__(16) float s_r[Maps ? 1 : TB][Rows][NP];                                        // sums over c: dC, then dB

    __shared__ __align__(16) float s_own[2][CH], s_sum[Maps ? 1 : 2][Maps ? 1 : kScanThreads][PW];

    const int segments = Maps ? p.n_seg - 1 : p.n_seg;           // (nothing precedes the first segment's map)
    TileT w(p, segments);
    if (Maps) ++w.k;
    const int T = p.a.T, D = p.a.D, N = p.a.N, t0 = w.k * p.seg, t1 = min(T, t0 + p.seg);
    const Seqs q{p.a.cu_seqlens, p.a.cu_seqlens ? p.a.n_seqs : 1, T};
    const int dead = q.end();
    const bool has_z = p.a.z != nullptr;

    const int cg = (threadIdx.x % Groups) * PW, valid = min(PW, w.count - cg), dch = w.d0 + cg;
    // in shared memory because registers are short here: the channels' dt_bias and skip weight, and this thread's sums of ddt, g x
    for (int c = threadIdx.x; c < CH; c += kScanThreads) {
        s_own[0][c] = p.a.dt_bias && c < w.count ? p.a.dt_bias[w.d0 + c] : 0.f;
        s_own[1][c] = p.a.skip && c < w.count ? p.a.skip[w.d0 + c] : 0.f;
    }
    if constexpr (!Maps)
        *reinterpret_cast<float4*>(s_sum[0][threadIdx.x]) = *reinterpret_cast<float4*>(s_sum[1][threadIdx.x]) = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
    constexpr int Ahead = kScanThreads / Groups;                 // tokens between a thread's pieces
    const int tok0 = threadIdx.x / Groups, last = t0 + (t1 - 1 - t0) / TB * TB, n0 = 4 * w.nl;
    Walk fx = Walk::of<DT>(p.a.x, w.b * p.a.x_batch + (last + tok0) * p.a.x_token + dch, p.a.x_token, Ahead);
    Walk fd = Walk::of<DT>(p.a.dt, w.b * p.a.dt_batch + (last + tok0) * p.a.dt_token + dch, p.a.dt_token, Ahead);
    Walk fz = Walk::of<DT>(p.a.z, w.b * p.a.z_batch + (last + tok0) * p.a.z_token + dch, p.a.z_token, Ahead);
    Walk fy = Walk::of<DT>(p.a.dy, ((long long)w.b * T + last + tok0) * D + dch, D, Ahead);
    const float* saved = p.a.checkpoints + (((size_t)w.b * ((T + kCheckpoint - 1) / kCheckpoint) + last / kCheckpoint) * D + w.d0 + w.c0) * NP + n0;
    BcTile<DT, NL, TB> bc(p, w.b, w.group, last);
    // the tile before this one is brought to L2 while this one is worked on (there are no registers to hold it)
    auto prefetch = [&] {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int ok = tok0 + i * Ahead < TB ? valid : 0;
            if (!Maps) fx.prefetch(i, ok, -TB);
            fd.prefetch(i, ok, -TB);
            if (has_z) fz.prefetch(i, ok, -TB);
            if (p.a.dy) fy.prefetch(i, ok, -TB);
        }
        bc.prefetch(-TB);
        if (!Maps)
#pragma unroll
            for (int c = 0; c < CT; ++c)
                if (w.c0 + c < w.count) prefetch_l2(saved - (size_t)D * NP + c * NP);
    };

    f2 A[CT][2], carry[CT][2], dA[CT][2], sum_d[CT];             // carry: exp(d_{t+1} A) dh_{t+1}
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        sum_d[c] = 0;
        A[c][0] = A[c][1] = carry[c][0] = carry[c][1] = dA[c][0] = dA[c][1] = 0;
        if (w.c0 + c < w.count) {
            ld_state(p.a.A + (size_t)(w.d0 + w.c0 + c) * N, n0, N, p.vec_state, A[c]);
            A[c][0] = f2_mul(A[c][0], f2_dup(kLog2e));
            A[c][1] = f2_mul(A[c][1], f2_dup(kLog2e));
        }
    }
    auto state_at = [&](int s, int c) { return ((size_t)(w.b + s) * D + w.d0 + w.c0 + c) * N; };
    auto from_end = [&](int s, f2 (&to)[CT][2]) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            to[c][0] = to[c][1] = 0;
            if (p.a.dht && w.c0 + c < w.count) ld_state(p.a.dht + state_at(s, c), n0, N, p.vec_state, to[c]);
        }
    };
    auto store_dh0 = [&](int s, const f2 (&from)[CT][2]) {
        if constexpr (!Maps) {
            if (!p.a.dh0) return;
#pragma unroll
            for (int c = 0; c < CT; ++c)
                if (w.c0 + c < w.count) st_state(p.a.dh0 + state_at(s, c), n0, N, p.vec_state, from[c]);
        }
    };
    auto empty = [&](int s) {                                    // an empty sequence: dh0 = dht
        f2 v[CT][2];
        from_end(s, v);
        store_dh0(s, v);
    };
    int s = q.starts_before(t1);
    if (t1 == T)
        for (int i = s + 1; i < q.n; ++i) empty(i);              // empty sequences at the back
    if (!Maps && q.off(s + 1) > t1) {                            // chain the maps of the segments up to the sequence's end
        const size_t row = (size_t)w.b * p.n_seg;
        const int ke = (q.off(s + 1) - 1) / p.seg;
#pragma unroll
        for (int c = 0; c < CT; ++c)
            if (w.c0 + c < w.count) {
                const int d = w.d0 + w.c0 + c;
                ld_quad(p.map_h + ((row + ke) * D + d) * NP + n0, carry[c]);
#pragma unroll 4
                for (int k = ke - 1; k > w.k; --k) {
                    f2 R[2];
                    ld_quad(p.map_h + ((row + k) * D + d) * NP + n0, R);
                    const f2 sd = f2_dup(p.map_d[(row + k) * D + d]);
                    carry[c][0] = f2_fma(ex2_pair(f2_mul(sd, A[c][0])), carry[c][0], R[0]);
                    carry[c][1] = f2_fma(ex2_pair(f2_mul(sd, A[c][1])), carry[c][1], R[1]);
                }
            }
    }
    // the block's sum over channels of what is in s_r, to the tile's share of dB (which = 0) or dC (1)
    constexpr int Parts = NL < 16 ? 16 / NL : 1, PerPass = kScanThreads / (Parts * NL);      // lanes that share an output, tokens at once
    const int out_tok = threadIdx.x / (Parts * NL), out_quad = threadIdx.x % NL, part = threadIdx.x / NL % Parts;
    const long long share_token = 2LL * p.a.G * NP;
    float* share = Maps ? nullptr : p.part_bc + (((size_t)(w.tile - p.first_tile) * p.a.B + w.b) * T + last + out_tok) * share_token + w.group * (2 * NP) +
                                       4 * out_quad + scatter_at<4, Parts>(w.lane, NL);
    auto add_channels = [&](int tokens, int which) {
#pragma unroll
        for (int o = 0; o < TB; o += PerPass) {
            f2 sum[2] = {0, 0};
#pragma unroll
            for (int r = 0; r < Rows / Parts; ++r) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&s_r[o + out_tok][r * Parts + part][4 * out_quad]);
                sum[0] = f2_add(sum[0], v.x);
                sum[1] = f2_add(sum[1], v.y);
            }
            float v[4];
            unpair(sum, v);
            scatter_sum<4, Parts>(v, w.lane, NL);
            if (o + out_tok < tokens && scatter_owner<4, Parts>(w.lane, NL))
#pragma unroll
                for (int i = 0; i < (Parts < 4 ? 4 / Parts : 1); ++i) {
                    float* to = share + o * share_token + which * NP + i;
                    *to = p.first_tile ? *to + v[i] : v[i];
                }
        }
    };
    const long long out0 = ((long long)w.b * T + last + tok0) * D + dch;

    for (int tb = last; tb >= t0; tb -= TB) {
        const int tokens = t1 - tb, live = dead - tb;            // (may be more than a tile; those from `live` on are of no sequence)
        f2 h[CT][2];
        if constexpr (!Maps)
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                h[c][0] = h[c][1] = 0;
                if (w.c0 + c < w.count) ld_quad(saved + c * NP, h[c]);
            }
        bc.template request<Vec>(min(tokens, live));                 // (rows of no sequence may hold anything, and anything times 0 is not 0)
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int tok = tok0 + i * Ahead, ok = tok < min(tokens, TB) ? valid : 0;
            if (Items % kScanThreads && tok >= TB) continue;
            Pack<DT, PW> rx = {}, rz = {};
            if (!Maps) rx = fx.load<DT, Vec>(i, ok);
            const Pack<DT, PW> rd = fd.load<DT, Vec>(i, ok), ry = fy.load<DT, Vec>(i, p.a.dy ? ok : 0);
            if (has_z) rz = fz.load<DT, Vec>(i, ok);
            f2 x[2], d[2], g[2], z[2], bias[2];
            ld_quad(&s_own[0][cg], bias);
            unpack_pairs<DT>(rx, x);
            unpack_pairs<DT>(rd, d);
            unpack_pairs<DT>(ry, g);
            unpack_pairs<DT>(rz, z);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                d[c] = f2_add(d[c], bias[c]);
                if (p.a.softplus) d[c] = softplus_pair(d[c]);
                if (has_z) g[c] = f2_mul(g[c], f2_mul(z[c], sigmoid_pair(z[c])));
                if (!Maps) x[c] = f2_mul(x[c], d[c]);
            }
            if (live < TB && tok >= live) d[0] = d[1] = g[0] = g[1] = x[0] = x[1] = 0;
            st_pairs(&s_d[tok][cg], d);
            st_pairs(&s_g[tok][cg], g);
            if (!Maps) st_pairs(&s_u[tok][cg], x);
        }
        bc.put(&s_B[0][0], &s_C[0][0]);
        if (tb > t0) prefetch();
        __syncthreads();

        // sequences that start in this tile, and whether one ends there
        unsigned starts = 0;
        for (int i = s; i >= 0; --i) {
            const int o = q.off(i);
            if (o < tb) break;
            if (o < tb + TB) starts |= 1u << (o - tb);
        }
        const bool edge = starts != 0 || q.off(s + 1) <= tb + TB;

        f2 before[Maps ? 1 : TB][CT][2], y[IT][2];               // the state that token j's decay multiplies; y before the gate
        // the two ways over the tile; without edges they are free of branches, so that the tokens' latencies overlap
        auto there = [&](auto edges) {
            constexpr bool with_edges = decltype(edges)::value;
#pragma unroll
            for (int j = 0; j < TB; ++j) {
                if (with_edges && (starts >> j & 1)) {
                    const int first = q.ends_behind(tb + j);
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        h[c][0] = h[c][1] = 0;
                        if (first < q.n && p.a.h0 && w.c0 + c < w.count)
                            ld_state(p.a.h0 + state_at(first, c), n0, N, p.vec_state, h[c]);
                    }
                }
                f2 d[CT], u[CT], g[CT], B[2], C[2], dC[2];
                ld_twice<CT>(&s_d[j][w.c0], d);
                ld_twice<CT>(&s_u[j][w.c0], u);
                ld_twice<CT>(&s_g[j][w.c0], g);
                ld_quad(&s_B[j][n0], B);
                ld_quad(&s_C[j][n0], C);
                float sum[CT];
#pragma unroll
                for (int c = 0; c < CT; ++c) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        before[j][c][i] = h[c][i];
                        h[c][i] = f2_fma(ex2_pair(f2_mul(d[c], A[c][i])), h[c][i], f2_mul(u[c], B[i]));
                        dC[i] = c ? f2_fma(g[c], h[c][i], dC[i]) : f2_mul(g[c], h[c][i]);
                    }
                    sum[c] = f2_sum(f2_fma(C[1], h[c][1], f2_mul(C[0], h[c][0])));
                }
                st_channels<CT>(&s_1[j * NL + w.nl][w.c0], sum);
                st_quad(&s_r[j][w.warp * LC + w.lane / NL][n0], dC);
            }
        };
        auto back = [&](auto edges) {
            constexpr bool with_edges = decltype(edges)::value;
#pragma unroll
            for (int j = TB - 1; j >= 0; --j) {
                const int t = tb + j;
                if (with_edges && q.off(s + 1) == t + 1) from_end(s, carry);
                f2 d[CT], g[CT], C[2];
                ld_twice<CT>(&s_d[j][w.c0], d);
                ld_twice<CT>(&s_g[j][w.c0], g);
                ld_quad(&s_C[j][n0], C);
                if constexpr (Maps) {
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        sum_d[c] = f2_add(sum_d[c], d[c]);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            carry[c][i] = f2_mul(ex2_pair(f2_mul(d[c], A[c][i])), f2_fma(g[c], C[i], carry[c][i]));
                    }
                } else {
                    f2 u[CT], B[2], dB[2];
                    float dot[CT], dec[CT];
                    ld_twice<CT>(&s_u[j][w.c0], u);
                    ld_quad(&s_B[j][n0], B);
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        f2 sum_b, sum_a;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const f2 a = ex2_pair(f2_mul(d[c], A[c][i]));
                            const f2 dh = f2_fma(g[c], C[i], carry[c][i]);
                            carry[c][i] = f2_mul(a, dh);
                            const f2 v = f2_mul(carry[c][i], before[j][c][i]);
                            dB[i] = c ? f2_fma(u[c], dh, dB[i]) : f2_mul(u[c], dh);
                            sum_b = i ? f2_fma(dh, B[i], sum_b) : f2_mul(dh, B[i]);
                            sum_a = i ? f2_fma(v, A[c][i], sum_a) : f2_mul(v, A[c][i]);
                            dA[c][i] = f2_fma(v, d[c], dA[c][i]);
                        }
                        dot[c] = f2_sum(sum_b);
                        dec[c] = f2_sum(sum_a);
                    }
                    st_channels<CT>(&s_1[j * NL + w.nl][w.c0], dot);
                    st_channels<CT>(&s_2[j * NL + w.nl][w.c0], dec);
                    st_quad(&s_r[j][w.warp * LC + w.lane / NL][n0], dB);
                }
                if (with_edges) {
                    while (s >= 0 && q.off(s) >= t) {            // token t is a sequence's first (and empty ones precede it)
                        if (q.off(s + 1) > t) store_dh0(s, carry);
                        else empty(s);
                        --s;
                    }
                    if (s < 0) s = 0;                            // (only at token 0)
                }
            }
        };
        if constexpr (!Maps) {
            if (edge) there(std::true_type());
            else there(std::false_type());
            __syncthreads();
            add_channels(tokens, 1);
            if (has_z)
#pragma unroll
                for (int i = 0; i < IT; ++i)
                    if (Items % kScanThreads == 0 || tok0 + i * Ahead < TB) add_partial<NL>(&s_1[(tok0 + i * Ahead) * NL][cg], Pitch, y[i]);
            __syncthreads();
        }
        if (edge) back(std::true_type());
        else back(std::false_type());
        __syncthreads();
        if constexpr (!Maps) {
            add_channels(tokens, 0);
            share -= TB * share_token;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int tok = tok0 + i * Ahead;
                if (tok >= min(TB, tokens)) continue;
                // (the inputs come from L1 or L2 once more)
                Pack<DT, PW> rz = {};
                const Pack<DT, PW> rx = fx.load<DT, Vec>(i, valid), rd = fd.load<DT, Vec>(i, valid), ry = fy.load<DT, Vec>(i, p.a.dy ? valid : 0);
                if (has_z) rz = fz.load<DT, Vec>(i, valid);
                f2 x[2], v[2], z[2], dy[2], d[2], dot[2], dec[2], dx[2], dd[2], dz[2], g[2], bias[2], skip[2];
                ld_quad(&s_d[tok][cg], d);
                ld_quad(&s_g[tok][cg], g);
                ld_quad(&s_own[0][cg], bias);
                ld_quad(&s_own[1][cg], skip);
                add_partial<NL>(&s_1[tok * NL][cg], Pitch, dot);
                add_partial<NL>(&s_2[tok * NL][cg], Pitch, dec);
                unpack_pairs<DT>(rx, x);
                unpack_pairs<DT>(rd, v);
                unpack_pairs<DT>(ry, dy);
                unpack_pairs<DT>(rz, z);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (has_z) {                                 // silu' = s + z s (1 - s)
                        const f2 sg = sigmoid_pair(z[c]), zs = f2_mul(z[c], sg);
                        const f2 slope = f2_fma(zs, f2_fma(sg, f2_dup(-1.f), f2_dup(1.f)), sg);
                        dz[c] = f2_mul(f2_mul(dy[c], f2_fma(skip[c], x[c], y[i][c])), slope);
                    }
                    dx[c] = f2_fma(d[c], dot[c], f2_mul(skip[c], g[c]));
                    dd[c] = f2_fma(x[c], dot[c], f2_mul(dec[c], f2_dup(kLn2)));      // (A is held times log2 e)
                    if (p.a.softplus) dd[c] = f2_mul(dd[c], sigmoid_pair(f2_add(v[c], bias[c])));
                    if (live < TB && tok >= live) dx[c] = dd[c] = dz[c] = x[c] = 0;  // (g is zero)
                }
                {
                    f2 dskip[2], dbias[2];
                    ld_quad(s_sum[0][threadIdx.x], dbias);
                    ld_quad(s_sum[1][threadIdx.x], dskip);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        dskip[c] = f2_fma(g[c], x[c], dskip[c]);
                        dbias[c] = f2_add(dbias[c], dd[c]);
                    }
                    st_pairs(s_sum[0][threadIdx.x], dbias);
                    st_pairs(s_sum[1][threadIdx.x], dskip);
                }
                const long long at = out0 + (long long)(tb - last + i * Ahead) * D;
                float out[PW];
                unpair(dx, out);
                st_pack<DT, PW, Vec>(p.a.dx, at, valid, out);
                unpair(dd, out);
                st_pack<DT, PW, Vec>(p.a.ddt, at, valid, out);
                unpair(dz, out);
                if (has_z) st_pack<DT, PW, Vec>(p.a.dz, at, valid, out);
            }
        }
        fx.move(-TB); fd.move(-TB); fz.move(-TB); fy.move(-TB);
        bc.from.move(-TB);
        saved -= (size_t)D * NP;
    }
    const size_t row = (size_t)w.b * p.n_seg + w.k;
#pragma unroll
    for (int c = 0; c < CT; ++c)
        if (w.c0 + c < w.count) {
            const size_t at = row * D + w.d0 + w.c0 + c;
            if (Maps) {
                float a, b;
                f2_unpack(sum_d[c], a, b);
                st_quad(p.map_h + at * NP + n0, carry[c]);
                if (w.nl == 0) p.map_d[at] = a;
            } else {
                st_quad(p.part_a + at * NP + n0, dA[c]);
            }
        }
    if constexpr (!Maps) {                                       // dskip and dbias: over the threads of a group of channels
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * w.count; i += kScanThreads) {
            const int what = i >= w.count, c = i - what * w.count;         // 0: g x, 1: ddt
            float sum = 0.f;
            for (int k = c / PW; k < kScanThreads; k += Groups) sum += s_sum[what ? 0 : 1][k][c % PW];
            p.part_v[(row * 2 + what) * D + w.d0 + c] = sum;
        }
    }
}

}  // namespace

int selective_scan_bwd(const HdlaScanArgs& a, unsigned char* ws, cudaStream_t st) {
    const ScanPlan r = scan_plan(a, true);
    const ScanP p = scan_params(a, r, scan_work(a, r, true), ws);
    const long long blocks = (long long)a.G * r.tiles * a.B;
    if (blocks * r.n_seg > 0x7fffffffLL) return fail(HDLA_ERR_UNSUPPORTED, "selective_scan: %lld blocks", blocks * r.n_seg);
    auto launch = [&](bool maps, const ScanP& part) {
        const unsigned grid = static_cast<unsigned>((long long)a.G * part.tile_count * a.B * (r.n_seg - maps));
        with_type(a.dtype, scan_vec(a), [&](auto dt, auto vec) {
            with_lanes(scan_lanes(a.N), [&](auto nl) {
                constexpr int ct = nl == 2 || nl == 32 ? 1 : 2;  // (as in scan_plan; two channels a lane would not fit into shared memory)
                if (maps) scan_bwd_kernel<dt, vec, nl, ct, true><<<grid, kScanThreads, 0, st>>>(part);
                else scan_bwd_kernel<dt, vec, nl, ct, false><<<grid, kScanThreads, 0, st>>>(part);
            });
        });
    };
    if (r.n_seg > 1) {
        launch(true, p);
        HDLA_CHECK_LAUNCH("scan_bwd_maps_kernel");
    }
    const int slots = scan_slots(a, r);
    for (int t = 0; t < r.tiles; t += slots) {
        ScanP part = p;
        part.first_tile = t;
        part.tile_count = r.tiles - t < slots ? r.tiles - t : slots;
        launch(false, part);
        HDLA_CHECK_LAUNCH("scan_bwd_kernel");
    }
    const int np = 4 * scan_lanes(a.N), rows = a.B * r.n_seg;
    ColJobs js{};
    js.j[js.n++] = ColJob{p.part_bc, {a.dB, a.dC, nullptr}, (long long)a.B * a.T * a.G * 2 * np, slots, 2, np, a.N, a.dtype, 0, 0, 0};
    js.j[js.n++] = ColJob{p.part_a, {a.dA, nullptr, nullptr}, (long long)a.D * np, rows, 1, np, a.N, HDLA_F32, 0, 0, 0};
    if (a.dskip || a.ddt_bias)
        js.j[js.n++] = ColJob{p.part_v, {a.dskip, a.ddt_bias, nullptr}, 2LL * a.D, rows, 2, a.D, a.D, HDLA_F32, 0, 0, 0};
    return column_sum_launch(js, st);
}

}  // namespace hdla
