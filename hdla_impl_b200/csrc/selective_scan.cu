// Selective state space scan.  Per channel c with N states, c's group sharing B and C:
//     d_t = softplus(dt_t + bias) (or dt_t + bias),  h_t[n] = exp(d_t A[n]) h_{t-1}[n] + d_t x_t B_t[n]
//     y_t = (sum_n C_t[n] h_t[n] + skip x_t) silu(z_t)
//
// Layout of the work.  A warp holds the states of (32 / NL) * CT channels in registers: NL lanes share a channel's states,
// four a lane, and a lane has CT channels, so that one 16-byte broadcast read of B (and C) serves 4 * CT states and the sum
// over n takes log2(NL) shuffles for CT channels together.  Four warps make a block; it walks over its tokens in tiles, in
// three steps: what is done once per (token, channel) -- softplus, d x, gates -- by all threads on 16-byte pieces into
// shared memory; the recurrence; the outputs.  The next tile's inputs are requested before the recurrence of this one.
// All arithmetic is fp32, the outputs are rounded once.
//
// What bounds it: the exponentials, one per (token, channel, state) and 16 a clock and SM, and four fused multiply-adds
// beside each; HBM traffic is a third of that time at N = 16.
//
// Long rows of few channels are cut into segments.  What a segment does to a state is exp(A sum d) h + F, and its sum of d
// and F come from a first kernel that runs the recurrence alone, from zero; the second kernel's blocks chain the maps of
// the segments before theirs.
//
// Backward.  With g = dy silu(z) and dh carried from the right, dh_t = C_t g_t + exp(d_{t+1} A) dh_{t+1}.  The states are
// computed again, eight tokens at a time, from checkpoints that forward left every eight tokens (states cannot be run
// backwards: the decays underflow), and stay in registers for the eight steps back.  Sums over channels (dB, dC) are
// taken over lanes and warps, written per tile of channels and added up in a fixed order by a last kernel.
#include "f32x2.cuh"
#include "ssm.cuh"

namespace hdla {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kCheckpoint = 8;                     // tokens between two saved states
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct ScanP {
    HdlaScanArgs a;
    int Dg, tiles;             // channels of a group, tiles of channels per group
    int seg, n_seg;            // tokens of a segment (a multiple of 16), segments
    bool vec_bc, vec_state;    // 4 states of B and C / of the states as one access
    float *map_h, *map_d;      // [B][n_seg][D][NP], [B][n_seg][D]
    float *part_bc, *part_a, *part_v;      // [tiles][B][T][G][2][NP], [B * n_seg][D][NP], [B * n_seg][2][D]
};

__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ f2 ex2_pair(f2 x) {
    float a, b;
    f2_unpack(x, a, b);
    return f2_pack(ex2(a), ex2(b));
}

// Sums over M lanes whose numbers differ in the bits from `low` on, of N values each: each step halves the values a lane
// still carries, and once one is left it is summed by all.  Lane ends with max(1, N / M) sums, from scatter_at() on.
template <int N, int M>
__device__ __forceinline__ void scatter_sum(float (&v)[N], int lane, int low) {
    int n = N;
#pragma unroll
    for (int m = 1; m < M; m <<= 1) {
        if (n > 1) {
            const bool up = (lane & (m * low)) != 0;
            n >>= 1;
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                if (i < n) {
                    const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, give, m * low);
                }
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], m * low);
        }
    }
}
template <int N, int M>
__device__ __forceinline__ int scatter_at(int lane, int low) {
    int n = N, at = 0;
#pragma unroll
    for (int m = 1; m < M; m <<= 1)
        if (n > 1) {
            n >>= 1;
            if (lane & (m * low)) at += n;
        }
    return at;
}

// four states of one channel (state 0 of the channel at `at`, this lane's first at n0), zero beyond N
__device__ __forceinline__ void ld_state(const float* at, int n0, int N, bool vec, f2 (&h)[2]) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (vec) {
        if (n0 < N) {
            const float4 q = *reinterpret_cast<const float4*>(at + n0);
            v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + i < N) v[i] = at[n0 + i];
    }
    h[0] = f2_pack(v[0], v[1]);
    h[1] = f2_pack(v[2], v[3]);
}
__device__ __forceinline__ void st_state(float* at, int n0, int N, bool vec, const f2 (&h)[2]) {
    float v[4];
    f2_unpack(h[0], v[0], v[1]);
    f2_unpack(h[1], v[2], v[3]);
    if (vec) {
        if (n0 < N) *reinterpret_cast<float4*>(at + n0) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + i < N) at[n0 + i] = v[i];
    }
}
// ... of the library's own arrays, where NP states are laid out
__device__ __forceinline__ void ld_quad(const float* at, f2 (&h)[2]) {
    const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(at);
    h[0] = q.x; h[1] = q.y;
}
__device__ __forceinline__ void st_quad(float* at, const f2 (&h)[2]) { *reinterpret_cast<ulonglong2*>(at) = make_ulonglong2(h[0], h[1]); }

template <int CT>
__device__ __forceinline__ void ld_channels(const float* at, float (&v)[CT]) {
    if constexpr (CT == 4) {
        const float4 q = *reinterpret_cast<const float4*>(at);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else if constexpr (CT == 2) {
        const float2 q = *reinterpret_cast<const float2*>(at);
        v[0] = q.x; v[1] = q.y;
    } else {
        v[0] = *at;
    }
}

// Which part of the problem a block has, and its lanes their states.
template <int NL, int CT>
struct Tile {
    static constexpr int LC = 32 / NL, NP = 4 * NL, CPW = LC * CT, CH = kWarps * CPW;
    int b, group, tile, k;            // sequence row, group, tile of the group, segment
    int d0, count;                    // first channel of the tile, channels it has
    int lane, warp, nl, c0;           // this lane's first state is 4 * nl, its first channel c0 (in the tile)
    __device__ __forceinline__ explicit Tile(const ScanP& p, int segments) {
        const int per_row = p.a.G * p.tiles;
        const int x = blockIdx.x % per_row, r = blockIdx.x / per_row;
        group = x / p.tiles; tile = x % p.tiles;
        k = r % segments; b = r / segments;
        d0 = group * p.Dg + tile * CH;
        count = min(CH, p.Dg - tile * CH);
        lane = threadIdx.x & 31; warp = threadIdx.x >> 5;
        nl = lane % NL;
        c0 = warp * CPW + lane / NL * CT;
    }
};

// B and C of a tile of tokens: four states a piece, requested early and put into shared memory as fp32.
template <int DT, int NL, int TB>
struct BcTile {
    static constexpr int NP = 4 * NL, Pieces = TB * NL * 2, PerThread = (Pieces + kThreads - 1) / kThreads;
    Pack<DT, 4> raw[PerThread];
    __device__ __forceinline__ void request(const ScanP& p, int b, int group, int tb) {
#pragma unroll
        for (int i = 0; i < PerThread; ++i) {
            const int piece = threadIdx.x + i * kThreads, quad = piece % NL, which = piece / NL % 2, t = tb + piece / (2 * NL);
            const int valid = piece < Pieces && t < p.a.T ? min(4, p.a.N - 4 * quad) : 0;
            const void* base = which ? p.a.Cm : p.a.Bm;
            const long long at = (which ? b * p.a.C_batch + t * p.a.C_token + group * p.a.C_group
                                        : b * p.a.B_batch + t * p.a.B_token + group * p.a.B_group) + 4 * quad;
            raw[i] = p.vec_bc ? ld_pack<DT, 4, true>(base, at, valid) : ld_pack<DT, 4, false>(base, at, valid);
        }
    }
    __device__ __forceinline__ void put(float* sB, float* sC) const {
#pragma unroll
        for (int i = 0; i < PerThread; ++i) {
            const int piece = threadIdx.x + i * kThreads, quad = piece % NL, which = piece / NL % 2, tok = piece / (2 * NL);
            if (piece < Pieces) {
                float f[4];
                unpack<DT, 4>(raw[i], f);
                *reinterpret_cast<float4*>((which ? sC : sB) + tok * NP + 4 * quad) = make_float4(f[0], f[1], f[2], f[3]);
            }
        }
    }
};

// ------------------------------------------------------------------------------------------ forward
// Maps: only the recurrence, from zero at the segment's first token (or from the initial state of a sequence that starts
// inside it); its last state and sum of d are the segment's map.
template <int DT, bool Vec, int NL, int CT, bool Maps>
__global__ void __launch_bounds__(kThreads) scan_fwd_kernel(const __grid_constant__ ScanP p) {
    using TileT = Tile<NL, CT>;
    constexpr int NP = TileT::NP, CH = TileT::CH, PW = DT == HDLA_F32 ? 4 : 8;
    constexpr int TB = CH > 128 ? 8 : 16, Groups = CH / PW, Items = TB * Groups, IT = (Items + kThreads - 1) / kThreads;
    static_assert(CH % PW == 0 && (kThreads % Groups) == 0, "a thread's pieces are of one group of channels");
    __shared__ __align__(16) float s_d[TB][CH], s_u[TB][CH], s_y[Maps ? 1 : TB][CH], s_B[TB][NP], s_C[TB][NP];

    const int segments = Maps ? p.n_seg - 1 : p.n_seg;           // (nothing follows the last segment's map)
    const TileT w(p, segments);
    const int T = p.a.T, D = p.a.D, N = p.a.N, t0 = w.k * p.seg, t1 = min(T, t0 + p.seg);
    const Seqs q{p.a.cu_seqlens, p.a.cu_seqlens ? p.a.n_seqs : 1, T};
    const int dead = q.end();

    // pieces of a (token, channels) tile: this thread's are all of one group of channels
    const int cg = (threadIdx.x % Groups) * PW, valid = min(PW, w.count - cg), dch = w.d0 + cg;
    float bias[PW], skip[PW];
#pragma unroll
    for (int c = 0; c < PW; ++c) {
        bias[c] = p.a.dt_bias && c < valid ? p.a.dt_bias[dch + c] : 0.f;
        skip[c] = !Maps && p.a.skip && c < valid ? p.a.skip[dch + c] : 0.f;
    }
    Pack<DT, PW> nx[IT], nd[IT], nz[IT];
    BcTile<DT, NL, TB> bc;
    auto request = [&](int tb) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int item = threadIdx.x + i * kThreads, t = tb + item / Groups;
            const int ok = item < Items && t < t1 ? valid : 0;
            nx[i] = ld_pack<DT, PW, Vec>(p.a.x, w.b * p.a.x_batch + t * p.a.x_token + dch, ok);
            nd[i] = ld_pack<DT, PW, Vec>(p.a.dt, w.b * p.a.dt_batch + t * p.a.dt_token + dch, ok);
            if (!Maps && p.a.z) nz[i] = ld_pack<DT, PW, Vec>(p.a.z, w.b * p.a.z_batch + t * p.a.z_token + dch, ok);
        }
        bc.request(p, w.b, w.group, tb);
    };
    request(t0);

    // the lane's decay rates and states
    f2 A[CT][2], h[CT][2];
    float sum_d[CT];
    const int n0 = 4 * w.nl;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        sum_d[c] = 0.f;
        A[c][0] = A[c][1] = 0;
        if (w.c0 + c < w.count) {
            ld_state(p.a.A + (size_t)(w.d0 + w.c0 + c) * N, n0, N, p.vec_state, A[c]);
            A[c][0] = f2_mul(A[c][0], f2_dup(kLog2e));
            A[c][1] = f2_mul(A[c][1], f2_dup(kLog2e));
        }
    }
    auto begin = [&](int s) {                                    // the state before a sequence's first token
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            h[c][0] = h[c][1] = 0;
            if (s < q.n && p.a.h0 && w.c0 + c < w.count)
                ld_state(p.a.h0 + ((size_t)(w.b + s) * D + w.d0 + w.c0 + c) * N, n0, N, p.vec_state, h[c]);
        }
    };
    auto finish = [&](int s) {
        if constexpr (!Maps) {
            if (!p.a.ht) return;
#pragma unroll
            for (int c = 0; c < CT; ++c)
                if (w.c0 + c < w.count) st_state(p.a.ht + ((size_t)(w.b + s) * D + w.d0 + w.c0 + c) * N, n0, N, p.vec_state, h[c]);
        }
    };
    int s = q.ends_behind(t0);
    if (t0 == 0)
        for (int i = 0; i < s; ++i) { begin(i); finish(i); }     // empty sequences at the front
    const int start = s < q.n ? min(q.off(s), t0) : t0;
    begin(start == t0 ? s : q.n);
    if (!Maps && start < t0) {                                   // chain the maps of the segments since the sequence's start
        const size_t row = (size_t)w.b * p.n_seg;
#pragma unroll
        for (int c = 0; c < CT; ++c)
            if (w.c0 + c < w.count) {
                const int d = w.d0 + w.c0 + c, k0 = start / p.seg;
                ld_quad(p.map_h + ((row + k0) * D + d) * NP + n0, h[c]);
#pragma unroll 4
                for (int k = k0 + 1; k < w.k; ++k) {
                    f2 F[2];
                    ld_quad(p.map_h + ((row + k) * D + d) * NP + n0, F);
                    const f2 sd = f2_dup(p.map_d[(row + k) * D + d]);
                    h[c][0] = f2_fma(ex2_pair(f2_mul(sd, A[c][0])), h[c][0], F[0]);
                    h[c][1] = f2_fma(ex2_pair(f2_mul(sd, A[c][1])), h[c][1], F[1]);
                }
            }
    }
    int end = s < q.n ? q.off(s + 1) : 0x7fffffff;

    auto token = [&](int tb, int j) {
        if (!Maps && j % kCheckpoint == 0 && p.a.checkpoints && tb + j < t1) {
            const size_t at = ((size_t)w.b * ((T + kCheckpoint - 1) / kCheckpoint) + (tb + j) / kCheckpoint) * D + w.d0 + w.c0;
#pragma unroll
            for (int c = 0; c < CT; ++c)
                if (w.c0 + c < w.count) st_quad(p.a.checkpoints + (at + c) * NP + n0, h[c]);
        }
        float d[CT], u[CT], y[CT];
        f2 B[2], C[2];
        ld_channels<CT>(&s_d[j][w.c0], d);
        ld_channels<CT>(&s_u[j][w.c0], u);
        ld_quad(&s_B[j][n0], B);
        if (!Maps) ld_quad(&s_C[j][n0], C);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const f2 d2 = f2_dup(d[c]), u2 = f2_dup(u[c]);
            h[c][0] = f2_fma(ex2_pair(f2_mul(d2, A[c][0])), h[c][0], f2_mul(u2, B[0]));
            h[c][1] = f2_fma(ex2_pair(f2_mul(d2, A[c][1])), h[c][1], f2_mul(u2, B[1]));
            if (Maps) sum_d[c] += d[c];
            else y[c] = f2_sum(f2_fma(C[1], h[c][1], f2_mul(C[0], h[c][0])));
        }
        if (!Maps) {
            scatter_sum<CT, NL>(y, w.lane, 1);
            const int at = w.c0 + scatter_at<CT, NL>(w.lane, 1);
#pragma unroll
            for (int i = 0; i < (CT > NL ? CT / NL : 1); ++i) s_y[j][at + i] = y[i];
        }
    };

    for (int tb = t0; tb < t1; tb += TB) {
        Pack<DT, PW> cx[IT], cz[IT];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int item = threadIdx.x + i * kThreads, tok = item / Groups, t = tb + tok;
            cx[i] = nx[i];
            if (!Maps) cz[i] = nz[i];
            if (item >= Items) continue;
            float x[PW], d[PW], e;
            unpack<DT, PW>(nx[i], x);
            unpack<DT, PW>(nd[i], d);
#pragma unroll
            for (int c = 0; c < PW; ++c) {
                d[c] += bias[c];
                if (p.a.softplus) d[c] = softplus_of(d[c], e);
                if (t >= dead) d[c] = x[c] = 0.f;                // a token of no sequence, or behind the last one
                x[c] *= d[c];
            }
#pragma unroll
            for (int c = 0; c < PW; c += 4) {
                *reinterpret_cast<float4*>(&s_d[tok][cg + c]) = make_float4(d[c], d[c + 1], d[c + 2], d[c + 3]);
                *reinterpret_cast<float4*>(&s_u[tok][cg + c]) = make_float4(x[c], x[c + 1], x[c + 2], x[c + 3]);
            }
        }
        bc.put(&s_B[0][0], &s_C[0][0]);
        if (tb + TB < t1) request(tb + TB);
        __syncthreads();
        if (end > tb + TB) {
#pragma unroll 8
            for (int j = 0; j < TB; ++j) token(tb, j);
        } else {                                                 // a sequence ends in this tile
            const int nt = min(TB, t1 - tb);
#pragma unroll 1
            for (int j = 0; j < nt; ++j) {
                token(tb, j);
                while (end <= tb + j + 1) {
                    finish(s);
                    ++s;
                    begin(s);
                    end = s < q.n ? q.off(s + 1) : 0x7fffffff;
                }
            }
        }
        __syncthreads();
        if (!Maps) {
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int item = threadIdx.x + i * kThreads, tok = item / Groups, t = tb + tok;
                if (item >= Items || t >= t1) continue;
                float x[PW], z[PW], y[PW];
                unpack<DT, PW>(cx[i], x);
#pragma unroll
                for (int c = 0; c < PW; c += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(&s_y[tok][cg + c]);
                    y[c] = v.x; y[c + 1] = v.y; y[c + 2] = v.z; y[c + 3] = v.w;
                }
                if (p.a.z) unpack<DT, PW>(cz[i], z);
#pragma unroll
                for (int c = 0; c < PW; ++c) {
                    if (p.a.skip) y[c] = fmaf(skip[c], x[c], y[c]);
                    if (p.a.z) y[c] *= z[c] * sigmoid_of(z[c]);
                    if (t >= dead) y[c] = 0.f;
                }
                st_pack<DT, PW, Vec>(p.a.y, ((long long)w.b * T + t) * D + dch, valid, y);
            }
        }
    }
    if (Maps) {
        const size_t row = ((size_t)w.b * p.n_seg + w.k) * D + w.d0 + w.c0;
#pragma unroll
        for (int c = 0; c < CT; ++c)
            if (w.c0 + c < w.count) {
                st_quad(p.map_h + (row + c) * NP + n0, h[c]);
                if (w.nl == 0) p.map_d[row + c] = sum_d[c];
            }
    }
}

// ------------------------------------------------------------------------------------------ backward
// Walks over the segment's tokens from the last to the first.  Maps: only dh, from zero behind the segment (or from the final
// state's gradient of a sequence that ends inside it); what leaves at the segment's first token, with the sum of d, is the
// segment's map.
template <int DT, bool Vec, int NL, int CT, bool Maps>
__global__ void __launch_bounds__(kThreads) scan_bwd_kernel(const __grid_constant__ ScanP p) {
    using TileT = Tile<NL, CT>;
    constexpr int NP = TileT::NP, CH = TileT::CH, LC = TileT::LC, PW = 4, TB = kCheckpoint;
    constexpr int Groups = CH / PW, Items = TB * Groups, IT = (Items + kThreads - 1) / kThreads;
    static_assert(CH % PW == 0 && (kThreads % Groups) == 0, "a thread's pieces are of one group of channels");
    __shared__ __align__(16) float s_d[TB][CH], s_g[TB][CH], s_B[TB][NP], s_C[TB][NP];
    __shared__ __align__(16) float s_u[Maps ? 1 : TB][CH], s_dot[Maps ? 1 : TB][CH], s_dec[Maps ? 1 : TB][CH], s_y[Maps ? 1 : TB][CH];
    __shared__ __align__(16) float red[Maps ? 1 : kWarps][TB][2 * NP];

    const int segments = Maps ? p.n_seg - 1 : p.n_seg;           // (nothing precedes the first segment's map)
    TileT w(p, segments);
    if (Maps) ++w.k;
    const int T = p.a.T, D = p.a.D, N = p.a.N, t0 = w.k * p.seg, t1 = min(T, t0 + p.seg);
    const Seqs q{p.a.cu_seqlens, p.a.cu_seqlens ? p.a.n_seqs : 1, T};
    const int dead = q.end();
    const bool has_z = p.a.z != nullptr;

    const int cg = (threadIdx.x % Groups) * PW, valid = min(PW, w.count - cg), dch = w.d0 + cg;
    float bias[PW], skip[PW], dskip[PW] = {}, dbias[PW] = {};
#pragma unroll
    for (int c = 0; c < PW; ++c) {
        bias[c] = p.a.dt_bias && c < valid ? p.a.dt_bias[dch + c] : 0.f;
        skip[c] = p.a.skip && c < valid ? p.a.skip[dch + c] : 0.f;
    }
    Pack<DT, PW> nx[IT], nd[IT], nz[IT], ny[IT];
    BcTile<DT, NL, TB> bc;
    f2 nh[CT][2];                                                // the next tile's checkpoint
    const int n0 = 4 * w.nl;
    auto request = [&](int tb) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int item = threadIdx.x + i * kThreads, t = tb + item / Groups;
            const int ok = item < Items && t < t1 ? valid : 0;
            if (!Maps) nx[i] = ld_pack<DT, PW, Vec>(p.a.x, w.b * p.a.x_batch + t * p.a.x_token + dch, ok);
            nd[i] = ld_pack<DT, PW, Vec>(p.a.dt, w.b * p.a.dt_batch + t * p.a.dt_token + dch, ok);
            if (has_z) nz[i] = ld_pack<DT, PW, Vec>(p.a.z, w.b * p.a.z_batch + t * p.a.z_token + dch, ok);
            ny[i] = ld_pack<DT, PW, Vec>(p.a.dy, ((long long)w.b * T + t) * D + dch, p.a.dy ? ok : 0);
        }
        bc.request(p, w.b, w.group, tb);
        if (!Maps) {
            const size_t at = ((size_t)w.b * ((T + kCheckpoint - 1) / kCheckpoint) + tb / kCheckpoint) * D + w.d0 + w.c0;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                nh[c][0] = nh[c][1] = 0;
                if (w.c0 + c < w.count) ld_quad(p.a.checkpoints + (at + c) * NP + n0, nh[c]);
            }
        }
    };
    const int last = t0 + (t1 - 1 - t0) / TB * TB;
    request(last);

    f2 A[CT][2], carry[CT][2], dA[CT][2];                        // carry: exp(d_{t+1} A) dh_{t+1}
    float sum_d[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        sum_d[c] = 0.f;
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

    for (int tb = last; tb >= t0; tb -= TB) {
        Pack<DT, PW> cx[IT], cd[IT], cz[IT], cy[IT];
        f2 h[CT][2];
#pragma unroll
        for (int c = 0; c < CT; ++c) { h[c][0] = nh[c][0]; h[c][1] = nh[c][1]; }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int item = threadIdx.x + i * kThreads, tok = item / Groups, t = tb + tok;
            cx[i] = nx[i]; cd[i] = nd[i]; cz[i] = nz[i]; cy[i] = ny[i];
            if (item >= Items) continue;
            float x[PW], d[PW], g[PW], z[PW], e;
            if (!Maps) unpack<DT, PW>(nx[i], x);
            unpack<DT, PW>(nd[i], d);
            unpack<DT, PW>(ny[i], g);
            if (has_z) unpack<DT, PW>(nz[i], z);
#pragma unroll
            for (int c = 0; c < PW; ++c) {
                d[c] += bias[c];
                if (p.a.softplus) d[c] = softplus_of(d[c], e);
                if (has_z) g[c] *= z[c] * sigmoid_of(z[c]);
                if (t >= dead) d[c] = g[c] = x[c] = 0.f;
                if (!Maps) x[c] *= d[c];
            }
            *reinterpret_cast<float4*>(&s_d[tok][cg]) = make_float4(d[0], d[1], d[2], d[3]);
            *reinterpret_cast<float4*>(&s_g[tok][cg]) = make_float4(g[0], g[1], g[2], g[3]);
            if (!Maps) *reinterpret_cast<float4*>(&s_u[tok][cg]) = make_float4(x[0], x[1], x[2], x[3]);
        }
        bc.put(&s_B[0][0], &s_C[0][0]);
        if (tb > t0) request(tb - TB);
        __syncthreads();

        // sequences that start in this tile, and whether one ends there
        unsigned starts = 0;
        for (int i = s; i >= 0; --i) {
            const int o = q.off(i);
            if (o < tb) break;
            if (o < tb + TB) starts |= 1u << (o - tb);
        }
        const bool edge = starts != 0 || q.off(s + 1) <= tb + TB;

        f2 before[TB][CT][2];                                    // the state that token j's decay multiplies
        if (!Maps) {
#pragma unroll
            for (int j = 0; j < TB; ++j) {
                if (starts >> j & 1) {
                    const int first = q.ends_behind(tb + j);
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        h[c][0] = h[c][1] = 0;
                        if (first < q.n && p.a.h0 && w.c0 + c < w.count)
                            ld_state(p.a.h0 + state_at(first, c), n0, N, p.vec_state, h[c]);
                    }
                }
                float d[CT], u[CT], y[CT];
                f2 B[2], C[2];
                ld_channels<CT>(&s_d[j][w.c0], d);
                ld_channels<CT>(&s_u[j][w.c0], u);
                ld_quad(&s_B[j][n0], B);
                ld_quad(&s_C[j][n0], C);
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const f2 d2 = f2_dup(d[c]), u2 = f2_dup(u[c]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        before[j][c][i] = h[c][i];
                        h[c][i] = f2_fma(ex2_pair(f2_mul(d2, A[c][i])), h[c][i], f2_mul(u2, B[i]));
                    }
                    y[c] = f2_sum(f2_fma(C[1], h[c][1], f2_mul(C[0], h[c][0])));
                }
                if (has_z) {                                     // the gate's gradient needs y before the gate
                    scatter_sum<CT, NL>(y, w.lane, 1);
                    const int at = w.c0 + scatter_at<CT, NL>(w.lane, 1);
#pragma unroll
                    for (int i = 0; i < (CT > NL ? CT / NL : 1); ++i) s_y[j][at + i] = y[i];
                }
            }
        }
#pragma unroll
        for (int j = TB - 1; j >= 0; --j) {
            const int t = tb + j;
            if (edge && q.off(s + 1) == t + 1) from_end(s, carry);
            float d[CT], g[CT];
            f2 C[2];
            ld_channels<CT>(&s_d[j][w.c0], d);
            ld_channels<CT>(&s_g[j][w.c0], g);
            ld_quad(&s_C[j][n0], C);
            if constexpr (Maps) {
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const f2 d2 = f2_dup(d[c]), g2 = f2_dup(g[c]);
                    sum_d[c] += d[c];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        carry[c][i] = f2_mul(ex2_pair(f2_mul(d2, A[c][i])), f2_fma(g2, C[i], carry[c][i]));
                }
            } else {
                float u[CT], dot[CT], dec[CT];
                f2 B[2], dB[2] = {0, 0}, dC[2] = {0, 0};
                ld_channels<CT>(&s_u[j][w.c0], u);
                ld_quad(&s_B[j][n0], B);
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const f2 d2 = f2_dup(d[c]), u2 = f2_dup(u[c]), g2 = f2_dup(g[c]);
                    f2 sum_b = 0, sum_a = 0;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const f2 a = ex2_pair(f2_mul(d2, A[c][i]));
                        const f2 ah = f2_mul(a, before[j][c][i]);
                        const f2 dh = f2_fma(g2, C[i], carry[c][i]);
                        dC[i] = f2_fma(g2, f2_fma(u2, B[i], ah), dC[i]);
                        dB[i] = f2_fma(u2, dh, dB[i]);
                        const f2 q2 = f2_mul(dh, ah);
                        sum_b = f2_fma(dh, B[i], sum_b);
                        sum_a = f2_fma(q2, A[c][i], sum_a);
                        dA[c][i] = f2_fma(q2, d2, dA[c][i]);
                        carry[c][i] = f2_mul(a, dh);
                    }
                    dot[c] = f2_sum(sum_b);
                    dec[c] = f2_sum(sum_a);
                }
                scatter_sum<CT, NL>(dot, w.lane, 1);
                scatter_sum<CT, NL>(dec, w.lane, 1);
                const int at = w.c0 + scatter_at<CT, NL>(w.lane, 1);
#pragma unroll
                for (int i = 0; i < (CT > NL ? CT / NL : 1); ++i) {
                    s_dot[j][at + i] = dot[i];
                    s_dec[j][at + i] = dec[i];
                }
                // over the warp's channels: values 0..3 are this lane's states of dB, 4..7 of dC
                float v[8];
                f2_unpack(dB[0], v[0], v[1]); f2_unpack(dB[1], v[2], v[3]);
                f2_unpack(dC[0], v[4], v[5]); f2_unpack(dC[1], v[6], v[7]);
                scatter_sum<8, LC>(v, w.lane, NL);
                const int first = scatter_at<8, LC>(w.lane, NL);
#pragma unroll
                for (int i = 0; i < (LC < 8 ? 8 / LC : 1); ++i) {
                    const int m = first + i;
                    red[w.warp][j][(m >> 2) * NP + n0 + (m & 3)] = v[i];
                }
            }
            if (edge) {
                while (s >= 0 && q.off(s) >= t) {                // token t is a sequence's first (and empty ones precede it)
                    if (q.off(s + 1) > t) store_dh0(s, carry);
                    else empty(s);
                    --s;
                }
                if (s < 0) s = 0;                                // (only at token 0)
            }
        }
        __syncthreads();
        if constexpr (!Maps) {
            for (int i = threadIdx.x; i < TB * 2 * NP; i += kThreads) {
                const int tok = i / (2 * NP), m = i % (2 * NP);
                float v = 0.f;
#pragma unroll
                for (int j = 0; j < kWarps; ++j) v += red[j][tok][m];
                if (tb + tok < t1)
                    p.part_bc[((((size_t)w.tile * p.a.B + w.b) * T + tb + tok) * p.a.G + w.group) * (2 * NP) + m] = v;
            }
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int item = threadIdx.x + i * kThreads, tok = item / Groups, t = tb + tok;
                if (item >= Items || t >= t1) continue;
                float x[PW], d[PW], z[PW], dy[PW], dot[PW], dec[PW], y[PW], dx[PW], dz[PW];
                unpack<DT, PW>(cx[i], x);
                unpack<DT, PW>(cd[i], d);
                unpack<DT, PW>(cy[i], dy);
                if (has_z) unpack<DT, PW>(cz[i], z);
                ld_channels<4>(&s_dot[tok][cg], dot);
                ld_channels<4>(&s_dec[tok][cg], dec);
                ld_channels<4>(&s_y[tok][cg], y);
#pragma unroll
                for (int c = 0; c < PW; ++c) {
                    const float v = d[c] + bias[c];
                    float e, dt = v, slope = 1.f;
                    if (p.a.softplus) {
                        dt = softplus_of(v, e);
                        slope = __fdividef(v >= 0.f ? 1.f : e, 1.f + e);
                    }
                    float g = dy[c];
                    if (has_z) {
                        const float sg = sigmoid_of(z[c]);
                        g *= z[c] * sg;
                        dz[c] = dy[c] * fmaf(skip[c], x[c], y[c]) * sg * (1.f + z[c] * (1.f - sg));
                    }
                    dx[c] = fmaf(dt, dot[c], skip[c] * g);
                    d[c] = fmaf(x[c], dot[c], dec[c] * kLn2) * slope;      // (A is held times log2 e)
                    if (t >= dead) dx[c] = d[c] = dz[c] = g = 0.f;
                    dskip[c] = fmaf(g, x[c], dskip[c]);
                    dbias[c] += d[c];
                }
                const long long at = ((long long)w.b * T + t) * D + dch;
                st_pack<DT, PW, Vec>(p.a.dx, at, valid, dx);
                st_pack<DT, PW, Vec>(p.a.ddt, at, valid, d);
                if (has_z) st_pack<DT, PW, Vec>(p.a.dz, at, valid, dz);
            }
        }
    }
    const size_t row = (size_t)w.b * p.n_seg + w.k;
#pragma unroll
    for (int c = 0; c < CT; ++c)
        if (w.c0 + c < w.count) {
            const size_t at = row * D + w.d0 + w.c0 + c;
            if (Maps) {
                st_quad(p.map_h + at * NP + n0, carry[c]);
                if (w.nl == 0) p.map_d[at] = sum_d[c];
            } else {
                st_quad(p.part_a + at * NP + n0, dA[c]);
            }
        }
    if constexpr (!Maps) {                                       // dskip and dbias: over the threads of a group of channels
        float* r = &red[0][0][0];
#pragma unroll
        for (int what = 0; what < 2; ++what) {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < PW; ++c) r[threadIdx.x * PW + c] = what ? dbias[c] : dskip[c];
            __syncthreads();
            for (int c = threadIdx.x; c < w.count; c += kThreads) {
                float v = 0.f;
                for (int i = c / PW; i < kThreads; i += Groups) v += r[i * PW + c % PW];
                p.part_v[(row * 2 + what) * D + w.d0 + c] = v;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------ single tokens
// NL lanes a channel, four states a lane; a thread has the same channel in Rows sequences, so that A is read once and the
// states' loads of Rows sequences are in flight together.  Bound by HBM: the fp32 state is read and written once.
template <int DT, int NL, int Rows>
__global__ void __launch_bounds__(128) scan_step_kernel(const __grid_constant__ ScanP p) {
    const int D = p.a.D, N = p.a.N, nl = threadIdx.x % NL, n0 = 4 * nl;
    const int blocks = (D + 128 / NL - 1) / (128 / NL);
    const int d = blockIdx.x % blocks * (128 / NL) + threadIdx.x / NL, dd = min(d, D - 1), group = dd / p.Dg;
    const long long b0 = (long long)(blockIdx.x / blocks) * Rows;
    f2 A[2], h[Rows][2];
#pragma unroll
    for (int r = 0; r < Rows; ++r)
        if (b0 + r < p.a.B) ld_state(p.a.h0 + ((size_t)(b0 + r) * D + dd) * N, n0, N, p.vec_state, h[r]);
    ld_state(p.a.A + (size_t)dd * N, n0, N, p.vec_state, A);
    const float bias = p.a.dt_bias ? p.a.dt_bias[dd] : 0.f, skip = p.a.skip ? p.a.skip[dd] : 0.f;
    A[0] = f2_mul(A[0], f2_dup(kLog2e));
    A[1] = f2_mul(A[1], f2_dup(kLog2e));
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        const long long b = b0 + r;
        if (b >= p.a.B) break;
        float f[4], e;
        f2 B[2], C[2];
        const long long ba = b * p.a.B_batch + group * p.a.B_group + n0, ca = b * p.a.C_batch + group * p.a.C_group + n0;
        const int valid = min(4, N - n0);
        unpack<DT, 4>(p.vec_bc ? ld_pack<DT, 4, true>(p.a.Bm, ba, valid) : ld_pack<DT, 4, false>(p.a.Bm, ba, valid), f);
        B[0] = f2_pack(f[0], f[1]); B[1] = f2_pack(f[2], f[3]);
        unpack<DT, 4>(p.vec_bc ? ld_pack<DT, 4, true>(p.a.Cm, ca, valid) : ld_pack<DT, 4, false>(p.a.Cm, ca, valid), f);
        C[0] = f2_pack(f[0], f[1]); C[1] = f2_pack(f[2], f[3]);
        const float x = ld_elem(p.a.x, b * p.a.x_batch + dd, DT);
        float dt = ld_elem(p.a.dt, b * p.a.dt_batch + dd, DT) + bias;
        if (p.a.softplus) dt = softplus_of(dt, e);
        const f2 d2 = f2_dup(dt), u2 = f2_dup(dt * x);
#pragma unroll
        for (int i = 0; i < 2; ++i) h[r][i] = f2_fma(ex2_pair(f2_mul(d2, A[i])), h[r][i], f2_mul(u2, B[i]));
        float y = f2_sum(f2_fma(C[1], h[r][1], f2_mul(C[0], h[r][0])));
#pragma unroll
        for (int m = 1; m < NL; m <<= 1) y += __shfl_xor_sync(0xffffffffu, y, m);
        y = fmaf(skip, x, y);
        if (d >= D) continue;
        st_state(p.a.ht + ((size_t)b * D + d) * N, n0, N, p.vec_state, h[r]);
        if (nl == 0) {
            if (p.a.z) {
                const float z = ld_elem(p.a.z, b * p.a.z_batch + d, DT);
                y *= z * sigmoid_of(z);
            }
            st_elem(p.a.y, b * D + d, DT, y);
        }
    }
}

// ------------------------------------------------------------------------------------------ launches
int lanes_of(int N) {                    // lanes that share a channel's states, four each
    int nl = 2;
    while (4 * nl < N) nl *= 2;
    return nl;
}
constexpr int kBwdCT = 2;

// Segments: enough blocks for kBusy an SM, which is what it takes to hide the latencies here; never shorter than 64 tokens.
// The maps cost the recurrence once more, so a row is cut only where its blocks would leave more than half of that empty.
constexpr int kBusy = 4;
struct Plan { int ct, ch, tiles, seg, n_seg; };
Plan plan_of(const HdlaScanArgs& a, bool backward) {
    const int nl = lanes_of(a.N), dg = a.D / a.G;
    Plan r{};
    r.ct = backward ? kBwdCT : 4;
    const long long want = (long long)kBusy * sm_count();
    auto blocks = [&](int ct) {
        r.ch = kWarps * (32 / nl) * ct;
        r.tiles = (dg + r.ch - 1) / r.ch;
        return (long long)a.B * a.G * r.tiles;
    };
    long long n = blocks(r.ct);
    if (!backward && n < want) { r.ct = 2; n = blocks(r.ct); }
    long long cut = 2 * n > want ? 1 : (want + n - 1) / n;
    const long long most = (a.T + 63) / 64;
    if (cut > most) cut = most;
    r.seg = static_cast<int>(((a.T + cut - 1) / cut + 15) / 16 * 16);
    r.n_seg = (a.T + r.seg - 1) / r.seg;
    return r;
}
struct Work { size_t map_h, map_d, bc, a, v, total; };
Work work_of(const HdlaScanArgs& a, const Plan& r, bool backward) {
    const size_t np = 4 * (size_t)lanes_of(a.N), rows = (size_t)a.B * r.n_seg, D = a.D;
    Work w{};
    auto take = [&](size_t floats) { const size_t at = w.total; w.total += up256(floats * sizeof(float)); return at; };
    if (r.n_seg > 1) { w.map_h = take(rows * D * np); w.map_d = take(rows * D); }
    if (backward) {
        w.bc = take((size_t)r.tiles * a.B * a.T * a.G * 2 * np);
        w.a = take(rows * D * np);
        w.v = take(rows * 2 * D);
    }
    return w;
}
bool scan_vec(const HdlaScanArgs& a) {
    const int per = a.dtype == HDLA_F32 ? 4 : 8;                 // elements of 16 bytes
    for (int64_t st : {a.x_batch, a.x_token, a.dt_batch, a.dt_token})
        if (st % per) return false;
    if (a.z && (a.z_batch % per || a.z_token % per)) return false;
    for (const void* q : {a.x, a.dt, a.z, (const void*)a.y, a.dy, (const void*)a.dx, (const void*)a.ddt, (const void*)a.dz})
        if (!aligned16(q)) return false;
    return a.D % per == 0 && (a.D / a.G) % per == 0;
}
ScanP params_of(const HdlaScanArgs& a, const Plan& r) {
    ScanP p{};
    p.a = a;
    p.Dg = a.D / a.G;
    p.tiles = r.tiles; p.seg = r.seg; p.n_seg = r.n_seg;
    const int bytes = a.dtype == HDLA_F32 ? 16 : 8;
    p.vec_bc = a.N % 4 == 0 && reinterpret_cast<uintptr_t>(a.Bm) % bytes == 0 && reinterpret_cast<uintptr_t>(a.Cm) % bytes == 0;
    for (int64_t st : {a.B_batch, a.B_token, a.B_group, a.C_batch, a.C_token, a.C_group}) p.vec_bc = p.vec_bc && st % 4 == 0;
    p.vec_state = a.N % 4 == 0;
    for (const void* q : {(const void*)a.A, (const void*)a.h0, (const void*)a.ht, (const void*)a.dht, (const void*)a.dh0})
        p.vec_state = p.vec_state && aligned16(q);
    return p;
}

template <typename F>
void with_lanes(int nl, F f) {
    if (nl == 2) f(std::integral_constant<int, 2>());
    else if (nl == 4) f(std::integral_constant<int, 4>());
    else if (nl == 8) f(std::integral_constant<int, 8>());
    else if (nl == 16) f(std::integral_constant<int, 16>());
    else f(std::integral_constant<int, 32>());
}
template <typename F>
void with_type(int dtype, bool vec, F f) {
    using F32 = std::integral_constant<int, HDLA_F32>;
    using BF16 = std::integral_constant<int, HDLA_BF16>;
    if (dtype == HDLA_F32) vec ? f(F32(), std::true_type()) : f(F32(), std::false_type());
    else vec ? f(BF16(), std::true_type()) : f(BF16(), std::false_type());
}
int check_grid(long long blocks) {
    return blocks > 0x7fffffffLL ? fail(HDLA_ERR_UNSUPPORTED, "selective_scan: %lld blocks", blocks) : HDLA_OK;
}

}  // namespace

size_t selective_scan_checkpoint_bytes(const HdlaScanArgs& a) {
    return (size_t)a.B * ((a.T + kCheckpoint - 1) / kCheckpoint) * a.D * 4 * lanes_of(a.N) * sizeof(float);
}
size_t selective_scan_workspace(const HdlaScanArgs& a, bool backward) { return work_of(a, plan_of(a, backward), backward).total; }

int selective_scan_fwd(const HdlaScanArgs& a, unsigned char* ws, cudaStream_t st) {
    const Plan r = plan_of(a, false);
    const Work at = work_of(a, r, false);
    ScanP p = params_of(a, r);
    p.map_h = reinterpret_cast<float*>(ws + at.map_h);
    p.map_d = reinterpret_cast<float*>(ws + at.map_d);
    const long long blocks = (long long)a.G * r.tiles * a.B;
    if (int rc = check_grid(blocks * r.n_seg)) return rc;
    for (int maps = r.n_seg > 1 ? 1 : 0; maps >= 0; --maps) {
        const unsigned grid = static_cast<unsigned>(blocks * (r.n_seg - maps));
        with_type(a.dtype, scan_vec(a), [&](auto dt, auto vec) {
            with_lanes(lanes_of(a.N), [&](auto nl) {
                if (maps) r.ct == 4 ? scan_fwd_kernel<dt, vec, nl, 4, true><<<grid, kThreads, 0, st>>>(p)
                                    : scan_fwd_kernel<dt, vec, nl, 2, true><<<grid, kThreads, 0, st>>>(p);
                else r.ct == 4 ? scan_fwd_kernel<dt, vec, nl, 4, false><<<grid, kThreads, 0, st>>>(p)
                               : scan_fwd_kernel<dt, vec, nl, 2, false><<<grid, kThreads, 0, st>>>(p);
            });
        });
        HDLA_CHECK_LAUNCH(maps ? "scan_fwd_maps_kernel" : "scan_fwd_kernel");
    }
    return HDLA_OK;
}

int selective_scan_bwd(const HdlaScanArgs& a, unsigned char* ws, cudaStream_t st) {
    const Plan r = plan_of(a, true);
    const Work at = work_of(a, r, true);
    ScanP p = params_of(a, r);
    p.map_h = reinterpret_cast<float*>(ws + at.map_h);
    p.map_d = reinterpret_cast<float*>(ws + at.map_d);
    p.part_bc = reinterpret_cast<float*>(ws + at.bc);
    p.part_a = reinterpret_cast<float*>(ws + at.a);
    p.part_v = reinterpret_cast<float*>(ws + at.v);
    const long long blocks = (long long)a.G * r.tiles * a.B;
    if (int rc = check_grid(blocks * r.n_seg)) return rc;
    for (int maps = r.n_seg > 1 ? 1 : 0; maps >= 0; --maps) {
        const unsigned grid = static_cast<unsigned>(blocks * (r.n_seg - maps));
        with_type(a.dtype, scan_vec(a), [&](auto dt, auto vec) {
            with_lanes(lanes_of(a.N), [&](auto nl) {
                if (maps) scan_bwd_kernel<dt, vec, nl, kBwdCT, true><<<grid, kThreads, 0, st>>>(p);
                else scan_bwd_kernel<dt, vec, nl, kBwdCT, false><<<grid, kThreads, 0, st>>>(p);
            });
        });
        HDLA_CHECK_LAUNCH(maps ? "scan_bwd_maps_kernel" : "scan_bwd_kernel");
    }
    const int np = 4 * lanes_of(a.N), rows = a.B * r.n_seg;
    ColJobs js{};
    js.j[js.n++] = ColJob{p.part_bc, {a.dB, a.dC, nullptr}, (long long)a.B * a.T * a.G * 2 * np, r.tiles, 2, np, a.N, a.dtype, 0, 0, 0};
    js.j[js.n++] = ColJob{p.part_a, {a.dA, nullptr, nullptr}, (long long)a.D * np, rows, 1, np, a.N, HDLA_F32, 0, 0, 0};
    if (a.dskip || a.ddt_bias)
        js.j[js.n++] = ColJob{p.part_v, {a.dskip, a.ddt_bias, nullptr}, 2LL * a.D, rows, 2, a.D, a.D, HDLA_F32, 0, 0, 0};
    return column_sum_launch(js, st);
}

int selective_scan_step(const HdlaScanArgs& a, cudaStream_t st) {
    Plan r{};
    r.tiles = 1; r.n_seg = 1;
    const ScanP p = params_of(a, r);
    const int nl = lanes_of(a.N);
    const long long columns = (a.D + 128 / nl - 1) / (128 / nl);
    const bool many = columns * ((a.B + 3) / 4) >= 8LL * sm_count();       // four sequences a thread where enough blocks are left
    const long long grid = columns * (many ? (a.B + 3) / 4 : a.B);
    if (int rc = check_grid(grid)) return rc;
    with_lanes(nl, [&](auto l) {
        using F32 = std::integral_constant<int, HDLA_F32>;
        using BF16 = std::integral_constant<int, HDLA_BF16>;
        auto go = [&](auto dt) {
            if (many) scan_step_kernel<dt, l, 4><<<(unsigned)grid, 128, 0, st>>>(p);
            else scan_step_kernel<dt, l, 1><<<(unsigned)grid, 128, 0, st>>>(p);
        };
        a.dtype == HDLA_F32 ? go(F32()) : go(BF16());
    });
    HDLA_CHECK_LAUNCH("scan_step_kernel");
    return HDLA_OK;
}

}  // namespace hdla
