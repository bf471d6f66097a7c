// Selective state space scan: what its kernels share (selective_scan.cu forward and single tokens, selective_scan_bwd.cu).
// Per channel c with N states, c's group sharing B and C:
//     d_t = softplus(dt_t + bias) (or dt_t + bias),  h_t[n] = exp(d_t A[n]) h_{t-1}[n] + d_t x_t B_t[n]
//     y_t = (sum_n C_t[n] h_t[n] + skip x_t) silu(z_t)
//
// Layout of the work.  A warp holds the states of (32 / NL) * CT channels in registers: NL lanes share a channel's states,
// four a lane, and a lane has CT channels, so that one 16-byte read of B (and C) serves 4 * CT states.  Four warps make a
// block; it walks over its tokens in tiles, in three steps: what is done once per (token, channel) -- softplus, d x, gates --
// by all threads on pieces of four channels into shared memory; the recurrence; the outputs.  Sums over n are left in shared
// memory as NL partial sums, which the threads of the third step add: fewer instructions than shuffles and selects.  The next
// tile's inputs are requested before the recurrence of this one (backward: brought to L2).  All arithmetic is fp32, the
// outputs are rounded once.
//
// Long rows of few channels are cut into segments.  What a segment does to a state is exp(A sum d) h + F, and its sum of d
// and F come from a first kernel that runs the recurrence alone, from zero; the second kernel's blocks chain the maps of
// the segments before theirs.
#pragma once
#include "lane_sums.cuh"
#include "ssm.cuh"

namespace hdla {

constexpr int kScanWarps = 4, kScanThreads = 32 * kScanWarps;
constexpr int kCheckpoint = 8;                     // tokens between two saved states

struct ScanP {
    HdlaScanArgs a;
    int Dg, tiles;             // channels of a group, tiles of channels per group
    int first_tile, tile_count;      // those of this launch
    int seg, n_seg;            // tokens of a segment (a multiple of 16), segments
    bool vec_state;            // 4 of a channel's states as one access
    float *map_h, *map_d;      // [B][n_seg][D][NP], [B][n_seg][D]
    float *part_bc, *part_a, *part_v;      // [tiles][B][T][G][2][NP], [B * n_seg][D][NP], [B * n_seg][2][D]
};

struct ScanPlan { int ct, tiles, seg, n_seg; };
struct ScanWork { size_t map_h, map_d, bc, a, v, total; };
int scan_lanes(int N);                             // lanes that share a channel's states, four each
ScanPlan scan_plan(const HdlaScanArgs& a, bool backward);
ScanWork scan_work(const HdlaScanArgs& a, const ScanPlan& r, bool backward);
ScanP scan_params(const HdlaScanArgs& a, const ScanPlan& r, const ScanWork& at, unsigned char* ws);
int scan_slots(const HdlaScanArgs& a, const ScanPlan& r);
bool scan_vec(const HdlaScanArgs& a);              // four channels, and four states of B and C, as one access

namespace {

// log(1 + e^v) = max(v, 0) + log1p(e), e = e^-|v| in (0, 1]; log1p(e) = 2 artanh(s) with s = e / (2 + e) <= 1/3, and artanh(s)
// = s p(s^2), p the polynomial of degree 4 through the Chebyshev nodes of [0, 1/9], 4e-9 off at most.  (A logarithm of 1 + e
// would lose the small time steps, which are e itself.)
__device__ __forceinline__ f2 softplus_pair(f2 v) {
    float a, b, c, d;
    f2_unpack(v, a, b);
    const f2 e = f2_pack(ex2(-fabsf(a) * kLog2e), ex2(-fabsf(b) * kLog2e));
    f2_unpack(f2_add(e, f2_dup(2.f)), c, d);
    const f2 s = f2_mul(e, f2_pack(rcp(c), rcp(d))), q = f2_mul(s, s);
    f2 p = f2_fma(q, f2_dup(0.14078889787197113f), f2_dup(0.13982579112052917f));
    p = f2_fma(p, q, f2_dup(0.20012298226356506f));
    p = f2_fma(p, q, f2_dup(0.3333316147327423f));
    p = f2_fma(p, q, f2_dup(1.f));
    return f2_fma(f2_mul(s, p), f2_dup(2.f), f2_pack(fmaxf(a, 0.f), fmaxf(b, 0.f)));
}

// four neighbouring channels as two pairs
template <int DT>
__device__ __forceinline__ void unpack_pairs(const Pack<DT, 4>& r, f2 (&v)[2]) {
    float f[4];
    unpack<DT, 4>(r, f);
    v[0] = f2_pack(f[0], f[1]);
    v[1] = f2_pack(f[2], f[3]);
}
__device__ __forceinline__ void unpair(const f2 (&v)[2], float (&f)[4]) {
    f2_unpack(v[0], f[0], f[1]);
    f2_unpack(v[1], f[2], f[3]);
}
__device__ __forceinline__ void st_pairs(float* at, const f2 (&v)[2]) { *reinterpret_cast<ulonglong2*>(at) = make_ulonglong2(v[0], v[1]); }
// a lane's channels, each as a pair of itself (copied here: stored as pairs they would cost twice the shared-memory cycles,
// which are scarcer than instructions)
template <int CT>
__device__ __forceinline__ void ld_twice(const float* at, f2 (&v)[CT]) {
    if constexpr (CT == 2) {
        const float2 q = *reinterpret_cast<const float2*>(at);
        v[0] = f2_dup(q.x); v[1] = f2_dup(q.y);
    } else {
        v[0] = f2_dup(*at);
    }
}
template <int CT>
__device__ __forceinline__ void st_channels(float* at, const float (&v)[CT]) {
    if constexpr (CT == 2) *reinterpret_cast<float2*>(at) = make_float2(v[0], v[1]);
    else *at = v[0];
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
// ... of states that pass through once (single tokens), marked as such for the caches.  Vec is known at compile time here: where
// two ways of loading meet, the value is waited for, and the loads of several sequences would follow one another.
template <bool Vec>
__device__ __forceinline__ void ld_state_once(const float* at, int n0, int N, f2 (&h)[2]) {
    if constexpr (Vec) {
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (n0 < N) q = __ldcs(reinterpret_cast<const float4*>(at + n0));
        h[0] = f2_pack(q.x, q.y);
        h[1] = f2_pack(q.z, q.w);
    } else {
        ld_state(at, n0, N, false, h);
    }
}
template <bool Vec>
__device__ __forceinline__ void st_state_once(float* at, int n0, int N, const f2 (&h)[2]) {
    if constexpr (Vec) {
        float4 q;
        f2_unpack(h[0], q.x, q.y);
        f2_unpack(h[1], q.z, q.w);
        if (n0 < N) __stcs(reinterpret_cast<float4*>(at + n0), q);
    } else {
        st_state(at, n0, N, false, h);
    }
}
// ... of the library's own arrays, where NP states are laid out
__device__ __forceinline__ void ld_quad(const float* at, f2 (&h)[2]) {
    const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(at);
    h[0] = q.x; h[1] = q.y;
}
__device__ __forceinline__ void st_quad(float* at, const f2 (&h)[2]) { *reinterpret_cast<ulonglong2*>(at) = make_ulonglong2(h[0], h[1]); }

// Which part of the problem a block has, and its lanes their states.
template <int NL, int CT>
struct Tile {
    static constexpr int LC = 32 / NL, NP = 4 * NL, CPW = LC * CT, CH = kScanWarps * CPW;
    // a row of partial sums over n: so many floats that the NL lanes of a channel write to different banks
    static constexpr int Pitch = CH + (NL >= 8 ? 4 : 32 / NL);
    int b, group, tile, k;            // sequence row, group, tile of the group, segment
    int d0, count;                    // first channel of the tile, channels it has
    int lane, warp, nl, c0;           // this lane's first state is 4 * nl, its first channel c0 (in the tile)
    __device__ __forceinline__ explicit Tile(const ScanP& p, int segments) {
        const int per_row = p.a.G * p.tile_count;
        const int x = blockIdx.x % per_row, r = blockIdx.x / per_row;
        group = x / p.tile_count; tile = p.first_tile + x % p.tile_count;
        k = r % segments; b = r / segments;
        d0 = group * p.Dg + tile * CH;
        count = min(CH, p.Dg - tile * CH);
        lane = threadIdx.x & 31; warp = threadIdx.x >> 5;
        nl = lane % NL;
        c0 = warp * CPW + lane / NL * CT;
    }
};

__device__ __forceinline__ void prefetch_l2(const void* at) { asm volatile("prefetch.global.L2 [%0];" ::"l"(at)); }

// A thread's pieces of a [tokens, channels] tensor: where they are in the present tile.  Addresses are moved on from tile to
// tile, not formed anew.
struct Walk {
    const char* at;
    long long token, piece;                    // bytes between tokens, between this thread's pieces
    template <int DT>
    __device__ __forceinline__ static Walk of(const void* base, long long first, long long token, int piece_tokens) {
        constexpr int size = DT == HDLA_F32 ? 4 : 2;
        return Walk{static_cast<const char*>(base) + first * size, token * size, token * size * piece_tokens};
    }
    __device__ __forceinline__ void move(int tokens) { at += tokens * token; }
    template <int DT, bool Vec>
    __device__ __forceinline__ Pack<DT, 4> load(int i, int valid) const { return ld_pack<DT, 4, Vec>(at + i * piece, 0, valid); }
    __device__ __forceinline__ void prefetch(int i, int valid, int tokens) const { if (valid > 0) prefetch_l2(at + i * piece + tokens * token); }
};

// B and C of a tile of tokens: four states a piece, requested early and put into shared memory as fp32.
template <int DT, int NL, int TB>
struct BcTile {
    static constexpr int NP = 4 * NL, Pieces = TB * NL * 2, PerThread = (Pieces + kScanThreads - 1) / kScanThreads;
    static constexpr int Ahead = kScanThreads / (2 * NL);      // tokens between a thread's pieces
    Pack<DT, 4> raw[PerThread];
    Walk from;
    int tok, valid;
    __device__ __forceinline__ BcTile(const ScanP& p, int b, int group, int tb) {
        const int quad = threadIdx.x % NL, which = threadIdx.x / NL % 2;
        tok = threadIdx.x / (2 * NL);
        valid = threadIdx.x < Pieces ? min(4, p.a.N - 4 * quad) : 0;
        from = which ? Walk::of<DT>(p.a.Cm, b * p.a.C_batch + (tb + tok) * p.a.C_token + group * p.a.C_group + 4 * quad, p.a.C_token, Ahead)
                     : Walk::of<DT>(p.a.Bm, b * p.a.B_batch + (tb + tok) * p.a.B_token + group * p.a.B_group + 4 * quad, p.a.B_token, Ahead);
    }
    // of the tile's first `tokens` tokens (zeros behind them)
    template <bool Vec>
    __device__ __forceinline__ void request(int tokens) {
#pragma unroll
        for (int i = 0; i < PerThread; ++i) {
            const int ok = tok + i * Ahead < tokens ? valid : 0;
            raw[i] = from.load<DT, Vec>(i, ok);
        }
    }
    __device__ __forceinline__ void prefetch(int tokens) const {
#pragma unroll
        for (int i = 0; i < PerThread; ++i) from.prefetch(i, valid, tokens);
    }
    __device__ __forceinline__ void put(float* sB, float* sC) const {
        float* to = (threadIdx.x / NL % 2 ? sC : sB) + tok * NP + 4 * (threadIdx.x % NL);
#pragma unroll
        for (int i = 0; i < PerThread; ++i)
            if (threadIdx.x < Pieces) {
                float f[4];
                unpack<DT, 4>(raw[i], f);
                *reinterpret_cast<float4*>(to + i * Ahead * NP) = make_float4(f[0], f[1], f[2], f[3]);
            }
    }
};

// Four channels' sums over n: NL rows of partial sums, `pitch` floats apart.
template <int NL>
__device__ __forceinline__ void add_partial(const float* at, int pitch, f2 (&v)[2]) {
    v[0] = v[1] = 0;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(at + i * pitch);
        v[0] = f2_add(v[0], q.x);
        v[1] = f2_add(v[1], q.y);
    }
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

}  // namespace
}  // namespace hdla
