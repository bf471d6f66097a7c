// Shared by the short convolution, the selective scan and the norms round a block: packed sequences, groups of channels
// moved as one access, activations, and sums over partial rows in a fixed order.
#pragma once
#include "common.cuh"
#include "f32x2.cuh"

namespace hdla {
namespace {

// ------------------------------------------------------------------------------------------ sequences
// The sequences along one row of T tokens: the whole row, or those of a packed batch.  Offsets are cut to 0..T where they
// are read, so that no offset makes a kernel leave its tensors.
struct Seqs {
    const int64_t* cu;
    int n, T;
    __device__ __forceinline__ int off(int i) const {
        if (i == 0) return 0;
        if (!cu) return T;
        const long long c = __ldg(reinterpret_cast<const long long*>(cu) + i);
        return static_cast<int>(c < 0 ? 0 : c > T ? T : c);
    }
    __device__ __forceinline__ int end() const { return off(n); }          // rows from here on belong to no sequence
    // the first sequence that ends behind token t, or n
    __device__ __forceinline__ int ends_behind(int t) const {
        int lo = 0, hi = n;
        while (lo < hi) {
            const int m = (lo + hi) >> 1;
            if (off(m + 1) > t) hi = m; else lo = m + 1;
        }
        return lo;
    }
    // the last sequence that starts before token t (t > 0)
    __device__ __forceinline__ int starts_before(int t) const {
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            const int m = (lo + hi + 1) >> 1;
            if (off(m) < t) lo = m; else hi = m - 1;
        }
        return lo;
    }
};

// ------------------------------------------------------------------------------------------ channels
// PW neighbouring channels of a row.  Vec: one access of PW elements (the address is a multiple of its size and all
// channels exist); otherwise element by element, `valid` of them.
template <int DT, int PW>
struct Pack { uint32_t w[PW * (DT == HDLA_F32 ? 4 : 2) / 4]; };

// Once: what is read for the only time is marked as such for the caches.
template <int N, bool Once>
__device__ __forceinline__ void ld_words(uint32_t* w, const void* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4* at = reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(p) + i);
            const uint4 v = Once ? __ldcs(at) : *at;
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const uint2 v = Once ? __ldcs(static_cast<const uint2*>(p)) : *static_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
        w[0] = *static_cast<const uint32_t*>(p);
    }
}
template <int N>
__device__ __forceinline__ void st_words(void* p, const uint32_t* w) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            *reinterpret_cast<uint4*>(static_cast<uint32_t*>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    } else if constexpr (N == 2) {
        *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
        *static_cast<uint32_t*>(p) = w[0];
    }
}
template <int DT>
__device__ __forceinline__ const char* elem_ptr(const void* base, long long i) {
    return static_cast<const char*>(base) + i * (DT == HDLA_F32 ? 4 : 2);
}

template <int DT, int PW, bool Vec, bool Once = false>
__device__ __forceinline__ Pack<DT, PW> ld_pack(const void* base, long long i, int valid) {
    Pack<DT, PW> r;
    constexpr int NW = sizeof(r.w) / 4;
    if constexpr (Vec) {
        if (valid > 0) ld_words<NW, Once>(r.w, elem_ptr<DT>(base, i));
        else
#pragma unroll
            for (int j = 0; j < NW; ++j) r.w[j] = 0;
    } else if constexpr (DT == HDLA_F32) {
#pragma unroll
        for (int j = 0; j < PW; ++j) r.w[j] = j < valid ? static_cast<const uint32_t*>(base)[i + j] : 0u;
    } else {
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            const uint32_t lo = 2 * j < valid ? static_cast<const uint16_t*>(base)[i + 2 * j] : 0u;
            const uint32_t hi = 2 * j + 1 < valid ? static_cast<const uint16_t*>(base)[i + 2 * j + 1] : 0u;
            r.w[j] = lo | hi << 16;
        }
    }
    return r;
}
template <int DT, int PW>
__device__ __forceinline__ void unpack(const Pack<DT, PW>& r, float* f) {
    if constexpr (DT == HDLA_F32) {
#pragma unroll
        for (int j = 0; j < PW; ++j) f[j] = __uint_as_float(r.w[j]);
    } else {
#pragma unroll
        for (int j = 0; j < PW / 2; ++j) {
            f[2 * j] = __uint_as_float(r.w[j] << 16);
            f[2 * j + 1] = __uint_as_float(r.w[j] & 0xffff0000u);
        }
    }
}
// The one rounding of an output to its type.
template <int DT, int PW, bool Vec>
__device__ __forceinline__ void st_pack(void* base, long long i, int valid, const float* f) {
    if constexpr (Vec) {
        if (valid <= 0) return;
        Pack<DT, PW> r;
        if constexpr (DT == HDLA_F32) {
#pragma unroll
            for (int j = 0; j < PW; ++j) r.w[j] = __float_as_uint(f[j]);
        } else {
#pragma unroll
            for (int j = 0; j < PW / 2; ++j) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                r.w[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        st_words<sizeof(r.w) / 4>(const_cast<char*>(elem_ptr<DT>(base, i)), r.w);
    } else {
#pragma unroll
        for (int j = 0; j < PW; ++j)
            if (j < valid) st_elem(base, i + j, DT, f[j]);
    }
}

// ------------------------------------------------------------------------------------------ activations
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float rcp(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ f2 ex2_pair(f2 x) {
    float a, b;
    f2_unpack(x, a, b);
    return f2_pack(ex2(a), ex2(b));
}
__device__ __forceinline__ float sigmoid_of(float v) { return rcp(1.f + ex2(-kLog2e * v)); }           // (e^-v = inf: 0)
__device__ __forceinline__ f2 sigmoid_pair(f2 v) {
    float a, b;
    f2_unpack(f2_add(ex2_pair(f2_mul(v, f2_dup(-kLog2e))), f2_dup(1.f)), a, b);
    return f2_pack(rcp(a), rcp(b));
}
// ------------------------------------------------------------------------------------------ sums over partial rows
// out[c] = sum over P rows of part[row, c], by 8 or 32 threads each with every 8th or 32nd row, whose sums are added at the end: an order that depends on the sizes alone.
// Column c = (r * K + k) * NP + n goes to out[k][r * N + n] where n < N; with `turned` column n * K + k of a [NP, K] matrix
// (r = 0), as the convolution's taps are laid out.
struct ColJob {
    const float* part;
    void* out[3];
    long long C;
    int P, K, NP, N, dt, turned, per_lane;
    unsigned first_block;
};
struct ColJobs { ColJob j[3]; int n; };

__device__ __forceinline__ void col_store(const ColJob& j, long long c, float v) {
    const long long rk = c / j.NP;
    const int n = static_cast<int>(c - rk * j.NP), k = static_cast<int>(rk % j.K);
    if (n >= j.N) return;
    if (j.turned) {                                   // rows 0..K-2 are the taps, row K-1 the bias
        if (k < j.K - 1) st_elem(j.out[0], (size_t)n * (j.K - 1) + k, j.dt, v);
        else if (j.out[1]) st_elem(j.out[1], n, j.dt, v);
        return;
    }
    void* out = k == 0 ? j.out[0] : k == 1 ? j.out[1] : j.out[2];
    if (out) st_elem(out, (rk / j.K) * j.N + n, j.dt, v);
}

template <int kColRows>
__global__ void __launch_bounds__(32 * kColRows) column_sum_kernel(ColJobs js) {
    __shared__ float red[kColRows][4][32];
    int which = 0;
    while (which + 1 < js.n && blockIdx.x >= js.j[which + 1].first_block) ++which;
    const ColJob& j = js.j[which];
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const long long c0 = (long long)(blockIdx.x - j.first_block) * 32 * j.per_lane + lane;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const bool whole = j.per_lane == 4 && c0 - lane + 128 <= j.C;
    if (whole) {
#pragma unroll 4
        for (int p = row; p < j.P; p += kColRows) {
            const float* at = j.part + (long long)p * j.C + c0;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += at[32 * i];
        }
    } else {
#pragma unroll 8
        for (int p = row; p < j.P; p += kColRows) {
            const float* at = j.part + (long long)p * j.C + c0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < j.per_lane && c0 + 32 * i < j.C) s[i] += at[32 * i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) red[row][i][lane] = s[i];
    __syncthreads();
    if (row < j.per_lane) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < kColRows; ++r) t += red[r][row][lane];
        const long long c = c0 + 32 * row;
        if (c < j.C) col_store(j, c, t);
    }
}

// Wide jobs (enough columns to fill the GPU at four a lane) take four a lane and eight rows at once; where all are narrow, 32 rows
// at once keep more loads in flight (1 M columns of 32 rows: 39 us, with 16 rows at once 53 us; 6144 columns of 296 rows: with
// 8 rows at once 16 us, with 16 12 us).
inline int column_sum_launch(ColJobs& js, cudaStream_t st) {
    long long at = 0;
    bool wide = false;
    for (int i = 0; i < js.n; ++i) {
        ColJob& j = js.j[i];
        j.first_block = static_cast<unsigned>(at);
        j.per_lane = j.C >= 128LL * 4 * sm_count() ? 4 : 1;
        wide = wide || j.per_lane == 4;
        at += (j.C + 32 * j.per_lane - 1) / (32 * j.per_lane);
    }
    if (at > 0x7fffffffLL) return fail(HDLA_ERR_UNSUPPORTED, "column sums: %lld blocks", at);
    if (wide) column_sum_kernel<8><<<static_cast<unsigned>(at), 32 * 8, 0, st>>>(js);
    else column_sum_kernel<32><<<static_cast<unsigned>(at), 32 * 32, 0, st>>>(js);
    HDLA_CHECK_LAUNCH("column_sum_kernel");
    return HDLA_OK;
}

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace hdla
