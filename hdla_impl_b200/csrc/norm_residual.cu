// RMS norms after and before a block, with the block's gate, residual scale and residual sum, per row of D channels:
//     v = x or rms(x) post;   v = v act(gate);   r = residual + scale v;   u = rms(r) pre,   rms(a) = sqrt(D) a / sqrt(sum a^2 + eps)
// forward and backward as one kernel each: every tensor is read or written once, which is what bounds them (HBM).
//
// A thread owns eight neighbouring channels of a row (16-byte accesses of bf16) and holds them, as packed pairs, between the
// sums; a row takes as many whole warps as it needs, narrow rows share a block.  Blocks walk over rows and request the next
// row's tensors before the sums of this one; the weights wait in shared memory, so that two (backward) or four (forward) blocks
// of 256 threads fit on an SM: with them in registers backward had one, and took 686 instead of 319 us for 32768 rows of 2048.
// Backward computes r again from the inputs in fp32 (as many bytes as reading the rounded r), reads the norms' factors that
// forward left (305 -> 276 us when that was done: a sum and a barrier less), takes the two sums that remain (the dot products of
// the norms' gradients), and keeps the sums over rows (gradients of the weights and of scale) in registers until its last row;
// blocks' sums are added in a fixed order.  The row that a dot product belongs to is normed before the two meet: the cube of a
// norm's factor need not be an fp32 number where the gradient is one, as for rows of 1e12 or of 1e-14.  Rows of more than 4096
// channels need 1024 threads of 64 registers: there those sums are in shared memory too, and nothing is requested ahead.
// 32768 rows of 2048, bf16, all parts: forward 139 us = 4.8 TB/s (0.75 of the measured copy), backward 269 us = 4.0 TB/s
// (0.62); what backward waits for is the chain of its two sums.
#include "ssm.cuh"

namespace hdla {
namespace {

constexpr int kPw = 8, kPairs = kPw / 2, kMaxD = 1024 * kPw;

struct NrP {
    HdlaNormResidualArgs a;
    int per_row;             // threads of a row (whole warps)
    int stride;              // floats of a vector in shared memory: kPw * per_row
    float* part;             // backward: [blocks][3][D] (post, pre, scale)
};

// Sums over the warps of a row: over the lanes, then every warp over the warps' sums.  `red` has two buffers, used in turn, so
// that one barrier a sum is enough.
struct RowSum {
    float (*red)[32];
    int turn, first, warps;
    __device__ __forceinline__ float one(float a) {
#pragma unroll
        for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        if (warps == 1) return a;
        float* at = red[turn];
        if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = a;
        __syncthreads();
        const int w = threadIdx.x & (warps > 8 ? 31 : 7);
        a = w < warps ? at[first + w] : 0.f;
        if (warps > 8) {
            a += __shfl_xor_sync(0xffffffffu, a, 16);
            a += __shfl_xor_sync(0xffffffffu, a, 8);
        }
#pragma unroll
        for (int o = 4; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        turn ^= 1;
        return a;
    }
};

// Where a thread stands.  Its eight channels are neighbours where a row can be read in 16-byte pieces (Vec); else they lie
// per_row apart, so that neighbouring threads read neighbouring channels (4096 bf16 rows of 8191 channels, backward: 378 us;
// with neighbours for each thread there too 556 us).
template <bool Vec>
struct Place {
    int rows, group, lane, per_row, D;
    int col, valid;                                             // (Vec)
    __device__ __forceinline__ explicit Place(const NrP& p) : per_row(p.per_row), D(p.a.D) {
        rows = blockDim.x / per_row;
        group = threadIdx.x / per_row;
        lane = threadIdx.x % per_row;
        col = lane * kPw;
        valid = max(0, min(kPw, D - col));
    }
    __device__ __forceinline__ bool any() const { return Vec ? valid > 0 : lane < D; }
    template <int DT>
    __device__ __forceinline__ Pack<DT, kPw> load(const void* base, long long row, bool exists) const {
        if constexpr (Vec) {
            return ld_pack<DT, kPw, true, true>(base, row * D + col, exists ? valid : 0);
        } else {
            Pack<DT, kPw> r = {};
#pragma unroll
            for (int c = 0; c < kPw; ++c) {
                const int col = lane + c * per_row;
                if (!exists || col >= D) continue;
                if constexpr (DT == HDLA_F32) r.w[c] = static_cast<const uint32_t*>(base)[row * D + col];
                else r.w[c / 2] |= static_cast<uint32_t>(static_cast<const uint16_t*>(base)[row * D + col]) << (c % 2 * 16);
            }
            return r;
        }
    }
    template <int DT>
    __device__ __forceinline__ void store(void* base, long long row, bool exists, const f2 (&v)[kPairs]) const {
        float f[kPw];
#pragma unroll
        for (int c = 0; c < kPairs; ++c) f2_unpack(v[c], f[2 * c], f[2 * c + 1]);
        if constexpr (Vec) {
            st_pack<DT, kPw, true>(base, row * D + col, exists ? valid : 0, f);
        } else {
#pragma unroll
            for (int c = 0; c < kPw; ++c)
                if (exists && lane + c * per_row < D) st_elem(base, row * D + lane + c * per_row, DT, f[c]);
        }
    }
    // this thread's channels of a vector in shared memory
    __device__ __forceinline__ void get(const float* vector, f2 (&v)[kPairs]) const {
        if constexpr (Vec) {
#pragma unroll
            for (int i = 0; i < kPairs; i += 2) {
                const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(vector + col + 2 * i);
                v[i] = q.x; v[i + 1] = q.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[i] = f2_pack(vector[lane + 2 * i * per_row], vector[lane + (2 * i + 1) * per_row]);
        }
    }
    __device__ __forceinline__ void put(float* vector, const f2 (&v)[kPairs]) const {
        if constexpr (Vec) {
#pragma unroll
            for (int i = 0; i < kPairs; i += 2) *reinterpret_cast<ulonglong2*>(vector + col + 2 * i) = make_ulonglong2(v[i], v[i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) f2_unpack(v[i], vector[lane + 2 * i * per_row], vector[lane + (2 * i + 1) * per_row]);
        }
    }
};

// The three vectors of weights in shared memory, `otherwise` where there is no tensor and zero behind the row's end.
__device__ __forceinline__ void put_weights(const NrP& p, float* to) {
    for (int i = threadIdx.x; i < p.stride; i += blockDim.x) {
        const bool in = i < p.a.D;
        to[i] = !in ? 0.f : p.a.post_weight ? ld_elem(p.a.post_weight, i, p.a.w_dtype) : 1.f;
        to[p.stride + i] = !in ? 0.f : p.a.pre_weight ? ld_elem(p.a.pre_weight, i, p.a.w_dtype) : 1.f;
        to[2 * p.stride + i] = !in ? 0.f : p.a.scale ? ld_elem(p.a.scale, i, p.a.w_dtype) : p.a.scale_value;
    }
    __syncthreads();
}
template <int DT>
__device__ __forceinline__ void unpack_pairs(const Pack<DT, kPw>& r, f2 (&v)[kPairs]) {
    float f[kPw];
    unpack<DT, kPw>(r, f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) v[i] = f2_pack(f[2 * i], f[2 * i + 1]);
}
// The gate's activation and its derivative.  silu and sigmoid are one expression: s t with t = g or 1, derivative m s + s (1 - s) t
// with m = 1 or 0.
struct GateAct {
    bool plain;
    f2 m, rest;
    __device__ __forceinline__ explicit GateAct(int act) : plain(act == HDLA_ACT_NONE) {
        m = f2_dup(act == HDLA_ACT_SILU ? 1.f : 0.f);
        rest = f2_dup(act == HDLA_ACT_SILU ? 0.f : 1.f);
    }
    // from g and its sigmoid
    __device__ __forceinline__ f2 value(f2 g, f2 s) const { return plain ? g : f2_mul(s, f2_fma(g, m, rest)); }
    __device__ __forceinline__ f2 slope(f2 g, f2 s) const {
        return plain ? f2_dup(1.f) : f2_fma(f2_fma(s, f2_dup(-1.f), f2_dup(1.f)), f2_mul(s, f2_fma(g, m, rest)), f2_mul(m, s));
    }
};

template <int DT, int RDT, bool Vec, int MaxThreads>
__global__ void __launch_bounds__(MaxThreads, MaxThreads == 256 ? 4 : MaxThreads == 512 ? 2 : 1)
norm_residual_fwd_kernel(const __grid_constant__ NrP p) {
    extern __shared__ __align__(16) float weights[];
    __shared__ float red[2][32];
    put_weights(p, weights);
    const Place<Vec> at(p);
    const int D = p.a.D;
    RowSum sum{red, 0, at.group * (p.per_row / 32), p.per_row / 32};
    const GateAct act(p.a.activation);
    const float root = sqrtf((float)D);
    constexpr bool Ahead = MaxThreads <= 512;
    Pack<DT, kPw> nx = {}, ng = {};
    Pack<RDT, kPw> nr = {};
    auto request = [&](long long row) {
        const bool exists = row < p.a.rows;
        if (at.rows == 1 && !(exists && at.any())) return;      // (a thread behind the row's end keeps its zeros)
        nx = at.template load<DT>(p.a.x, row, exists);
        if (p.a.residual) nr = at.template load<RDT>(p.a.residual, row, exists);
        if (p.a.gate) ng = at.template load<DT>(p.a.gate, row, exists);
    };
    long long first = (long long)blockIdx.x * at.rows;
    const long long step = (long long)gridDim.x * at.rows;
    if (Ahead) request(first + at.group);
    for (; first < p.a.rows; first += step) {
        const long long row = first + at.group;
        if (!Ahead) request(row);
        f2 v[kPairs], g[kPairs], r[kPairs], w[kPairs];
        unpack_pairs<DT>(nx, v);
        unpack_pairs<DT>(ng, g);
        unpack_pairs<RDT>(nr, r);
        if (Ahead && first + step < p.a.rows) request(row + step);
        if (p.a.post_weight) {
            f2 ss = 0;
#pragma unroll
            for (int c = 0; c < kPairs; ++c) ss = f2_fma(v[c], v[c], ss);
            const float factor = root * rsqrtf(sum.one(f2_sum(ss)) + p.a.eps);
            if (p.a.factors && at.lane == 0 && row < p.a.rows) p.a.factors[2 * row] = factor;
            const f2 k = f2_dup(factor);
            at.get(weights, w);
#pragma unroll
            for (int c = 0; c < kPairs; ++c) v[c] = f2_mul(v[c], f2_mul(k, w[c]));
        }
        if (p.a.gate)
#pragma unroll
            for (int c = 0; c < kPairs; ++c) v[c] = f2_mul(v[c], act.value(g[c], sigmoid_pair(g[c])));
        at.get(weights + 2 * p.stride, w);
        f2 ss = 0;
#pragma unroll
        for (int c = 0; c < kPairs; ++c) {
            r[c] = f2_fma(w[c], v[c], r[c]);
            ss = f2_fma(r[c], r[c], ss);
        }
        at.template store<RDT>(p.a.r, row, row < p.a.rows, r);
        if (p.a.pre_weight) {
            const float factor = root * rsqrtf(sum.one(f2_sum(ss)) + p.a.eps);
            if (p.a.factors && at.lane == 0 && row < p.a.rows) p.a.factors[2 * row + 1] = factor;
            const f2 k = f2_dup(factor);
            at.get(weights + p.stride, w);
#pragma unroll
            for (int c = 0; c < kPairs; ++c) r[c] = f2_mul(r[c], f2_mul(k, w[c]));
            at.template store<DT>(p.a.u, row, row < p.a.rows, r);
        }
    }
}

template <int DT, int RDT, bool Vec, int MaxThreads>
__global__ void __launch_bounds__(MaxThreads, MaxThreads == 256 ? 2 : 1) norm_residual_bwd_kernel(const __grid_constant__ NrP p) {
    extern __shared__ __align__(16) float weights[];        // 3 vectors; 3 of sums behind them where those are not in registers
    __shared__ float red[2][32];
    constexpr bool Lean = MaxThreads > 512;
    put_weights(p, weights);
    const Place<Vec> at(p);
    const int D = p.a.D;
    RowSum sum{red, 0, at.group * (p.per_row / 32), p.per_row / 32};
    const GateAct act(p.a.activation);
    f2 acc[Lean ? 1 : 3][kPairs];                           // post, pre, scale
    float* sums = weights + 3 * p.stride;
#pragma unroll
    for (int c = 0; c < kPairs; ++c) acc[0][c] = 0;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if (Lean) at.put(sums + k * p.stride, acc[0]);
        else
#pragma unroll
            for (int c = 0; c < kPairs; ++c) acc[Lean ? 0 : k][c] = 0;
    }
    auto add = [&](int k, const f2 (&a)[kPairs], const f2 (&b)[kPairs]) {      // sum k += a b
        if constexpr (Lean) {
            f2 t[kPairs];
            at.get(sums + k * p.stride, t);
#pragma unroll
            for (int c = 0; c < kPairs; ++c) t[c] = f2_fma(a[c], b[c], t[c]);
            at.put(sums + k * p.stride, t);
        } else {
#pragma unroll
            for (int c = 0; c < kPairs; ++c) acc[k][c] = f2_fma(a[c], b[c], acc[k][c]);
        }
    };
    const float per = 1.f / (float)D;
    float fx = 0.f, fr = 0.f;                               // the norms' factors of the next row
    auto factors = [&](long long row) {
        if (row >= p.a.rows) return;
        if (p.a.post_weight) fx = __ldg(p.a.factors + 2 * row);
        if (p.a.pre_weight) fr = __ldg(p.a.factors + 2 * row + 1);
    };
    Pack<DT, kPw> nx = {}, ng = {}, nu = {};
    Pack<RDT, kPw> nr = {}, nd = {};
    auto request = [&](long long row) {
        const bool exists = row < p.a.rows;
        if (at.rows == 1 && !(exists && at.any())) return;      // (a thread behind the row's end keeps its zeros)
        nx = at.template load<DT>(p.a.x, row, exists);
        if (p.a.residual) nr = at.template load<RDT>(p.a.residual, row, exists);
        if (p.a.gate) ng = at.template load<DT>(p.a.gate, row, exists);
        if (p.a.dr) nd = at.template load<RDT>(p.a.dr, row, exists);
        if (p.a.du) nu = at.template load<DT>(p.a.du, row, exists);
    };
    long long first = (long long)blockIdx.x * at.rows;
    const long long step = (long long)gridDim.x * at.rows;
    if (!Lean) request(first + at.group);
    factors(first + at.group);
    for (; first < p.a.rows; first += step) {
        const long long row = first + at.group;
        if (Lean) request(row);
        const Pack<DT, kPw> cx = nx, cg = ng, cu = nu;
        const Pack<RDT, kPw> cr = nr, cd = nd;
        if (!Lean && first + step < p.a.rows) request(row + step);
        const bool exists = row < p.a.rows;                 // (a block's last rows may not)
        // what is used twice is unpacked twice: registers are short
        f2 s[kPairs], d[kPairs];                            // the gate's sigmoid; the gradient on its way from r to x
        // n = x kx post, v = n act(g), r = residual + scale v
        const float kx = !p.a.post_weight ? 1.f : exists ? fx : 0.f, kr = exists ? fr : 0.f;
        if (first + step < p.a.rows) factors(row + step);
        if (p.a.gate) {
            unpack_pairs<DT>(cg, s);
#pragma unroll
            for (int c = 0; c < kPairs; ++c) s[c] = sigmoid_pair(s[c]);
        }
        unpack_pairs<RDT>(cd, d);
        if (p.a.pre_weight) {
            f2 x[kPairs], r[kPairs], w[kPairs], k[kPairs], dot = 0;
            unpack_pairs<DT>(cx, x);
            at.get(weights, w);
#pragma unroll
            for (int c = 0; c < kPairs; ++c) x[c] = f2_mul(x[c], f2_mul(w[c], f2_dup(kx)));
            if (p.a.gate) {
                f2 g[kPairs];
                unpack_pairs<DT>(cg, g);
#pragma unroll
                for (int c = 0; c < kPairs; ++c) x[c] = f2_mul(x[c], act.value(g[c], s[c]));
            }
            unpack_pairs<RDT>(cr, r);
            at.get(weights + 2 * p.stride, k);
            at.get(weights + p.stride, w);
            f2 t[kPairs];
            unpack_pairs<DT>(cu, t);
#pragma unroll
            for (int c = 0; c < kPairs; ++c) {
                r[c] = f2_fma(k[c], x[c], r[c]);
                dot = f2_fma(f2_mul(t[c], w[c]), r[c], dot);
            }
            const float back = kr * (kr * per * sum.one(f2_sum(dot)));
#pragma unroll
            for (int c = 0; c < kPairs; ++c) {
                r[c] = f2_mul(r[c], f2_dup(kr));
                d[c] = f2_fma(f2_mul(t[c], f2_dup(kr)), w[c], f2_fma(f2_dup(-back), r[c], d[c]));
            }
            add(1, t, r);
        }
        if (p.a.dresidual) at.template store<RDT>(p.a.dresidual, row, exists, d);
        f2 x[kPairs], w[kPairs];
        unpack_pairs<DT>(cx, x);
        at.get(weights, w);
        {
            f2 n[kPairs], k[kPairs];
#pragma unroll
            for (int c = 0; c < kPairs; ++c) n[c] = f2_mul(x[c], f2_mul(w[c], f2_dup(kx)));
            at.get(weights + 2 * p.stride, k);
            if (p.a.gate) {
                f2 g[kPairs], v[kPairs];
                unpack_pairs<DT>(cg, g);
#pragma unroll
                for (int c = 0; c < kPairs; ++c) {
                    const f2 a = act.value(g[c], s[c]), dv = f2_mul(k[c], d[c]);
                    v[c] = f2_mul(n[c], a);
                    g[c] = f2_mul(f2_mul(dv, n[c]), act.slope(g[c], s[c]));
                    k[c] = f2_mul(dv, a);
                }
                add(2, d, v);
                if (p.a.dgate) at.template store<DT>(p.a.dgate, row, exists, g);
            } else {
                add(2, d, n);
#pragma unroll
                for (int c = 0; c < kPairs; ++c) k[c] = f2_mul(k[c], d[c]);
            }
#pragma unroll
            for (int c = 0; c < kPairs; ++c) d[c] = k[c];
        }
        if (p.a.post_weight) {
            f2 dot = 0;
#pragma unroll
            for (int c = 0; c < kPairs; ++c) dot = f2_fma(f2_mul(d[c], w[c]), x[c], dot);
            const float back = kx * (kx * per * sum.one(f2_sum(dot)));
#pragma unroll
            for (int c = 0; c < kPairs; ++c) x[c] = f2_mul(x[c], f2_dup(kx));
            add(0, d, x);
#pragma unroll
            for (int c = 0; c < kPairs; ++c) d[c] = f2_fma(f2_mul(d[c], f2_dup(kx)), w[c], f2_mul(f2_dup(-back), x[c]));
        }
        at.template store<DT>(p.a.dx, row, exists, d);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        float* to = p.part + ((long long)blockIdx.x * 3 + k) * D;
        __syncthreads();                                    // (the weights are not read any more, nor the sums before)
        if (Lean) {
            for (int c = threadIdx.x; c < D; c += blockDim.x) to[c] = weights[(3 + k) * p.stride + c];
        } else {
            at.put(weights + at.group * p.stride, acc[Lean ? 0 : k]);
            __syncthreads();
            for (int c = threadIdx.x; c < D; c += blockDim.x) {
                float v = 0.f;
                for (int g = 0; g < at.rows; ++g) v += weights[g * p.stride + c];
                to[c] = v;
            }
        }
    }
}

// A row's threads, and the block: at least 256 threads, so narrow rows share it.
int row_threads(int D) { return ((D + kPw - 1) / kPw + 31) / 32 * 32; }
int block_threads(int per_row) { return per_row >= 256 ? per_row : 256 / per_row * per_row; }

// the threads that a kernel for blocks of `threads` is built for
int built_for(int threads) { return threads > 512 ? 1024 : threads > 256 ? 512 : 256; }

bool norm_vec(const HdlaNormResidualArgs& a) {
    for (const void* q : {a.x, a.residual, a.gate, (const void*)a.r, (const void*)a.u, a.dr, a.du, (const void*)a.dx,
                          (const void*)a.dresidual, (const void*)a.dgate})
        if (!aligned16(q)) return false;
    return a.D % kPw == 0;
}

typedef void (*Kernel)(const NrP);
template <int DT, int RDT, bool Vec>
Kernel kernel_for(bool backward, int threads) {
    const int n = built_for(threads);
    if (backward)
        return n == 1024 ? norm_residual_bwd_kernel<DT, RDT, Vec, 1024> : n == 512 ? norm_residual_bwd_kernel<DT, RDT, Vec, 512>
                                                                                    : norm_residual_bwd_kernel<DT, RDT, Vec, 256>;
    return n == 1024 ? norm_residual_fwd_kernel<DT, RDT, Vec, 1024> : n == 512 ? norm_residual_fwd_kernel<DT, RDT, Vec, 512>
                                                                                : norm_residual_fwd_kernel<DT, RDT, Vec, 256>;
}
Kernel pick(const HdlaNormResidualArgs& a, bool backward, int threads) {
    const bool vec = norm_vec(a);
    if (a.dtype == HDLA_F32) return vec ? kernel_for<HDLA_F32, HDLA_F32, true>(backward, threads) : kernel_for<HDLA_F32, HDLA_F32, false>(backward, threads);
    if (a.r_dtype == HDLA_F32) return vec ? kernel_for<HDLA_BF16, HDLA_F32, true>(backward, threads) : kernel_for<HDLA_BF16, HDLA_F32, false>(backward, threads);
    return vec ? kernel_for<HDLA_BF16, HDLA_BF16, true>(backward, threads) : kernel_for<HDLA_BF16, HDLA_BF16, false>(backward, threads);
}
// as many blocks as there are rows for, and at most those that are resident at once (four of 256 threads an SM, two backward);
// they walk over the rows
unsigned blocks_of(const HdlaNormResidualArgs& a, bool backward) {
    const int per_row = row_threads(a.D), threads = block_threads(per_row), rows = threads / per_row;
    const long long need = (a.rows + rows - 1) / rows, each = (backward ? 512 : 1024) / threads, most = (long long)sm_count() * (each > 1 ? each : 1);
    return static_cast<unsigned>(need < most ? need : most);
}
// three vectors of weights, which at the end make room for a vector of sums for each row of the block; three more of sums
size_t shared_of(int per_row, int threads, bool backward) {
    const int rows = threads / per_row, vectors = !backward ? 3 : threads > 512 ? 6 : rows > 3 ? rows : 3;
    return sizeof(float) * kPw * per_row * vectors;
}
int launch(const HdlaNormResidualArgs& a, bool backward, float* part, cudaStream_t st) {
    const int per_row = row_threads(a.D), threads = block_threads(per_row);
    const NrP p{a, per_row, kPw * per_row, part};
    const Kernel kernel = pick(a, backward, threads);
    const size_t bytes = shared_of(per_row, threads, backward);
    if (bytes > 47 << 10) {                                      // (the sums have some of the 48 KB that need no request)
        // The limit is the kernel's, not this launch's, and other threads may be between setting it and launching: what all of
        // them set is the most that any launch of this kernel takes.
        const int most = built_for(threads);
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)shared_of(most, most, backward));
        if (e != cudaSuccess) return fail(HDLA_ERR_CUDA, "norm_residual: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    }
    kernel<<<blocks_of(a, backward), threads, bytes, st>>>(p);
    HDLA_CHECK_LAUNCH(backward ? "norm_residual_bwd_kernel" : "norm_residual_fwd_kernel");
    return HDLA_OK;
}

}  // namespace

int norm_residual_max_d() { return kMaxD; }

size_t norm_residual_bwd_workspace(const HdlaNormResidualArgs& a) { return up256((size_t)blocks_of(a, true) * 3 * a.D * sizeof(float)); }

int norm_residual_fwd(const HdlaNormResidualArgs& a, cudaStream_t st) { return launch(a, false, nullptr, st); }

int norm_residual_bwd(const HdlaNormResidualArgs& a, float* part, cudaStream_t st) {
    if (int rc = launch(a, true, part, st)) return rc;
    if (!a.dpost_weight && !a.dpre_weight && !a.dscale) return HDLA_OK;
    ColJobs js{};
    js.n = 1;
    js.j[0] = ColJob{part, {a.dpost_weight, a.dpre_weight, a.dscale}, 3LL * a.D, (int)blocks_of(a, true), 3, a.D, a.D, a.w_dtype, 0, 0, 0};
    return column_sum_launch(js, st);
}

}  // namespace hdla
