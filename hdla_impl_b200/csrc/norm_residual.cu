// RMS norms after and before a block, with the block's gate, residual scale and residual sum, per row of D channels:
//     v = x or rms(x) post;   v = v act(gate);   r = residual + scale v;   u = rms(r) pre,   rms(a) = sqrt(D) a / sqrt(sum a^2 + eps)
// forward and backward as one kernel each: every tensor is read or written once, which is what bounds them (HBM).
//
// A thread owns eight neighbouring channels of a row (16-byte accesses of bf16) and holds them between the sums; a row takes
// as many whole warps as it needs, narrow rows share a block.  Blocks walk over rows and request the next row's tensors
// before the sums of this one.  Backward computes r again from the inputs in fp32 (as many bytes as reading the rounded r),
// takes three sums (x^2; r^2 with the dot product of the pre norm's gradient; that of the post norm's), and keeps the sums
// over rows (gradients of the weights and of scale) in registers until its last row; blocks' sums are added in a fixed order.
#include "ssm.cuh"

namespace hdla {
namespace {

constexpr int kPw = 8, kMaxD = 1024 * kPw;

struct NrP {
    HdlaNormResidualArgs a;
    int per_row;             // threads of a row (whole warps)
    float* part;             // backward: [blocks][3][D] (post, pre, scale)
};

// Two sums over the warps of a row.  `red` has two buffers, used in turn, so that one barrier a sum is enough.
struct RowSum {
    float2 (*red)[32];
    int turn, first, warps;
    __device__ __forceinline__ float2 operator()(float a, float b) {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        if (warps == 1) return make_float2(a, b);
        if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        float2 t = make_float2(0.f, 0.f);
        for (int w = 0; w < warps; ++w) {
            const float2 v = red[turn][first + w];
            t.x += v.x; t.y += v.y;
        }
        turn ^= 1;
        return t;
    }
};

// Where a thread stands, and its channels' weights.
struct Place {
    int rows, group, col, valid;
    __device__ __forceinline__ explicit Place(const NrP& p) {
        rows = blockDim.x / p.per_row;
        group = threadIdx.x / p.per_row;
        col = (threadIdx.x % p.per_row) * kPw;
        valid = max(0, min(kPw, p.a.D - col));
    }
};
// eight weights: `otherwise` where there is no tensor
__device__ __forceinline__ void ld_weights(const void* w, int dt, int col, int valid, float otherwise, float (&f)[kPw]) {
#pragma unroll
    for (int c = 0; c < kPw; ++c) f[c] = w && c < valid ? ld_elem(w, col + c, dt) : otherwise;
}

template <int DT, int RDT, bool Vec, int MaxThreads>
__global__ void __launch_bounds__(MaxThreads) norm_residual_fwd_kernel(const __grid_constant__ NrP p) {
    __shared__ float2 red[2][32];
    const Place at(p);
    const int D = p.a.D;
    RowSum sum{red, 0, at.group * (p.per_row / 32), p.per_row / 32};
    float post[kPw], pre[kPw], scale[kPw];
    ld_weights(p.a.post_weight, p.a.w_dtype, at.col, at.valid, 1.f, post);
    ld_weights(p.a.pre_weight, p.a.w_dtype, at.col, at.valid, 1.f, pre);
    ld_weights(p.a.scale, p.a.w_dtype, at.col, at.valid, p.a.scale_value, scale);
    const float root = sqrtf((float)D);
    Pack<DT, kPw> nx, ng = {};
    Pack<RDT, kPw> nr = {};
    auto request = [&](long long row) {
        const int ok = row < p.a.rows ? at.valid : 0;
        const long long i = row * D + at.col;
        nx = ld_pack<DT, kPw, Vec>(p.a.x, i, ok);
        if (p.a.residual) nr = ld_pack<RDT, kPw, Vec>(p.a.residual, i, ok);
        if (p.a.gate) ng = ld_pack<DT, kPw, Vec>(p.a.gate, i, ok);
    };
    long long first = (long long)blockIdx.x * at.rows;
    request(first + at.group);
    for (; first < p.a.rows; first += (long long)gridDim.x * at.rows) {
        const long long row = first + at.group;
        float v[kPw], g[kPw], r[kPw];
        unpack<DT, kPw>(nx, v);
        unpack<DT, kPw>(ng, g);
        unpack<RDT, kPw>(nr, r);
        request(row + (long long)gridDim.x * at.rows);
        if (p.a.post_weight) {
            float ss = 0.f;
#pragma unroll
            for (int c = 0; c < kPw; ++c) ss = fmaf(v[c], v[c], ss);
            const float k = root * rsqrtf(sum(ss, 0.f).x + p.a.eps);
#pragma unroll
            for (int c = 0; c < kPw; ++c) v[c] *= k * post[c];
        }
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < kPw; ++c) {
            if (p.a.gate) v[c] *= act_of(g[c], p.a.activation);
            r[c] = fmaf(scale[c], v[c], r[c]);
            if (c < at.valid) ss = fmaf(r[c], r[c], ss);
        }
        const int ok = row < p.a.rows ? at.valid : 0;
        st_pack<RDT, kPw, Vec>(p.a.r, row * D + at.col, ok, r);
        if (p.a.pre_weight) {
            const float k = root * rsqrtf(sum(ss, 0.f).x + p.a.eps);
#pragma unroll
            for (int c = 0; c < kPw; ++c) r[c] *= k * pre[c];
            st_pack<DT, kPw, Vec>(p.a.u, row * D + at.col, ok, r);
        }
    }
}

template <int DT, int RDT, bool Vec, int MaxThreads>
__global__ void __launch_bounds__(MaxThreads) norm_residual_bwd_kernel(const __grid_constant__ NrP p) {
    __shared__ float2 red[2][32];
    __shared__ float over[kPw * 256];                       // rows that share a block (at most 256 threads then)
    const Place at(p);
    const int D = p.a.D;
    RowSum sum{red, 0, at.group * (p.per_row / 32), p.per_row / 32};
    float post[kPw], pre[kPw], scale[kPw], dpost[kPw] = {}, dpre[kPw] = {}, dscale[kPw] = {};
    ld_weights(p.a.post_weight, p.a.w_dtype, at.col, at.valid, 1.f, post);
    ld_weights(p.a.pre_weight, p.a.w_dtype, at.col, at.valid, 1.f, pre);
    ld_weights(p.a.scale, p.a.w_dtype, at.col, at.valid, p.a.scale_value, scale);
    const float root = sqrtf((float)D), per = 1.f / (float)D;
    Pack<DT, kPw> nx, ng = {}, nu = {};
    Pack<RDT, kPw> nr = {}, nd = {};
    auto request = [&](long long row) {
        const int ok = row < p.a.rows ? at.valid : 0;
        const long long i = row * D + at.col;
        nx = ld_pack<DT, kPw, Vec>(p.a.x, i, ok);
        if (p.a.residual) nr = ld_pack<RDT, kPw, Vec>(p.a.residual, i, ok);
        if (p.a.gate) ng = ld_pack<DT, kPw, Vec>(p.a.gate, i, ok);
        if (p.a.dr) nd = ld_pack<RDT, kPw, Vec>(p.a.dr, i, ok);
        if (p.a.du) nu = ld_pack<DT, kPw, Vec>(p.a.du, i, ok);
    };
    long long first = (long long)blockIdx.x * at.rows;
    request(first + at.group);
    for (; first < p.a.rows; first += (long long)gridDim.x * at.rows) {
        const long long row = first + at.group;
        float x[kPw], g[kPw], d[kPw];
        unpack<DT, kPw>(nx, x);
        unpack<DT, kPw>(ng, g);
        unpack<RDT, kPw>(nd, d);
        const Pack<RDT, kPw> cr = nr;
        const Pack<DT, kPw> cu = nu;
        request(row + (long long)gridDim.x * at.rows);
        float kx = 1.f;                                     // n = x kx post, v = n act(g), r = residual + scale v
        if (p.a.post_weight) {
            float ss = 0.f;
#pragma unroll
            for (int c = 0; c < kPw; ++c) ss = fmaf(x[c], x[c], ss);
            ss = sum(ss, 0.f).x;
            kx = row < p.a.rows ? root * rsqrtf(ss + p.a.eps) : 0.f;      // (a block's last rows may not exist)
        }
        if (p.a.pre_weight) {
            float r[kPw], t[kPw], ss = 0.f, dot = 0.f;
            unpack<RDT, kPw>(cr, r);
            unpack<DT, kPw>(cu, t);
#pragma unroll
            for (int c = 0; c < kPw; ++c) {
                float v = x[c] * kx * post[c];
                if (p.a.gate) v *= act_of(g[c], p.a.activation);
                r[c] = fmaf(scale[c], v, r[c]);
                if (c < at.valid) {
                    ss = fmaf(r[c], r[c], ss);
                    dot = fmaf(t[c] * pre[c], r[c], dot);
                }
            }
            const float2 s = sum(ss, dot);
            const float kr = row < p.a.rows ? root * rsqrtf(s.x + p.a.eps) : 0.f, back = kr * kr * kr * per * s.y;
#pragma unroll
            for (int c = 0; c < kPw; ++c) {
                d[c] += kr * (t[c] * pre[c]) - back * r[c];
                dpre[c] = fmaf(t[c] * kr, r[c], dpre[c]);
            }
        }
        const int ok = row < p.a.rows ? at.valid : 0;
        const long long i = row * D + at.col;
        if (p.a.dresidual) st_pack<RDT, kPw, Vec>(p.a.dresidual, i, ok, d);
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < kPw; ++c) {
            const float n = x[c] * kx * post[c];
            float v = n, dv = scale[c] * d[c];
            if (p.a.gate) {
                const float act = act_of(g[c], p.a.activation);
                v *= act;
                g[c] = dv * n * act_grad(g[c], p.a.activation);
                dv *= act;
            }
            dscale[c] = fmaf(d[c], v, dscale[c]);
            d[c] = dv;
            dot = fmaf(dv * post[c], x[c], dot);
        }
        if (p.a.dgate) st_pack<DT, kPw, Vec>(p.a.dgate, i, ok, g);
        if (p.a.post_weight) {
            const float back = kx * kx * kx * per * sum(dot, 0.f).x;
#pragma unroll
            for (int c = 0; c < kPw; ++c) {
                dpost[c] = fmaf(d[c] * kx, x[c], dpost[c]);
                d[c] = kx * (d[c] * post[c]) - back * x[c];
            }
        }
        st_pack<DT, kPw, Vec>(p.a.dx, i, ok, d);
    }
#pragma unroll
    for (int what = 0; what < 3; ++what) {
        const float* s = what == 0 ? dpost : what == 1 ? dpre : dscale;
        float* to = p.part + ((long long)blockIdx.x * 3 + what) * D;
        if (at.rows == 1) {
#pragma unroll
            for (int c = 0; c < kPw; ++c)
                if (c < at.valid) to[at.col + c] = s[c];
        } else {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < kPw; ++c) over[threadIdx.x * kPw + c] = s[c];
            __syncthreads();
            for (int c = threadIdx.x; c < D; c += blockDim.x) {
                float v = 0.f;
                for (int k = 0; k < at.rows; ++k) v += over[k * p.per_row * kPw + c];
                to[c] = v;
            }
        }
    }
}

// A row's threads, and the block: at least 256 threads, so narrow rows share it.
int row_threads(int D) { return ((D + kPw - 1) / kPw + 31) / 32 * 32; }
int block_threads(int per_row) { return per_row >= 256 ? per_row : 256 / per_row * per_row; }

bool norm_vec(const HdlaNormResidualArgs& a) {
    for (const void* q : {a.x, a.residual, a.gate, (const void*)a.r, (const void*)a.u, a.dr, a.du, (const void*)a.dx,
                          (const void*)a.dresidual, (const void*)a.dgate})
        if (!aligned16(q)) return false;
    return a.D % kPw == 0;
}

typedef void (*Kernel)(const NrP);
template <int DT, int RDT, bool Vec>
Kernel kernel_for(bool backward, int threads) {
    if (backward) return threads > 512 ? norm_residual_bwd_kernel<DT, RDT, Vec, 1024> : threads > 256 ? norm_residual_bwd_kernel<DT, RDT, Vec, 512> : norm_residual_bwd_kernel<DT, RDT, Vec, 256>;
    return threads > 512 ? norm_residual_fwd_kernel<DT, RDT, Vec, 1024> : threads > 256 ? norm_residual_fwd_kernel<DT, RDT, Vec, 512> : norm_residual_fwd_kernel<DT, RDT, Vec, 256>;
}
Kernel pick(const HdlaNormResidualArgs& a, bool backward, int threads) {
    const bool vec = norm_vec(a);
    if (a.dtype == HDLA_F32) return vec ? kernel_for<HDLA_F32, HDLA_F32, true>(backward, threads) : kernel_for<HDLA_F32, HDLA_F32, false>(backward, threads);
    if (a.r_dtype == HDLA_F32) return vec ? kernel_for<HDLA_BF16, HDLA_F32, true>(backward, threads) : kernel_for<HDLA_BF16, HDLA_F32, false>(backward, threads);
    return vec ? kernel_for<HDLA_BF16, HDLA_BF16, true>(backward, threads) : kernel_for<HDLA_BF16, HDLA_BF16, false>(backward, threads);
}
// as many blocks as there are rows for, and at most four (backward: two) of 256 threads an SM, which walk over the rows
unsigned blocks_of(const HdlaNormResidualArgs& a, bool backward) {
    const int per_row = row_threads(a.D), threads = block_threads(per_row), rows = threads / per_row;
    const long long need = (a.rows + rows - 1) / rows, most = (long long)sm_count() * ((backward ? 512 : 1024) / threads > 1 ? (backward ? 512 : 1024) / threads : 1);
    return static_cast<unsigned>(need < most ? need : most);
}

}  // namespace

int norm_residual_max_d() { return kMaxD; }

size_t norm_residual_bwd_workspace(const HdlaNormResidualArgs& a) { return up256((size_t)blocks_of(a, true) * 3 * a.D * sizeof(float)); }

int norm_residual_fwd(const HdlaNormResidualArgs& a, cudaStream_t st) {
    NrP p{a, row_threads(a.D), nullptr};
    const int threads = block_threads(p.per_row);
    pick(a, false, threads)<<<blocks_of(a, false), threads, 0, st>>>(p);
    HDLA_CHECK_LAUNCH("norm_residual_fwd_kernel");
    return HDLA_OK;
}

int norm_residual_bwd(const HdlaNormResidualArgs& a, float* part, cudaStream_t st) {
    NrP p{a, row_threads(a.D), part};
    const int threads = block_threads(p.per_row);
    const unsigned blocks = blocks_of(a, true);
    pick(a, true, threads)<<<blocks, threads, 0, st>>>(p);
    HDLA_CHECK_LAUNCH("norm_residual_bwd_kernel");
    if (!a.dpost_weight && !a.dpre_weight && !a.dscale) return HDLA_OK;
    ColJobs js{};
    js.n = 1;
    js.j[0] = ColJob{part, {a.dpost_weight, a.dpre_weight, a.dscale}, 3LL * a.D, (int)blocks, 3, a.D, a.D, a.w_dtype, 0, 0, 0};
    return column_sum_launch(js, st);
}

}  // namespace hdla
