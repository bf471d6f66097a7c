// Selective state space scan, forward and single tokens (the layout of the work is in selective_scan.cuh).
//
// What the forward pass cannot do without: the exponentials, one per (token, channel, state) and four more per (token, channel), 16
// a clock and SM; HBM traffic takes a third of that at N = 16.  8 x 4096 x 2048, N = 16, bf16, with checkpoints: 578 us, 1.9 times
// its exponentials; where rows are cut the maps take them a second time (one row of 65536 tokens: 2.3 times).  No pipe is full
// (with two channels a lane the exponentials' 62 %, shared-memory cycles 59 %, issue slots 52 %): the phases of a tile between its
// barriers do not overlap.  (A quarter of the exponentials as polynomials on the multiply-add pipes made it slower: 835 -> 879 us.)
#include "selective_scan.cuh"

namespace hdla {
namespace {

// Maps: only the recurrence, from zero at the segment's first token (or from the initial state of a sequence that starts
// inside it); its last state and sum of d are the segment's map.
template <int DT, bool Vec, int NL, int CT, bool Maps>
__global__ void __launch_bounds__(kScanThreads, CT == 1 && !Maps ? 4 : 5) scan_fwd_kernel(const __grid_constant__ ScanP p) {
    using TileT = Tile<NL, CT>;
    constexpr int NP = TileT::NP, CH = TileT::CH, Pitch = TileT::Pitch, PW = 4;
    constexpr int TB = CH > 64 || NL >= 16 ? 8 : 16, Groups = CH / PW, Items = TB * Groups, IT = (Items + kScanThreads - 1) / kScanThreads;
    static_assert(CH % PW == 0 && kScanThreads % Groups == 0, "a thread's pieces are of one group of channels");
    // tokens whose loads and exponentials may be mixed: sixteen with one channel a lane (eight: 616 instead of 595 us), eight with two
    // (sixteen outgrow the registers: 922 instead of 801 us; sizes as at scan_plan)
    constexpr int Unroll = CT == 2 ? 8 : TB;
    __shared__ __align__(16) float s_d[TB][CH], s_u[TB][CH], s_B[TB][NP], s_C[TB][NP], s_y[Maps ? 1 : TB * NL][Pitch];

    const int segments = Maps ? p.n_seg - 1 : p.n_seg;           // (nothing follows the last segment's map)
    const TileT w(p, segments);
    const int T = p.a.T, D = p.a.D, N = p.a.N, t0 = w.k * p.seg, t1 = min(T, t0 + p.seg);
    const Seqs q{p.a.cu_seqlens, p.a.cu_seqlens ? p.a.n_seqs : 1, T};
    const int dead = q.end();

    // pieces of a (token, channels) tile: this thread's are all of one group of channels
    const int cg = (threadIdx.x % Groups) * PW, valid = min(PW, w.count - cg), dch = w.d0 + cg;
    f2 bias[2], skip[2];
    {
        float b[PW], k[PW];
#pragma unroll
        for (int c = 0; c < PW; ++c) {
            b[c] = p.a.dt_bias && c < valid ? p.a.dt_bias[dch + c] : 0.f;
            k[c] = !Maps && p.a.skip && c < valid ? p.a.skip[dch + c] : 0.f;
        }
        bias[0] = f2_pack(b[0], b[1]); bias[1] = f2_pack(b[2], b[3]);
        skip[0] = f2_pack(k[0], k[1]); skip[1] = f2_pack(k[2], k[3]);
    }
    constexpr int Ahead = kScanThreads / Groups;                 // tokens between a thread's pieces
    const int tok0 = threadIdx.x / Groups;
    Walk fx = Walk::of<DT>(p.a.x, w.b * p.a.x_batch + (t0 + tok0) * p.a.x_token + dch, p.a.x_token, Ahead);
    Walk fd = Walk::of<DT>(p.a.dt, w.b * p.a.dt_batch + (t0 + tok0) * p.a.dt_token + dch, p.a.dt_token, Ahead);
    Walk fz = Walk::of<DT>(p.a.z, w.b * p.a.z_batch + (t0 + tok0) * p.a.z_token + dch, p.a.z_token, Ahead);
    const bool has_z = !Maps && p.a.z;
    Pack<DT, PW> nx[IT], nd[IT], nz[IT];
    BcTile<DT, NL, TB> bc(p, w.b, w.group, t0);
    auto request = [&](int tokens) {                             // of the next tile's first `tokens` tokens
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int ok = tok0 + i * Ahead < min(tokens, TB) ? valid : 0;
            nx[i] = fx.load<DT, Vec>(i, ok);
            nd[i] = fd.load<DT, Vec>(i, ok);
            if (has_z) nz[i] = fz.load<DT, Vec>(i, ok);
        }
        bc.template request<Vec>(min(tokens, dead - t1 + tokens));   // (rows of no sequence may hold anything, and anything times 0 is not 0)
        fx.move(TB); fd.move(TB); fz.move(TB);
        bc.from.move(TB);
    };
    request(t1 - t0);

    // the lane's decay rates and states
    f2 A[CT][2], h[CT][2], sum_d[CT];
    const int n0 = 4 * w.nl;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        sum_d[c] = 0;
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

    float* save = p.a.checkpoints + (((size_t)w.b * ((T + kCheckpoint - 1) / kCheckpoint) + t0 / kCheckpoint) * D + w.d0 + w.c0) * NP + n0;
    auto token = [&](int j, int tokens) {
        if (!Maps && j % kCheckpoint == 0 && p.a.checkpoints && j < tokens) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
                if (w.c0 + c < w.count) st_quad(save + ((size_t)(j / kCheckpoint) * D + c) * NP, h[c]);
        }
        f2 d[CT], u[CT], B[2], C[2];
        ld_twice<CT>(&s_d[j][w.c0], d);
        ld_twice<CT>(&s_u[j][w.c0], u);
        ld_quad(&s_B[j][n0], B);
        if (!Maps) ld_quad(&s_C[j][n0], C);
        float y[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            h[c][0] = f2_fma(ex2_pair(f2_mul(d[c], A[c][0])), h[c][0], f2_mul(u[c], B[0]));
            h[c][1] = f2_fma(ex2_pair(f2_mul(d[c], A[c][1])), h[c][1], f2_mul(u[c], B[1]));
            if (Maps) sum_d[c] = f2_add(sum_d[c], d[c]);
            else y[c] = f2_sum(f2_fma(C[1], h[c][1], f2_mul(C[0], h[c][0])));
        }
        if (!Maps) st_channels<CT>(&s_y[j * NL + w.nl][w.c0], y);
    };
    char* to = static_cast<char*>(p.a.y) + (((long long)w.b * T + t0 + tok0) * D + dch) * (DT == HDLA_F32 ? 4 : 2);
    const long long to_token = (long long)D * (DT == HDLA_F32 ? 4 : 2);

    for (int tb = t0; tb < t1; tb += TB) {
        const int tokens = t1 - tb, live = dead - tb;            // (may be more than a tile; those from `live` on are of no sequence)
        Pack<DT, PW> cx[IT], cz[IT];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int tok = tok0 + i * Ahead;
            cx[i] = nx[i];
            if (!Maps) cz[i] = nz[i];
            if (Items % kScanThreads && tok >= TB) continue;
            f2 x[2], d[2];
            unpack_pairs<DT>(nx[i], x);
            unpack_pairs<DT>(nd[i], d);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                d[c] = f2_add(d[c], bias[c]);
                if (p.a.softplus) d[c] = softplus_pair(d[c]);
                x[c] = f2_mul(x[c], d[c]);
            }
            if (live < TB && tok >= live) d[0] = d[1] = x[0] = x[1] = 0;
            st_pairs(&s_d[tok][cg], d);
            st_pairs(&s_u[tok][cg], x);
        }
        bc.put(&s_B[0][0], &s_C[0][0]);
        if (tokens > TB) request(tokens - TB);
        __syncthreads();
        if (end > tb + TB) {
#pragma unroll Unroll
            for (int j = 0; j < TB; ++j) token(j, tokens);
        } else {                                                 // a sequence ends in this tile
#pragma unroll 1
            for (int j = 0; j < min(TB, tokens); ++j) {
                token(j, tokens);
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
            save += (size_t)(TB / kCheckpoint) * D * NP;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int tok = tok0 + i * Ahead;
                if (tok >= min(TB, tokens)) continue;
                f2 x[2], z[2], y[2];
                unpack_pairs<DT>(cx[i], x);
                add_partial<NL>(&s_y[tok * NL][cg], Pitch, y);
                if (has_z) unpack_pairs<DT>(cz[i], z);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    y[c] = f2_fma(skip[c], x[c], y[c]);
                    if (has_z) y[c] = f2_mul(y[c], f2_mul(z[c], sigmoid_pair(z[c])));
                }
                if (live < TB && tok >= live) y[0] = y[1] = 0;
                float out[PW];
                unpair(y, out);
                st_pack<DT, PW, Vec>(to + i * Ahead * to_token, 0, valid, out);
            }
            to += TB * to_token;
        }
    }
    if (Maps) {
        const size_t row = ((size_t)w.b * p.n_seg + w.k) * D + w.d0 + w.c0;
#pragma unroll
        for (int c = 0; c < CT; ++c)
            if (w.c0 + c < w.count) {
                st_quad(p.map_h + (row + c) * NP + n0, h[c]);
                float a, b;
                f2_unpack(sum_d[c], a, b);
                if (w.nl == 0) p.map_d[row + c] = a;
            }
    }
}

// ------------------------------------------------------------------------------------------ single tokens
// NL lanes a channel, four states a lane; a thread has the same channel in Rows sequences, so that A is read once and the
// states' loads of Rows sequences are in flight together.  What is done once per (sequence, channel) -- softplus, gate, the
// loads and the store of x, dt, z, y -- each lane does for one of the sequences, and hands d and d x to the others of its
// channel: done by every lane for every sequence it was three quarters of the instructions, and took longer than the memory.
// Bound by HBM: the fp32 state is read and written once (256 sequences of 4096 channels of 16 states: 27 us; 41 us where the
// loads' width was a branch, see ld_state_once).
template <int DT, int NL, int Rows, bool Vec>
__global__ void __launch_bounds__(128) scan_step_kernel(const __grid_constant__ ScanP p) {
    static_assert(Rows == 1 || Rows <= NL, "a lane has one of the sequences");
    const int D = p.a.D, N = p.a.N, lane = threadIdx.x & 31, nl = lane % NL;
    const int blocks = (D + 128 / NL - 1) / (128 / NL);
    const int d = blockIdx.x % blocks * (128 / NL) + threadIdx.x / NL, dd = min(d, D - 1), group = dd / p.Dg;
    const int n0 = d < D ? 4 * nl : N;                         // (lanes behind the last channel have no states)
    const long long b0 = (long long)(blockIdx.x / blocks) * Rows;
    const int rows = static_cast<int>(min((long long)Rows, p.a.B - b0));
    f2 A[2], h[Rows][2];
    const float* state = p.a.h0 + ((size_t)b0 * D + dd) * N;
    const size_t state_row = (size_t)D * N;
#pragma unroll
    for (int r = 0; r < Rows; ++r)
        if (r < rows) ld_state_once<Vec>(state + r * state_row, n0, N, h[r]);
    ld_state(p.a.A + (size_t)dd * N, n0, N, p.vec_state, A);
    Pack<DT, 4> rB[Rows], rC[Rows];
    const Walk fB = Walk::of<DT>(p.a.Bm, b0 * p.a.B_batch + group * p.a.B_group + n0, p.a.B_batch, 1);
    const Walk fC = Walk::of<DT>(p.a.Cm, b0 * p.a.C_batch + group * p.a.C_group + n0, p.a.C_batch, 1);
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        const int valid = r < rows ? min(4, N - n0) : 0;
        rB[r] = fB.load<DT, Vec>(r, valid);
        rC[r] = fC.load<DT, Vec>(r, valid);
    }
    // this lane's sequence of the Rows
    const int mine = scatter_at<Rows, NL>(lane, 1);
    const long long b = b0 + min(mine, rows - 1);
    const float x = ld_elem(p.a.x, b * p.a.x_batch + dd, DT), skip = p.a.skip ? p.a.skip[dd] : 0.f;
    float dt = ld_elem(p.a.dt, b * p.a.dt_batch + dd, DT), z = 0.f;
    if (p.a.z) z = ld_elem(p.a.z, b * p.a.z_batch + dd, DT);
    if (p.a.dt_bias) dt += p.a.dt_bias[dd];
    if (p.a.softplus) {
        float unused;
        f2_unpack(softplus_pair(f2_dup(dt)), dt, unused);
    }
    A[0] = f2_mul(A[0], f2_dup(kLog2e));
    A[1] = f2_mul(A[1], f2_dup(kLog2e));
    float y[Rows];
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        int from = lane & ~(NL - 1);                           // the lane that has sequence r
#pragma unroll
        for (int l = 0; l < Rows; ++l)
            if (scatter_at<Rows, NL>(l, 1) == r) from |= l;
        const f2 d2 = f2_dup(Rows == 1 ? dt : __shfl_sync(0xffffffffu, dt, from));
        const f2 u2 = f2_dup(Rows == 1 ? dt * x : __shfl_sync(0xffffffffu, dt * x, from));
        f2 B[2], C[2];
        unpack_pairs<DT>(rB[r], B);
        unpack_pairs<DT>(rC[r], C);
#pragma unroll
        for (int i = 0; i < 2; ++i) h[r][i] = f2_fma(ex2_pair(f2_mul(d2, A[i])), h[r][i], f2_mul(u2, B[i]));
        y[r] = f2_sum(f2_fma(C[1], h[r][1], f2_mul(C[0], h[r][0])));
    }
    scatter_sum<Rows, NL>(y, lane, 1);
    if (d >= D) return;
    float* to = p.a.ht + ((size_t)b0 * D + d) * N;
#pragma unroll
    for (int r = 0; r < Rows; ++r)
        if (r < rows) st_state_once<Vec>(to + r * state_row, n0, N, h[r]);
    if (nl < Rows && mine < rows) {
        float v = fmaf(skip, x, y[0]);
        if (p.a.z) v *= z * sigmoid_of(z);
        st_elem(p.a.y, b * D + d, DT, v);
    }
}

int check_grid(long long blocks) {
    return blocks > 0x7fffffffLL ? fail(HDLA_ERR_UNSUPPORTED, "selective_scan: %lld blocks", blocks) : HDLA_OK;
}

}  // namespace

// ------------------------------------------------------------------------------------------ plans
int scan_lanes(int N) {
    int nl = 2;
    while (4 * nl < N) nl *= 2;
    return nl;
}

// Channels a lane, and segments.  Resident on an SM are four blocks forward with one channel a lane, five with two (and of the maps),
// three backward, and about so many hide the latencies.
// Two channels a lane are cheaper in shared-memory cycles than one, one channel a lane gives twice the blocks.  Cutting rows
// runs the recurrence once more for the maps, and pays only where too few blocks would be left.  Measured at N = 16, 8 rows of
// 2048 channels, T = 4096.  Forward: one channel, whole rows (512 blocks) 573 us; two channels, whole rows (256 blocks) 729 us;
// two channels, 16 segments 434 + 286 us for the maps.  Backward (two channels): whole rows 2070 us, 7 segments (4.04 rounds of
// resident blocks) 1584 + 365 us, 8 segments (4.6 rounds) 1485 + 368 us, 12 segments 1489 + 365 us.  One row of 2048
// channels, T = 65536, forward: 32 segments 1527 us, 64 segments 1389 us.  So rows are cut into segments of 64 tokens or more
// until there are thirteen blocks an SM.
ScanPlan scan_plan(const HdlaScanArgs& a, bool backward) {
    const int nl = scan_lanes(a.N), dg = a.D / a.G, sms = sm_count();
    ScanPlan r{};
    auto blocks = [&](int ct) {
        r.ct = ct;
        const int ch = kScanWarps * (32 / nl) * ct;
        r.tiles = (dg + ch - 1) / ch;
        return (long long)a.B * a.G * r.tiles;
    };
    long long n, cut = 1;
    if (backward) {
        n = blocks(nl == 2 || nl == 32 ? 1 : 2);
        if (n < 2.5 * sms) cut = (13LL * sms + n - 1) / n;
    } else if ((n = blocks(2)) < 3.5 * sms && (n = blocks(1)) < 2LL * sms) {
        n = blocks(2);
        cut = (13LL * sms + n - 1) / n;
    }
    const long long most = (a.T + 63) / 64;
    if (cut > most) cut = most;
    r.seg = static_cast<int>(((a.T + cut - 1) / cut + 15) / 16 * 16);
    r.n_seg = (a.T + r.seg - 1) / r.seg;
    return r;
}
// Tiles of channels that keep shares of dB and dC of their own: all, unless those shares would take over 1 GiB (many states
// make narrow tiles); then as many as 1 GiB holds, one at least.  The tiles take turns, a launch after another, and add to the
// shares of those before them.
int scan_slots(const HdlaScanArgs& a, const ScanPlan& r) {
    const size_t each = (size_t)a.B * a.T * a.G * 8 * scan_lanes(a.N) * sizeof(float), most = (size_t(1) << 30) / each;
    return most >= (size_t)r.tiles ? r.tiles : most < 1 ? 1 : (int)most;
}
ScanWork scan_work(const HdlaScanArgs& a, const ScanPlan& r, bool backward) {
    const size_t np = 4 * (size_t)scan_lanes(a.N), rows = (size_t)a.B * r.n_seg, D = a.D;
    ScanWork w{};
    auto take = [&](size_t floats) { const size_t at = w.total; w.total += up256(floats * sizeof(float)); return at; };
    if (r.n_seg > 1) { w.map_h = take(rows * D * np); w.map_d = take(rows * D); }
    if (backward) {
        w.bc = take((size_t)scan_slots(a, r) * a.B * a.T * a.G * 2 * np);
        w.a = take(rows * D * np);
        w.v = take(rows * 2 * D);
    }
    return w;
}
bool scan_vec(const HdlaScanArgs& a) {
    const int bytes = a.dtype == HDLA_F32 ? 16 : 8;              // of four channels or states
    if (a.N % 4 || reinterpret_cast<uintptr_t>(a.Bm) % bytes || reinterpret_cast<uintptr_t>(a.Cm) % bytes) return false;
    for (int64_t st : {a.B_batch, a.B_token, a.B_group, a.C_batch, a.C_token, a.C_group})
        if (st % 4) return false;
    for (int64_t st : {a.x_batch, a.x_token, a.dt_batch, a.dt_token})
        if (st % 4) return false;
    if (a.z && (a.z_batch % 4 || a.z_token % 4)) return false;
    for (const void* q : {a.x, a.dt, a.z, (const void*)a.y, a.dy, (const void*)a.dx, (const void*)a.ddt, (const void*)a.dz})
        if (reinterpret_cast<uintptr_t>(q) % bytes) return false;
    return (a.D / a.G) % 4 == 0;
}
ScanP scan_params(const HdlaScanArgs& a, const ScanPlan& r, const ScanWork& at, unsigned char* ws) {
    ScanP p{};
    p.a = a;
    p.Dg = a.D / a.G;
    p.tiles = r.tiles; p.tile_count = r.tiles; p.seg = r.seg; p.n_seg = r.n_seg;
    auto part = [&](size_t o) { return reinterpret_cast<float*>(ws + o); };
    p.map_h = part(at.map_h); p.map_d = part(at.map_d); p.part_bc = part(at.bc); p.part_a = part(at.a); p.part_v = part(at.v);
    p.vec_state = a.N % 4 == 0;
    for (const void* q : {(const void*)a.A, (const void*)a.h0, (const void*)a.ht, (const void*)a.dht, (const void*)a.dh0})
        p.vec_state = p.vec_state && aligned16(q);
    return p;
}

// ------------------------------------------------------------------------------------------ launches
size_t selective_scan_checkpoint_bytes(const HdlaScanArgs& a) {
    return (size_t)a.B * ((a.T + kCheckpoint - 1) / kCheckpoint) * a.D * 4 * scan_lanes(a.N) * sizeof(float);
}
size_t selective_scan_workspace(const HdlaScanArgs& a, bool backward) { return scan_work(a, scan_plan(a, backward), backward).total; }

int selective_scan_fwd(const HdlaScanArgs& a, unsigned char* ws, cudaStream_t st) {
    const ScanPlan r = scan_plan(a, false);
    const ScanP p = scan_params(a, r, scan_work(a, r, false), ws);
    const long long blocks = (long long)a.G * r.tiles * a.B;
    if (int rc = check_grid(blocks * r.n_seg)) return rc;
    for (int maps = r.n_seg > 1 ? 1 : 0; maps >= 0; --maps) {
        const unsigned grid = static_cast<unsigned>(blocks * (r.n_seg - maps));
        with_type(a.dtype, scan_vec(a), [&](auto dt, auto vec) {
            with_lanes(scan_lanes(a.N), [&](auto nl) {
                if (maps) r.ct == 2 ? scan_fwd_kernel<dt, vec, nl, 2, true><<<grid, kScanThreads, 0, st>>>(p)
                                    : scan_fwd_kernel<dt, vec, nl, 1, true><<<grid, kScanThreads, 0, st>>>(p);
                else r.ct == 2 ? scan_fwd_kernel<dt, vec, nl, 2, false><<<grid, kScanThreads, 0, st>>>(p)
                               : scan_fwd_kernel<dt, vec, nl, 1, false><<<grid, kScanThreads, 0, st>>>(p);
            });
        });
        HDLA_CHECK_LAUNCH(maps ? "scan_fwd_maps_kernel" : "scan_fwd_kernel");
    }
    return HDLA_OK;
}

int selective_scan_step(const HdlaScanArgs& a, cudaStream_t st) {
    ScanPlan r{};
    r.tiles = 1; r.n_seg = 1;
    const ScanP p = scan_params(a, r, ScanWork{}, nullptr);
    const int nl = scan_lanes(a.N);
    const long long columns = (a.D + 128 / nl - 1) / (128 / nl);
    const int rows = nl == 2 ? 2 : 4;
    const bool many = columns * ((a.B + rows - 1) / rows) >= 8LL * sm_count();     // several sequences a thread where enough blocks are left
    const long long grid = columns * (many ? (a.B + rows - 1) / rows : a.B);
    if (int rc = check_grid(grid)) return rc;
    with_type(a.dtype, scan_vec(a) && p.vec_state, [&](auto dt, auto vec) {
        with_lanes(nl, [&](auto l) {
            if (many) scan_step_kernel<dt, l, l == 2 ? 2 : 4, vec><<<(unsigned)grid, 128, 0, st>>>(p);
            else scan_step_kernel<dt, l, 1, vec><<<(unsigned)grid, 128, 0, st>>>(p);
        });
    });
    HDLA_CHECK_LAUNCH("scan_step_kernel");
    return HDLA_OK;
}

}  // namespace hdla
