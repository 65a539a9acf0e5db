// The norms before and after a block, its gate and the residual update, in one pass each way:
//   u = f r1,  r1 = 1 / sqrt(mean f^2 + eps)
//   y = rho x + s(gate) w_post u                      (s: the logistic function)
//   h = w_pre n,  n = y r2,  r2 = 1 / sqrt(mean y^2 + eps)
// Everything is bound by HBM: the forward reads x, f and writes y, h, the backward reads x, f, dy, dh and writes dx, df
// (y, n and u are recomputed from x, f and the two saved reciprocal norms of the row).  A row is therefore held in
// registers, 8 columns per thread, from its one load to its one store: a TEAM of threads owns a row, as many as the row
// has 16-byte (bf16) chunks, rounded up to a power of two inside a wave or to whole waves beyond; a workgroup of about
// 256 threads holds several teams and walks over rows, so the fp32 per-column weights stay in registers too (read per
// row they would be more L2 traffic than the row itself); the backward, which needs them beside five operands and three
// running column sums, keeps them in LDS instead (in registers it spilled).  Column sums leave a workgroup as one slab row
// and a second kernel adds the slabs in order.
// Measured (a large copy reaches 5.1 TB/s): 100352 rows of 2048, bf16, a gate row per 196: forward 364 us (4.5 TB/s),
// backward 517 + 15 us (4.8 TB/s); 3570 rows of 2400, fp32, a gate per row: 47 us (3.7 TB/s) and 67 + 5 us (4.1 TB/s);
// 14 rows of 1200: 4.7 us.
#include "common.h"
#include "vqa_hip.h"

namespace {

constexpr int MAX_D = 8192;                  // 1024 threads x 8 columns

// Teams of a workgroup for width D; rows_max: no more teams than this.
struct Team { int lanes, teams; };
Team team_of(int D, long rows_max) {
    const int v = D / 8;
    Team t;
    if (v <= 64) { t.lanes = 1; while (t.lanes < v) t.lanes *= 2; }
    else t.lanes = (v + 63) / 64 * 64;
    t.teams = t.lanes >= 256 ? 1 : 256 / t.lanes;
    if (t.teams > rows_max) t.teams = rows_max < 1 ? 1 : (int)rows_max;
    return t;
}

// Sums of N values over the lanes of each team; `red` holds 2 x N x (waves of the workgroup) floats and `phase`
// alternates, so that one barrier per call is enough: a wave can only be writing buffer p again after the barrier of
// the call in between, which every wave passes after it has read p.  Every thread of the workgroup calls it.
template <int N>
__device__ __forceinline__ void team_sum(float (&v)[N], int lanes, int first_wave, float* red, int& phase) {
    const int inner = lanes < 64 ? lanes : 64;
    for (int o = inner >> 1; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o, 64);
    }
    if (lanes <= 64) return;
    const int nw = blockDim.x >> 6;
    float* r = red + phase * N * nw;
    phase ^= 1;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i * nw + w] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float s = 0.f;
        for (int k = 0; k < (lanes >> 6); ++k) s += r[i * nw + first_wave + k];
        v[i] = s;
    }
}

template <typename T> __device__ __forceinline__ float sigmoid_of(float x) { return fast_sigmoid(x); }
template <> __device__ __forceinline__ float sigmoid_of<float>(float x) { return 1.0f / (1.0f + expf(-x)); }

__device__ __forceinline__ void load_w(const float* w, int col, bool on, float (&v)[8]) {
    if (w && on) Vec8<float>::load(w + col, v);
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 1.0f;
    }
}
// 8 columns of a row as they are stored: the next row's are requested before the current row is worked on
template <typename T> struct Raw8;
template <> struct Raw8<bf16_t> { u16x8 r; };
template <> struct Raw8<float> { f32x4 lo, hi; };
__device__ __forceinline__ void load_row(const bf16_t* p, long row, long ld, int col, bool on, Raw8<bf16_t>& x) {
    const u16x8 z = {};
        x.r = on ? *reinterpret_cast<const u16x8*>(p + (size_t)row * ld + col) : z;
}
__device__ __forceinline__ void load_row(const float* p, long row, long ld, int col, bool on, Raw8<float>& x) {
    const f32x4 z = {};
    const f32x4* q = reinterpret_cast<const f32x4*>(p + (size_t)row * ld + col);
    x.lo = on ? q[0] : z;
    x.hi = on ? q[1] : z;
}
__device__ __forceinline__ void values(const Raw8<bf16_t>& x, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf16_to_f32(x.r[i]);
}
__device__ __forceinline__ void values(const Raw8<float>& x, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = x.lo[i]; v[4 + i] = x.hi[i]; }
}

// WIDE: a team is whole waves, so its row is one number for a wave: rows are then addressed by scalars
template <bool WIDE> __device__ __forceinline__ int team_index(int lanes) {
    const int t = threadIdx.x / lanes;
    return WIDE ? __builtin_amdgcn_readfirstlane(t) : t;
}

template <typename T> struct FwdArgs {
    const T* x; long ldx; const T* f; long ldf; const T* gate; long ldg; int rows_per_gate;
    const float *rho, *w_post, *w_pre; float eps;
    T* y; long ldy; T* h; long ldh; float* stats; int rows, D, lanes, teams;
};

template <typename T, int BOUND, bool WIDE>
__global__ void __launch_bounds__(BOUND) k_norm_gate_fwd(FwdArgs<T> a) {
    __shared__ float red[2 * 16];
    const int team = team_index<WIDE>(a.lanes), tl = threadIdx.x - team * a.lanes;
    const int first_wave = (team * a.lanes) >> 6, col = tl * 8;
    const bool mine = col < a.D;
    const float inv_d = 1.0f / (float)a.D;
    int phase = 0;
    float rho[8], wpo[8], wpr[8];
    load_w(a.rho, col, mine, rho);
    load_w(a.w_post, col, mine, wpo);
    load_w(a.w_pre, col, mine, wpr);
    struct { Raw8<T> x, f, g; } cur, nxt;
    auto fetch = [&](int row) {
        const bool on = mine && row < a.rows;
        load_row(a.x, row, a.ldx, col, on, nxt.x);
        load_row(a.f, row, a.ldf, col, on && a.f, nxt.f);
        load_row(a.gate, a.rows_per_gate == 1 ? row : (int)((unsigned)row / (unsigned)a.rows_per_gate), a.ldg, col, on && a.gate, nxt.g);
    };
    const int step = gridDim.x * a.teams;
    fetch(blockIdx.x * a.teams + team);
    for (int r0 = blockIdx.x * a.teams; r0 < a.rows; r0 += step) {
        const int row = r0 + team;
        const bool on = mine && row < a.rows;
        cur = nxt;
        if (r0 + step < a.rows) fetch(row + step);
        float y[8], f[8], g[8];
        values(cur.x, y);
        float r1 = 1.0f, r2 = 1.0f;
        if (a.f) {
            values(cur.f, f);
            values(cur.g, g);
            float s[1] = {0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) s[0] += f[i] * f[i];
            team_sum(s, a.lanes, first_wave, red, phase);
            r1 = 1.0f / sqrtf(s[0] * inv_d + a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = wpo[i] * (f[i] * r1);
                y[i] = rho[i] * y[i] + (a.gate ? sigmoid_of<T>(g[i]) * u : u);
            }
            if (on && a.y) Vec8<T>::store(a.y + (size_t)row * a.ldy + col, y);
        }
        if (a.h) {
            // the norm of the fp32 y, not of the stored one: one rounding less
            float s[1] = {0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) s[0] += y[i] * y[i];
            if (!on) s[0] = 0.f;
            team_sum(s, a.lanes, first_wave, red, phase);
            r2 = 1.0f / sqrtf(s[0] * inv_d + a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = wpr[i] * (y[i] * r2);
            if (on) Vec8<T>::store(a.h + (size_t)row * a.ldh + col, y);
        }
        if (a.stats && tl == 0 && row < a.rows) { a.stats[2 * (size_t)row] = r1; a.stats[2 * (size_t)row + 1] = r2; }
    }
}

// Backward.  With dn = w_pre dh, s1 = mean(dn n), the gradient at y is dyt = dy + r2 (dn - n s1); dx = rho dyt.  With
// p = s(gate) w_post u the gradient at u is du = dyt s(gate) w_post and df = r1 (du - u s2), s2 = mean(du u) = mean(dyt p)
//    = mean((dy + r2 dn) p) - r2 s1 mean(n p),
// so the three sums of a row are taken in one reduction.  Column sums (drho, dw_post, dw_pre, a shared gate's dgate) stay
// in registers over the rows of a workgroup, are joined over its teams in team order and leave as one fp32 slab per
// workgroup; k_norm_gate_finish adds the slabs in order: no atomics, the same bits every time.
// Rows of a workgroup: unit `blockIdx.x` is `units` consecutive gate groups (sub == 1) or one of `sub` parts of one
// group (sub > 1); a gate of its own per row, or none, counts as groups of any convenient size.
struct Plan { int group, ngroups, sub, units, blocks; bool shared; };

// rows a workgroup walks over: enough to make its slab (12 D bytes) small beside its rows, few enough to fill the chip
Plan plan_of(long rows, int D, bool has_gate, long rows_per_gate) {
    const Team t = team_of(D, has_gate && rows_per_gate > 1 ? rows_per_gate : rows);
    const long waves = (long)t.lanes * t.teams / 64 > 0 ? (long)t.lanes * t.teams / 64 : 1;
    const long want = 256 * (12 / waves > 0 ? 12 / waves : 1);           // workgroups: 256 CUs, up to 12 waves on each
    long per = (rows + want - 1) / want;                                 // rows per workgroup
    if (per < t.teams) per = t.teams;
    Plan p;
    p.shared = has_gate && rows_per_gate > 1;
    p.sub = 1; p.units = 1;
    if (!p.shared) {
        p.group = (int)per;
        p.ngroups = (int)((rows + per - 1) / per);
    } else {
        p.group = (int)rows_per_gate;
        p.ngroups = (int)(rows / rows_per_gate);
        if (per >= p.group) p.units = (int)(per / p.group);
        else {
            // parts of a group: the number whose rounds over the chip cost the least, a part's slab counted as 8 rows
            long best = 0;
            for (int sub = 1; sub <= 256 && sub <= p.group; ++sub) {
                const long cost = (((long)p.ngroups * sub + want - 1) / want) * ((p.group + sub - 1) / sub + 8);
                if (sub == 1 || cost < best) { best = cost; p.sub = sub; }
            }
        }
    }
    p.blocks = p.sub > 1 ? p.ngroups * p.sub : (p.ngroups + p.units - 1) / p.units;
    return p;
}

template <typename T> struct BwdArgs {
    const T* dy; long lddy; const T* dh; long lddh; const T* x; long ldx; const T* f; long ldf;
    const T* gate; long ldg; const float *rho, *w_post, *w_pre, *stats;
    T* dx; long lddx; T* df; long lddf; T* dgate; long lddg;
    float* slab;                 // blocks x 3 x D: dw_pre, drho, dw_post
    float* gate_slab;            // blocks x D (sub > 1)
    int rows, D, lanes, teams; Plan p;
};

// acc summed over the teams in team order, in the threads of team 0
__device__ __forceinline__ void join_teams(float (&acc)[8], int teams, int lanes, int team, int tl, float* lds) {
    if (teams == 1) return;
    __syncthreads();
    if (team > 0) Vec8<float>::store(lds + ((team - 1) * lanes + tl) * 8, acc);
    __syncthreads();
    if (team == 0)
        for (int k = 1; k < teams; ++k) {
            float v[8];
            Vec8<float>::load(lds + ((k - 1) * lanes + tl) * 8, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += v[i];
        }
}

template <typename T, int BOUND, bool WIDE>
__global__ void __launch_bounds__(BOUND) k_norm_gate_bwd(BwdArgs<T> a) {
    __shared__ float red[2 * 3 * 16];
    extern __shared__ __attribute__((aligned(16))) float dyn[];
    float *wl = dyn, *join = dyn + 24 * a.lanes;             // weights; sums on their way to team 0
    const int team = team_index<WIDE>(a.lanes), tl = threadIdx.x - team * a.lanes;
    const int first_wave = (team * a.lanes) >> 6, col = tl * 8;
    const bool mine = col < a.D;
    const float inv_d = 1.0f / (float)a.D;
    int phase = 0;
    // the weights lie in LDS here, [weight][half][lane] x 4: in registers they cost the third wave per SIMD
    if (team == 0) {
        const float* src[3] = {a.rho, a.w_post, a.w_pre};
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            float w[8];
            load_w(src[k], col, mine, w);
            *reinterpret_cast<f32x4*>(wl + ((2 * k) * a.lanes + tl) * 4) = f32x4{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<f32x4*>(wl + ((2 * k + 1) * a.lanes + tl) * 4) = f32x4{w[4], w[5], w[6], w[7]};
        }
    }
    __syncthreads();
    auto weight = [&](int k, float (&w)[8]) {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(wl + ((2 * k) * a.lanes + tl) * 4);
        const f32x4 hi = *reinterpret_cast<const f32x4*>(wl + ((2 * k + 1) * a.lanes + tl) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { w[i] = lo[i]; w[4 + i] = hi[i]; }
    };
    float a_pre[8] = {}, a_rho[8] = {}, a_post[8] = {};
    const int g0 = a.p.sub > 1 ? blockIdx.x / a.p.sub : blockIdx.x * a.p.units;
    const int g1 = a.p.sub > 1 ? g0 + 1 : min(g0 + a.p.units, a.p.ngroups);
    for (int grp = g0; grp < g1; ++grp) {
        int lo = grp * a.p.group, hi = min(lo + a.p.group, a.rows);
        if (a.p.sub > 1) {
            const int part = (a.p.group + a.p.sub - 1) / a.p.sub, k = blockIdx.x % a.p.sub, end = hi;
            lo = min(lo + k * part, end);
            hi = min(lo + part, end);
        }
        float a_gate[8] = {}, sg[8];
        struct { Raw8<T> x, f, dy, dh, g; float r1, r2; } cur, nxt;
        auto fetch = [&](int row) {
            const bool on = mine && row < hi;
            load_row(a.x, row, a.ldx, col, on, nxt.x);
            load_row(a.f, row, a.ldf, col, on && a.f, nxt.f);
            load_row(a.dy, row, a.lddy, col, on && a.dy, nxt.dy);
            load_row(a.dh, row, a.lddh, col, on && a.dh, nxt.dh);
            if (!a.p.shared) load_row(a.gate, row, a.ldg, col, on && a.gate, nxt.g);
            nxt.r1 = row < hi ? a.stats[2 * (size_t)row] : 1.f;
            nxt.r2 = row < hi ? a.stats[2 * (size_t)row + 1] : 1.f;
        };
        fetch(lo + team);
        if (a.p.shared) {
            load_row(a.gate, grp, a.ldg, col, mine, cur.g);
            values(cur.g, sg);
#pragma unroll
            for (int i = 0; i < 8; ++i) sg[i] = sigmoid_of<T>(sg[i]);
        }
        for (int r0 = lo; r0 < hi; r0 += a.teams) {
            const int row = r0 + team;
            const bool on = mine && row < hi;
            cur = nxt;
            if (r0 + a.teams < hi) fetch(row + a.teams);
            float x[8], f[8], dy[8], dn[8], n[8], p[8];
            values(cur.x, x);
            values(cur.f, f);
            values(cur.dy, dy);
            values(cur.dh, dn);
            if (!a.p.shared) {
                values(cur.g, sg);
#pragma unroll
                for (int i = 0; i < 8; ++i) sg[i] = a.gate ? sigmoid_of<T>(sg[i]) : 1.f;
            }
            const float r1 = cur.r1, r2 = cur.r2;
            float s[3] = {0.f, 0.f, 0.f}, rho[8], wpo[8], wpr[8];
            weight(0, rho);
            weight(1, wpo);
            weight(2, wpr);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] *= r1;                                              // u
                p[i] = sg[i] * wpo[i] * f[i];
                n[i] = (a.f ? rho[i] * x[i] + p[i] : x[i]) * r2;
                a_pre[i] += dn[i] * n[i];
                dn[i] *= wpr[i];
                s[0] += dn[i] * n[i];
                s[1] += (dy[i] + r2 * dn[i]) * p[i];
                s[2] += n[i] * p[i];
            }
            team_sum(s, a.lanes, first_wave, red, phase);
            const float s1 = s[0] * inv_d, s2 = s[1] * inv_d - r2 * s1 * (s[2] * inv_d);
            if (on) {
                float dg[8];
                weight(0, rho);
                weight(1, wpo);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float dyt = dy[i] + r2 * (dn[i] - n[i] * s1);
                    a_rho[i] += dyt * x[i];
                    a_post[i] += dyt * f[i] * sg[i];
                    dg[i] = dyt * wpo[i] * f[i];
                    x[i] = a.f ? rho[i] * dyt : dyt;
                    f[i] = r1 * (dyt * sg[i] * wpo[i] - f[i] * s2);
                }
                Vec8<T>::store(a.dx + (size_t)row * a.lddx + col, x);
                if (a.f) Vec8<T>::store(a.df + (size_t)row * a.lddf + col, f);
                if (a.p.shared) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) a_gate[i] += dg[i];
                } else if (a.gate) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) dg[i] *= sg[i] * (1.f - sg[i]);
                    Vec8<T>::store(a.dgate + (size_t)row * a.lddg + col, dg);
                }
            }
        }
        if (a.p.shared) {
            join_teams(a_gate, a.teams, a.lanes, team, tl, join);
            if (team == 0 && mine) {
                if (a.p.sub > 1) Vec8<float>::store(a.gate_slab + (size_t)blockIdx.x * a.D + col, a_gate);
                else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) a_gate[i] *= sg[i] * (1.f - sg[i]);
                    Vec8<T>::store(a.dgate + (size_t)grp * a.lddg + col, a_gate);
                }
            }
        }
    }
    float* slab = a.slab + (size_t)blockIdx.x * 3 * a.D;
    join_teams(a_pre, a.teams, a.lanes, team, tl, join);
    if (team == 0 && mine) Vec8<float>::store(slab + col, a_pre);
    if (a.f) {
        join_teams(a_rho, a.teams, a.lanes, team, tl, join);
        if (team == 0 && mine) Vec8<float>::store(slab + a.D + col, a_rho);
        join_teams(a_post, a.teams, a.lanes, team, tl, join);
        if (team == 0 && mine) Vec8<float>::store(slab + 2 * a.D + col, a_post);
    }
}

// out[0:D], out[D:2D], out[2D:3D] = the slabs summed in order (32 row groups per column, then over the groups); the
// workgroups behind them join the parts of the shared gates' rows.
template <typename T> struct FinishArgs {
    const float* slab; long nslab; float *dw_pre, *drho, *dw_post; int D, cols;     // cols: 3 D or D
    const float* gate_slab; int sub; const T* gate; long ldg; T* dgate; long lddg; int col_blocks;
};
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_gate_finish(FinishArgs<T> a) {
    if ((int)blockIdx.x >= a.col_blocks) {
        const long grp = blockIdx.x - a.col_blocks;
        for (int c = threadIdx.x; c < a.D; c += 1024) {
            float s = 0.f;
            for (int k = 0; k < a.sub; ++k) s += a.gate_slab[((size_t)grp * a.sub + k) * a.D + c];
            const float g = sigmoid_of<T>(to_f32(a.gate[(size_t)grp * a.ldg + c]));
            a.dgate[(size_t)grp * a.lddg + c] = from_f32<T>(s * g * (1.f - g));
        }
        return;
    }
    __shared__ float part[32][33];
    const int cx = threadIdx.x & 31, rg = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
    if (c < a.cols) {
        const float* p = a.slab + c;
        const size_t ld = 3 * (size_t)a.D;
        long m = rg;
        for (; m + 96 < a.nslab; m += 128) {
            s0 += p[m * ld]; s1 += p[(m + 32) * ld]; s2 += p[(m + 64) * ld]; s3 += p[(m + 96) * ld];
        }
        for (; m < a.nslab; m += 32) s0 += p[m * ld];
    }
    part[rg][cx] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    if (rg == 0 && c < a.cols) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += part[k][cx];
        float* out = c < a.D ? a.dw_pre : c < 2 * a.D ? a.drho : a.dw_post;
        if (out) out[c < a.D ? c : c < 2 * a.D ? c - a.D : c - 2 * a.D] = s;
    }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool row_ok(const void* p, long ld, int D) { return aligned16(p) && ld >= D && ld % 8 == 0; }

#define NG_COMMON(fn)                                                                                                       \
    VQA_REQUIRE(dtype == VQA_F32 || dtype == VQA_BF16, fn ": dtype must be VQA_F32 or VQA_BF16");                          \
    VQA_REQUIRE(rows >= 0 && rows <= (1L << 30) && D > 0 && D % 8 == 0 && D <= MAX_D, fn ": D must be a multiple of 8 in [8, 8192], at most 2^30 rows");            \
    VQA_REQUIRE(f || (!gate && !rho && !w_post), fn ": gate, residual_scale and w_post need f");                           \
    VQA_REQUIRE(!gate || (rows_per_gate >= 1 && rows % rows_per_gate == 0), fn ": rows must be whole groups of rows_per_gate"); \
    VQA_REQUIRE(aligned16(rho) && aligned16(w_post) && aligned16(w_pre), fn ": weights must be 16-byte aligned");

template <typename T>
int fwd(const void* x, long ldx, const void* f, long ldf, const void* gate, long ldg, long rows_per_gate, const float* rho,
        const float* w_post, const float* w_pre, float eps, void* y, long ldy, void* h, long ldh, float* stats, long rows,
        int D, hipStream_t stream) {
    const Team t = team_of(D, rows);
    FwdArgs<T> a = {(const T*)x, ldx, (const T*)f, ldf, (const T*)gate, ldg, gate ? (int)rows_per_gate : 1, rho, w_post, w_pre, eps,
                    (T*)y, ldy, (T*)h, ldh, stats, (int)rows, D, t.lanes, t.teams};
    const int threads = t.lanes * t.teams;
    // as many workgroups as are resident at once (five waves per SIMD), each walking over its share of the rows
    const long units = (rows + t.teams - 1) / t.teams, most = 256 * (20 / ((threads + 63) / 64));
    const int grid = (int)(units < most ? units : most);
    if (t.lanes < 64) k_norm_gate_fwd<T, 512, false><<<grid, threads, 0, stream>>>(a);
    else if (threads <= 512) k_norm_gate_fwd<T, 512, true><<<grid, threads, 0, stream>>>(a);
    else k_norm_gate_fwd<T, 1024, true><<<grid, threads, 0, stream>>>(a);
    return vqa_check_launch("vqa_norm_gate_fwd");
}

template <typename T>
int bwd(const void* dy, long lddy, const void* dh, long lddh, const void* x, long ldx, const void* f, long ldf,
        const void* gate, long ldg, long rows_per_gate, const float* rho, const float* w_post, const float* w_pre,
        const float* stats, void* dx, long lddx, void* df, long lddf, void* dgate, long lddg, float* drho, float* dw_post,
        float* dw_pre, float* ws, long rows, int D, hipStream_t stream) {
    const Plan p = plan_of(rows, D, gate != nullptr, rows_per_gate);
    const Team t = team_of(D, p.group);
    BwdArgs<T> a = {(const T*)dy, lddy, (const T*)dh, lddh, (const T*)x, ldx, (const T*)f, ldf, (const T*)gate, ldg, rho, w_post,
                    w_pre, stats, (T*)dx, lddx, (T*)df, lddf, (T*)dgate, lddg, ws, ws + (size_t)p.blocks * 3 * D, (int)rows,
                    D, t.lanes, t.teams, p};
    const int threads = t.lanes * t.teams;
    const size_t lds = (size_t)t.lanes * 96 + (t.teams > 1 ? (size_t)threads * 32 : 0);
    if (t.lanes < 64) k_norm_gate_bwd<T, 512, false><<<p.blocks, threads, lds, stream>>>(a);
    else if (threads <= 512) k_norm_gate_bwd<T, 512, true><<<p.blocks, threads, lds, stream>>>(a);
    else k_norm_gate_bwd<T, 1024, true><<<p.blocks, threads, lds, stream>>>(a);
    int rc = vqa_check_launch("vqa_norm_gate_bwd");
    if (rc) return rc;
    const bool cols = dw_pre || drho || dw_post;
    const int ncols = f ? 3 * D : D, col_blocks = cols ? (ncols + 31) / 32 : 0;
    const long gates = p.sub > 1 ? p.ngroups : 0;
    if (col_blocks + gates == 0) return 0;
    FinishArgs<T> b = {ws, p.blocks, dw_pre, drho, dw_post, D, ncols, a.gate_slab, p.sub, (const T*)gate, ldg, (T*)dgate, lddg, col_blocks};
    k_norm_gate_finish<T><<<(int)(col_blocks + gates), 1024, 0, stream>>>(b);
    return vqa_check_launch("vqa_norm_gate_bwd (finish)");
}

}  // namespace

extern "C" {

int vqa_norm_gate_fwd(const void* x, long ldx, const void* f, long ldf, const void* gate, long ldg, long rows_per_gate,
                      const float* rho, const float* w_post, const float* w_pre, float eps, void* y, long ldy, void* h,
                      long ldh, float* stats, long rows, int D, int dtype, hipStream_t stream) {
    NG_COMMON("vqa_norm_gate_fwd")
    VQA_REQUIRE(eps >= 0.f, "vqa_norm_gate_fwd: eps must not be negative");
    VQA_REQUIRE((y || h) && (f || !y) && (h || !w_pre), "vqa_norm_gate_fwd: y needs f, w_pre needs h, one of y, h is wanted");
    if (rows == 0) return 0;
    VQA_REQUIRE(x && row_ok(x, ldx, D) && (!f || row_ok(f, ldf, D)) && (!gate || row_ok(gate, ldg, D)) &&
                (!y || row_ok(y, ldy, D)) && (!h || row_ok(h, ldh, D)),
                "vqa_norm_gate_fwd: matrices must be 16-byte aligned with leading dimensions >= D, multiples of 8");
    if (dtype == VQA_BF16)
        return fwd<bf16_t>(x, ldx, f, ldf, gate, ldg, rows_per_gate, rho, w_post, w_pre, eps, y, ldy, h, ldh, stats, rows, D, stream);
    return fwd<float>(x, ldx, f, ldf, gate, ldg, rows_per_gate, rho, w_post, w_pre, eps, y, ldy, h, ldh, stats, rows, D, stream);
}

size_t vqa_norm_gate_workspace_floats(long rows, int D, long rows_per_gate) {
    if (rows <= 0 || rows > (1L << 30) || D <= 0 || D % 8 || D > MAX_D || rows_per_gate < 0 || (rows_per_gate > 0 && rows % rows_per_gate)) return 0;
    const Plan p = plan_of(rows, D, rows_per_gate > 0, rows_per_gate);
    return (size_t)p.blocks * 3 * D + (p.sub > 1 ? (size_t)p.blocks * D : 0);
}

int vqa_norm_gate_bwd(const void* dy, long lddy, const void* dh, long lddh, const void* x, long ldx, const void* f, long ldf,
                      const void* gate, long ldg, long rows_per_gate, const float* rho, const float* w_post,
                      const float* w_pre, const float* stats, void* dx, long lddx, void* df, long lddf, void* dgate,
                      long lddg, float* drho, float* dw_post, float* dw_pre, float* workspace, long rows, int D, int dtype,
                      hipStream_t stream) {
    NG_COMMON("vqa_norm_gate_bwd")
    VQA_REQUIRE((dy || dh) && (f || !dy), "vqa_norm_gate_bwd: one of dy, dh is needed, and dy belongs to a y that f made");
    VQA_REQUIRE((!!f == !!df) && (!!gate == !!dgate) && (f || (!drho && !dw_post)), "vqa_norm_gate_bwd: df goes with f, dgate with gate, drho and dw_post need f");
    VQA_REQUIRE(rows > 0, "vqa_norm_gate_bwd: no rows (the gradients of the weights would be left unwritten)");
    VQA_REQUIRE(x && dx && stats && workspace && aligned16(workspace) && row_ok(x, ldx, D) && row_ok(dx, lddx, D) &&
                (!f || (row_ok(f, ldf, D) && row_ok(df, lddf, D))) && (!gate || (row_ok(gate, ldg, D) && row_ok(dgate, lddg, D))) &&
                (!dy || row_ok(dy, lddy, D)) && (!dh || row_ok(dh, lddh, D)),
                "vqa_norm_gate_bwd: matrices must be 16-byte aligned with leading dimensions >= D, multiples of 8");
    if (dtype == VQA_BF16)
        return bwd<bf16_t>(dy, lddy, dh, lddh, x, ldx, f, ldf, gate, ldg, rows_per_gate, rho, w_post, w_pre, stats, dx, lddx, df,
                           lddf, dgate, lddg, drho, dw_post, dw_pre, workspace, rows, D, stream);
    return bwd<float>(dy, lddy, dh, lddh, x, ldx, f, ldf, gate, ldg, rows_per_gate, rho, w_post, w_pre, stats, dx, lddx, df, lddf,
                      dgate, lddg, drho, dw_post, dw_pre, workspace, rows, D, stream);
}

}  // extern "C"
