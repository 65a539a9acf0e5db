// Gated linear recurrence over token sequences: the LSTM cell without its recurrent product,
//   c_t = s(f_t) c_{t-1} + s(i_t) tanh(g_t),   h_t = s(o_t) tanh(c_t)          (s: the logistic function)
// over gate rows of 4H in the order i, f, g, o, each sample for its own number of steps.  The recurrence is linear in c,
// so a stretch of steps acts on the state it starts from as x -> P x + C with P the product of its forget gates: long
// sequences are cut into chunks that run side by side (summary of every chunk, the chain of the summaries, then the
// chunks themselves from their true starting states), short ones run in one launch.
// The work is bound by HBM (forward: 4 gates read, h written; backward: 4 gates and dh read, 4 gradients written); a
// thread owns a few neighbouring units and walks over time with the next steps' loads in flight.
#include "common.h"
#include "vqa_hip.h"

namespace {

constexpr int SAVE = VQA_GATED_SCAN_SAVE;       // the forward saves the state every SAVE steps; the backward recomputes between
constexpr int BLK = 4;                          // steps whose loads a thread of the forward has in flight

// The hardware's exp2 and reciprocal, 1 ulp each (a division, or the library's exponential, would cost several times as
// many instructions): s(x) is good to 2^-22 relative, tanh x = 1 - 2 / (1 + e^2x) to 2^-22 absolute; both reach their
// limits without overflow (1 / inf = 0).
__device__ __forceinline__ float sigm(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }
__device__ __forceinline__ float tanh_(float x) { return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.8853900817779268f * x)); }

// V neighbouring values in storage form
template <typename T, int V> struct Raw;
template <> struct Raw<bf16_t, 4> { u16x4 r; };
template <> struct Raw<bf16_t, 2> { unsigned int r; };
template <> struct Raw<float, 4> { f32x4 r; };
template <> struct Raw<float, 1> { float r; };

template <typename T, int V> __device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
    Raw<T, V> x;
    x.r = *reinterpret_cast<const decltype(x.r)*>(p);
    return x;
}
__device__ __forceinline__ float value(const Raw<bf16_t, 4>& x, int i) { return bf16_to_f32(x.r[i]); }
__device__ __forceinline__ float value(const Raw<bf16_t, 2>& x, int i) {
    return __uint_as_float(i ? x.r & 0xffff0000u : x.r << 16);
}
__device__ __forceinline__ float value(const Raw<float, 4>& x, int i) { return x.r[i]; }
__device__ __forceinline__ float value(const Raw<float, 1>& x, int) { return x.r; }
template <typename T, int V> __device__ __forceinline__ void store_values(T* p, const float (&v)[V]) {
    Raw<T, V> x;
    if constexpr (V == 1) x.r = v[0];
    else if constexpr (sizeof(T) == 4) { for (int i = 0; i < V; ++i) x.r[i] = v[i]; }
    else if constexpr (V == 2) x.r = (unsigned)f32_to_bf16(v[0]) | ((unsigned)f32_to_bf16(v[1]) << 16);
    else { for (int i = 0; i < V; ++i) x.r[i] = f32_to_bf16(v[i]); }
    *reinterpret_cast<decltype(x.r)*>(p) = x.r;
}

// Arguments: gates (B, T) rows of 4H at b * sb + t * st; everything else is contiguous.
template <typename T> struct Args {
    const T* gates; long sb, st; const int32_t* lengths; const float* c0;
    T* h; float* c_last; float* saved;                       // saved[(t / SAVE - 1)][b][u], t = SAVE, 2 SAVE, ...
    const T* dh; const float* dc_last; T* dgates; float* dc0;
    float *prod, *add, *carry;                               // [chunk][b][u]; carry[k]: what chunk k starts from
    int B, T_, H, chunk, nchunk;
};

template <typename T> __device__ __forceinline__ int length_of(const Args<T>& a, int b) {
    return a.lengths ? max(0, min(a.lengths[b], a.T_)) : a.T_;
}

// SUMMARY: prod / add of chunk blockIdx.y (all but the last); otherwise h, the saved states and the last state
template <typename T, int V, bool SUMMARY>
__global__ void __launch_bounds__(256) k_scan_fwd(Args<T> a) {
    const int per = a.H / V;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long)a.B * per) return;
    const int b = (int)(id / per), u = (int)(id % per) * V, k = blockIdx.y;
    const long su = (long)b * a.H + u, plane = (long)a.B * a.H;
    const int len = length_of(a, b), t0 = k * a.chunk, t1 = min(t0 + a.chunk, a.T_), live = min(t1, len);
    float c[V], P[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        P[i] = 1.f;
        if (SUMMARY) c[i] = 0.f;
        else if (k > 0) c[i] = a.carry[k * plane + su + i];
        else c[i] = a.c0 ? a.c0[su + i] : 0.f;
    }
    const T* g = a.gates + (size_t)b * a.sb + u;
    T* h = a.h + ((size_t)b * a.T_) * a.H + u;
    constexpr int NG = SUMMARY ? 3 : 4;
    Raw<T, V> cur[BLK][NG], nxt[BLK][NG];
    auto fetch = [&](int t) {                                // steps past the end request the last one again: no branches
#pragma unroll
        for (int j = 0; j < BLK; ++j)
#pragma unroll
            for (int q = 0; q < NG; ++q) nxt[j][q] = load_raw<T, V>(g + (size_t)min(t + j, live - 1) * a.st + (size_t)q * a.H);
    };
    if (t0 < live) fetch(t0);
    for (int t = t0; t < live; t += BLK) {
#pragma unroll
        for (int j = 0; j < BLK; ++j)
#pragma unroll
            for (int q = 0; q < NG; ++q) cur[j][q] = nxt[j][q];
        if (t + BLK < live) fetch(t + BLK);
#pragma unroll
        for (int j = 0; j < BLK; ++j) {
            if (t + j < live) {
                if (!SUMMARY && a.saved && (t + j) % SAVE == 0 && t + j > 0) {
#pragma unroll
                    for (int i = 0; i < V; ++i) a.saved[((t + j) / SAVE - 1) * plane + su + i] = c[i];
                }
                float hv[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float f = sigm(value(cur[j][1], i));
                    c[i] = f * c[i] + sigm(value(cur[j][0], i)) * tanh_(value(cur[j][2], i));
                    if (SUMMARY) P[i] *= f;
                    else hv[i] = sigm(value(cur[j][NG - 1], i)) * tanh_(c[i]);
                }
                if (!SUMMARY) store_values<T, V>(h + (size_t)(t + j) * a.H, hv);
            }
        }
    }
    if (SUMMARY) {
#pragma unroll
        for (int i = 0; i < V; ++i) { a.prod[k * plane + su + i] = P[i]; a.add[k * plane + su + i] = c[i]; }
        return;
    }
    const float zero[V] = {};
    for (int t = max(live, t0); t < t1; ++t) store_values<T, V>(h + (size_t)t * a.H, zero);     // steps behind the sequence
    // the state after a sample's last step leaves from the chunk that holds it (chunk 0 for an empty sample)
    if (a.c_last && (len > t0 || k == 0) && len <= t1) {
#pragma unroll
        for (int i = 0; i < V; ++i) a.c_last[su + i] = c[i];
    }
}

// carry[k] for k = 1 .. nchunk - 1 (FORWARD: from c0 on; otherwise from dc_last back, carry[k] is what reaches the END of
// chunk k).  A workgroup takes 32 (sample, unit) columns and cuts the chunks into 8 runs: every thread folds its run, the
// runs are chained through LDS, then every thread walks its run again from its true start.
template <typename T, bool FORWARD>
__global__ void __launch_bounds__(256) k_scan_chain(Args<T> a) {
    __shared__ float sp[8][33], sa[8][33];
    const int cx = threadIdx.x & 31, run = threadIdx.x >> 5;
    const long plane = (long)a.B * a.H, col = (long)blockIdx.x * 32 + cx;
    const bool on = col < plane;
    const int n = a.nchunk - 1;                              // maps applied: chunks 0 .. n-1, or n .. 1
    const int per = (n + 7) / 8, lo = min(run * per, n), hi = min(lo + per, n);
    auto at = [&](int s) { return (FORWARD ? s : a.nchunk - 1 - s) * plane + col; };
    float P = 1.f, A = 0.f;
    if (on)
        for (int s0 = lo; s0 < hi; s0 += 8) {
            float p[8], q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (s0 + j < hi) { p[j] = a.prod[at(s0 + j)]; q[j] = a.add[at(s0 + j)]; }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (s0 + j < hi) { A = p[j] * A + q[j]; P *= p[j]; }
        }
    sp[run][cx] = P;
    sa[run][cx] = A;
    __syncthreads();
    if (!on) return;
    const float* first = FORWARD ? a.c0 : a.dc_last;
    float x = first ? first[col] : 0.f;
    if (!FORWARD && run == 0) a.carry[(a.nchunk - 1) * plane + col] = x;
    for (int r = 0; r < run; ++r) x = sp[r][cx] * x + sa[r][cx];
    for (int s0 = lo; s0 < hi; s0 += 8) {
        float p[8], q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (s0 + j < hi) { p[j] = a.prod[at(s0 + j)]; q[j] = a.add[at(s0 + j)]; }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (s0 + j < hi) {
                x = p[j] * x + q[j];
                a.carry[(FORWARD ? s0 + j + 1 : a.nchunk - 2 - s0 - j) * plane + col] = x;
            }
    }
}

// Backward through chunk blockIdx.y, SAVE steps at a time from its end: the states between are recomputed from the saved
// one, then with dct = dh s(o) (1 - tanh^2 c) + dc
//   di = dct tanh(g) s(i)(1-s(i)), df = dct c_{t-1} s(f)(1-s(f)), dg = dct s(i)(1-tanh^2 g), do = dh tanh(c) s(o)(1-s(o)),
//   dc <- dct s(f).
// SUMMARY: only dc's map over the chunk (prod, add), for every chunk but the first.
template <typename T, int V, bool SUMMARY>
__global__ void __launch_bounds__(256) k_scan_bwd(Args<T> a) {
    const int per = a.H / V;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long)a.B * per) return;
    const int b = (int)(id / per), u = (int)(id % per) * V, k = blockIdx.y + (SUMMARY ? 1 : 0);
    const long su = (long)b * a.H + u, plane = (long)a.B * a.H;
    const int len = length_of(a, b), t0 = k * a.chunk, t1 = min(t0 + a.chunk, a.T_), live = min(t1, len);
    const T* g = a.gates + (size_t)b * a.sb + u;
    const T* dh = a.dh ? a.dh + ((size_t)b * a.T_) * a.H + u : nullptr;
    T* dg = a.dgates + ((size_t)b * a.T_) * 4 * a.H + u;
    float dc[V], P[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        P[i] = 1.f;
        if (SUMMARY) dc[i] = 0.f;
        else if (a.nchunk > 1) dc[i] = a.carry[k * plane + su + i];
        else dc[i] = a.dc_last ? a.dc_last[su + i] : 0.f;
    }
    if (!SUMMARY) {
        const float zero[V] = {};
        for (int t = max(live, t0); t < t1; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q) store_values<T, V>(dg + ((size_t)t * 4 + q) * a.H, zero);
    }
    struct { Raw<T, V> r[SAVE][4], d[SAVE]; float c[V]; } cur, nxt;
    auto fetch = [&](int s0) {
#pragma unroll
        for (int j = 0; j < SAVE; ++j) {
            const size_t t = min(s0 + j, live - 1);
#pragma unroll
            for (int q = 0; q < 4; ++q) nxt.r[j][q] = load_raw<T, V>(g + t * a.st + (size_t)q * a.H);
            if (dh) nxt.d[j] = load_raw<T, V>(dh + t * a.H);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (s0 > 0) nxt.c[i] = a.saved[(s0 / SAVE - 1) * plane + su + i];
            else nxt.c[i] = a.c0 ? a.c0[su + i] : 0.f;
        }
    };
    const int s_last = live > t0 ? (live - 1) / SAVE * SAVE : t0 - SAVE;
    if (live > t0) fetch(s_last);
    for (int s0 = s_last; s0 >= t0; s0 -= SAVE) {
        cur = nxt;
        if (s0 > t0) fetch(s0 - SAVE);
        const int n = live - s0;
        float c[SAVE + 1][V], act[SAVE][3][V];               // c[j]: the state before step s0 + j
#pragma unroll
        for (int i = 0; i < V; ++i) c[0][i] = cur.c[i];
#pragma unroll
        for (int j = 0; j < SAVE; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {                    // (steps past the end: computed from the last one's gates, not used)
                act[j][0][i] = sigm(value(cur.r[j][0], i));
                act[j][1][i] = sigm(value(cur.r[j][1], i));
                act[j][2][i] = tanh_(value(cur.r[j][2], i));
                c[j + 1][i] = act[j][1][i] * c[j][i] + act[j][0][i] * act[j][2][i];
            }
#pragma unroll
        for (int j = SAVE - 1; j >= 0; --j)
            if (j < n) {
                float o4[4][V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float si = act[j][0][i], sf = act[j][1][i], tg = act[j][2][i], so = sigm(value(cur.r[j][3], i));
                    const float tc = tanh_(c[j + 1][i]), e = dh ? value(cur.d[j], i) : 0.f;
                    const float dct = e * so * (1.f - tc * tc) + dc[i];
                    o4[0][i] = dct * tg * si * (1.f - si);
                    o4[1][i] = dct * c[j][i] * sf * (1.f - sf);
                    o4[2][i] = dct * si * (1.f - tg * tg);
                    o4[3][i] = e * tc * so * (1.f - so);
                    dc[i] = dct * sf;
                    P[i] *= sf;
                }
                if (!SUMMARY) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) store_values<T, V>(dg + ((size_t)(s0 + j) * 4 + q) * a.H, o4[q]);
                }
            }
    }
    if (SUMMARY) {
#pragma unroll
        for (int i = 0; i < V; ++i) { a.prod[k * plane + su + i] = P[i]; a.add[k * plane + su + i] = dc[i]; }
    } else if (k == 0 && a.dc0) {
#pragma unroll
        for (int i = 0; i < V; ++i) a.dc0[su + i] = dc[i];
    }
}

// Chunks: one when the (sample, unit) pairs alone give every CU work or the sequence is short; otherwise as many as make
// about 2048 waves, at least 4 SAVE steps each.  A multiple of SAVE, so that a chunk starts at a saved state.
int chunk_of(int B, int T_, int H) {
    const long waves = ((long)B * H / 4 + 63) / 64;
    if (waves >= 1024 || T_ <= 8 * SAVE) return (T_ + SAVE - 1) / SAVE * SAVE;
    const long n = (2048 + waves - 1) / waves;
    long c = (T_ + n - 1) / n;
    c = (c + SAVE - 1) / SAVE * SAVE;
    return (int)(c < 4 * SAVE ? 4 * SAVE : c);
}
int chunks_of(int B, int T_, int H) { const int c = chunk_of(B, T_, H); return (T_ + c - 1) / c; }

template <typename T> void plan(Args<T>& a, float* ws) {
    a.chunk = chunk_of(a.B, a.T_, a.H);
    a.nchunk = chunks_of(a.B, a.T_, a.H);
    const size_t n = (size_t)a.nchunk * a.B * a.H;
    a.prod = ws; a.add = ws + n; a.carry = ws + 2 * n;
}

template <typename T, int V> int fwd(Args<T> a, hipStream_t stream) {
    const dim3 grid((unsigned)(((long)a.B * (a.H / V) + 255) / 256), (unsigned)a.nchunk);
    if (a.nchunk > 1) {
        k_scan_fwd<T, V, true><<<dim3(grid.x, grid.y - 1), 256, 0, stream>>>(a);
        k_scan_chain<T, true><<<(unsigned)(((long)a.B * a.H + 31) / 32), 256, 0, stream>>>(a);
    }
    k_scan_fwd<T, V, false><<<grid, 256, 0, stream>>>(a);
    return vqa_check_launch("vqa_gated_scan_fwd");
}
template <typename T, int V> int bwd(Args<T> a, hipStream_t stream) {
    const dim3 grid((unsigned)(((long)a.B * (a.H / V) + 255) / 256), (unsigned)a.nchunk);
    if (a.nchunk > 1) {
        k_scan_bwd<T, V, true><<<dim3(grid.x, grid.y - 1), 256, 0, stream>>>(a);
        k_scan_chain<T, false><<<(unsigned)(((long)a.B * a.H + 31) / 32), 256, 0, stream>>>(a);
    }
    k_scan_bwd<T, V, false><<<grid, 256, 0, stream>>>(a);
    return vqa_check_launch("vqa_gated_scan_bwd");
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

#define SCAN_COMMON(fn)                                                                                                \
    VQA_REQUIRE(dtype == VQA_F32 || dtype == VQA_BF16, fn ": dtype must be VQA_F32 or VQA_BF16");                      \
    VQA_REQUIRE(B > 0 && T > 0 && H > 0 && H % 8 == 0, fn ": B, T and H must be positive, H a multiple of 8");         \
    VQA_REQUIRE((long)B * H <= (1L << 30) && T <= VQA_GATED_SCAN_MAX_T, fn ": B * H <= 2^30 and T <= 2^20");           \
    VQA_REQUIRE(gates && aligned16(gates) && st >= 4 * (long)H && st % 8 == 0 && sb % 8 == 0 && (B == 1 || sb >= 0),   \
                fn ": gate rows must be 16-byte aligned rows of 4 H, strides multiples of 8");                         \
    VQA_REQUIRE(aligned16(c0) && aligned16(workspace), fn ": states and workspace must be 16-byte aligned");           \
    VQA_REQUIRE(workspace || chunks_of(B, T, H) == 1, fn ": this size needs the workspace");

}  // namespace

extern "C" {

size_t vqa_gated_scan_workspace_floats(int B, int T, int H) {
    if (B <= 0 || T <= 0 || H <= 0) return 0;
    const int n = chunks_of(B, T, H);
    return n > 1 ? (size_t)3 * n * B * H : 0;
}

size_t vqa_gated_scan_saved_floats(int B, int T, int H) {
    if (B <= 0 || T <= 0 || H <= 0) return 0;
    return (size_t)((T - 1) / SAVE) * B * H;
}

int vqa_gated_scan_fwd(const void* gates, long sb, long st, const int32_t* lengths, const float* c0, void* h, float* c_last,
                       float* saved, float* workspace, int B, int T, int H, int dtype, hipStream_t stream) {
    SCAN_COMMON("vqa_gated_scan_fwd")
    VQA_REQUIRE(h && aligned16(h) && aligned16(c_last) && aligned16(saved), "vqa_gated_scan_fwd: h is needed, outputs must be 16-byte aligned");
    if (dtype == VQA_BF16) {
        Args<bf16_t> a = {(const bf16_t*)gates, sb, st, lengths, c0, (bf16_t*)h, c_last, saved};
        a.B = B; a.T_ = T; a.H = H;
        plan(a, workspace);
        return fwd<bf16_t, 4>(a, stream);
    }
    Args<float> a = {(const float*)gates, sb, st, lengths, c0, (float*)h, c_last, saved};
    a.B = B; a.T_ = T; a.H = H;
    plan(a, workspace);
    return fwd<float, 4>(a, stream);
}

int vqa_gated_scan_bwd(const void* dh, const float* dc_last, const void* gates, long sb, long st, const int32_t* lengths,
                       const float* c0, const float* saved, void* dgates, float* dc0, float* workspace, int B, int T, int H,
                       int dtype, hipStream_t stream) {
    SCAN_COMMON("vqa_gated_scan_bwd")
    VQA_REQUIRE(dh || dc_last, "vqa_gated_scan_bwd: one of dh, dc_last is needed");
    VQA_REQUIRE(saved || T <= SAVE, "vqa_gated_scan_bwd: the states that the forward saved are needed");
    VQA_REQUIRE(dgates && aligned16(dgates) && aligned16(dh) && aligned16(dc_last) && aligned16(dc0) && aligned16(saved),
                "vqa_gated_scan_bwd: dgates is needed, arrays must be 16-byte aligned");
    if (dtype == VQA_BF16) {
        Args<bf16_t> a = {(const bf16_t*)gates, sb, st, lengths, c0, nullptr, nullptr, (float*)saved,
                          (const bf16_t*)dh, dc_last, (bf16_t*)dgates, dc0};
        a.B = B; a.T_ = T; a.H = H;
        plan(a, workspace);
        return bwd<bf16_t, 2>(a, stream);
    }
    Args<float> a = {(const float*)gates, sb, st, lengths, c0, nullptr, nullptr, (float*)saved,
                     (const float*)dh, dc_last, (float*)dgates, dc0};
    a.B = B; a.T_ = T; a.H = H;
    plan(a, workspace);
    return bwd<float, 1>(a, stream);
}

}  // extern "C"
