// Gated linear recurrence over token sequences: the LSTM cell without its recurrent product,
//   c_t = s(f_t) c_{t-1} + s(i_t) tanh(g_t),   h_t = s(o_t) tanh(c_t)          (s: the logistic function)
// over gate rows of 4H in the order i, f, g, o, each sample for its own number of steps.  The recurrence is linear in c,
// so a stretch of steps acts on the state it starts from as x -> P x + C with P the product of its forget gates.
// The bound is HBM (forward: 4 gates read, h written; backward: 4 gates and dh read, 4 gradients written), with the
// arithmetic close behind, and the gates are to be read ONCE: a workgroup takes 64 V neighbouring units and a block of 8 steps per wave, every wave
// reads its 8 steps into registers and folds them, the waves' maps are chained through LDS, and every wave then walks its
// steps again from its true starting state, out of registers, while the next block is on its way.  Only where the units of
// all samples together make too few workgroups is time itself cut into chunks for different workgroups; the maps of the
// chunks then take a pass over the gates of their own (with an atomic-free chain between the passes).
// Measured (bf16, medians under the profiler): 256 x 14 steps of 2400 units, ragged, 19 us forward and 34 backward; 1 x 16001
// steps of 2048 units, cut into 251 chunks, 52 (maps) + 72 us forward, 3.8 and 4.6 TB/s, and 87 + 152 us backward, 3.8 and
// 3.9 TB/s, where a large copy reaches 5.1; 7 x 577 steps of 1200 units, fp32, 28 - 32 and 41 - 46 us.  About sixty vector
// instructions a step and unit, ten of them transcendental, keep the vector units busy 97 % of the long forward walk's
// time, 67 - 77 % of its other passes', 51 and 64 % at 256 x 14, 23 and 30 % at 7 x 577.  Sixteen waves to a workgroup (half the blocks) made the backward spill, narrower
// tiles of units with more shares of steps per wave gained nothing.
#include "common.h"
#include "vqa_hip.h"

namespace {

constexpr int SAVE = VQA_GATED_SCAN_SAVE;       // steps of a wave's share; the forward saves the state in front of each
constexpr int MOST_WAVES = 8;

// The hardware's exp2 and reciprocal, 1 ulp each (a division, or the library's exponential, would cost several times as
// many instructions); both functions reach their limits without overflow (1 / inf = 0) and keep their digits: tanh x is good
// to 2^-20 of itself, s(x) to 2^-21 + 2^-24 |x|.
__device__ __forceinline__ float sigm(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }
// tanh x = 1 - 2 / (1 + e^2x) is good to 2^-23 absolute, which is that down to |x| = 0.18.  Below, where the difference would
// leave fewer and fewer digits, x + x^3 g(x^2): the line g through the two Chebyshev points of [0, 0.18^2] of
// (tanh x / x - 1) / x^2 leaves 2^-21.8 of tanh x.  (It costs six instructions in about fifty a step and unit: 256 x 14 steps
// 17.0 -> 19.1 us forward, 30.5 -> 33.3 backward; 1 x 16001 steps 62 -> 72 and 143 -> 152.)
__device__ __forceinline__ float tanh_(float x) {
    const float t = x * x;
    float near = fmaf(x * t, fmaf(0.13160463f, t, -0.33332634f), x);
    float far = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.8853900817779268f * x));
    asm("" : "+v"(near), "+v"(far));                         // (a select: the compiler would branch around one of them)
    return fabsf(x) < 0.18f ? near : far;
}

// V neighbouring values in storage form: 4 bytes per lane in both types
template <typename T> struct Raw;
template <> struct Raw<bf16_t> { static constexpr int V = 2; unsigned int r; };
template <> struct Raw<float> { static constexpr int V = 1; float r; };
template <typename T> __device__ __forceinline__ Raw<T> load_raw(const T* p) {
    Raw<T> x;
    x.r = *reinterpret_cast<const decltype(x.r)*>(p);
    return x;
}
__device__ __forceinline__ float value(const Raw<bf16_t>& x, int i) { return __uint_as_float(i ? x.r & 0xffff0000u : x.r << 16); }
__device__ __forceinline__ float value(const Raw<float>& x, int) { return x.r; }
__device__ __forceinline__ void store_values(bf16_t* p, const float (&v)[2]) {
    *reinterpret_cast<unsigned*>(p) = (unsigned)f32_to_bf16(v[0]) | ((unsigned)f32_to_bf16(v[1]) << 16);
}
__device__ __forceinline__ void store_values(float* p, const float (&v)[1]) { *p = v[0]; }

// Arguments: gates (B, T) rows of 4H at b * sb + t * st; everything else is contiguous.
template <typename T> struct Args {
    const T* gates; long sb, st; const int32_t* lengths; const float* c0;
    T* h; float* c_last; float* saved;                       // saved[t / SAVE][b][u], t = 0, SAVE, ...
    const T* dh; const float* dc_last; T* dgates; float* dc0;
    float *prod, *add, *carry;                               // [chunk][b][u]; carry[k]: what chunk k starts from
    int B, T_, H, chunk, nchunk;
};

template <typename T> __device__ __forceinline__ int length_of(const Args<T>& a, int b) {
    return a.lengths ? max(0, min(a.lengths[b], a.T_)) : a.T_;
}

// The maps (p, q) of the workgroup's waves, chained from `x` on (REVERSE: from the last wave back): the value that reaches
// this wave, and in `x` the value behind the block.  LDS holds two blocks' maps, so one barrier per block is enough.
template <int V, bool REVERSE>
__device__ __forceinline__ void chain(float* lds, int& phase, int wave, int nw, int lane, const float (&p)[V], const float (&q)[V],
                                      float (&x)[V], float (&mine)[V]) {
    float* m = lds + phase * nw * 2 * V * 64;
    phase ^= 1;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        m[((wave * 2 + 0) * V + i) * 64 + lane] = p[i];
        m[((wave * 2 + 1) * V + i) * 64 + lane] = q[i];
    }
    __syncthreads();
    for (int k = 0; k < nw; ++k) {
        const int w = REVERSE ? nw - 1 - k : k;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (w == wave) mine[i] = x[i];
            x[i] = m[((w * 2 + 0) * V + i) * 64 + lane] * x[i] + m[((w * 2 + 1) * V + i) * 64 + lane];
        }
    }
}

// SUMMARY: prod / add of chunk blockIdx.y (all but the last); otherwise h, the last state and, with KEEP, the saved states.
// No load or store of a whole block stands under a branch, so the next block's loads are waited for by count.
// ONE: the chunk is a single block, nothing is requested ahead.
template <typename T, bool SUMMARY, bool KEEP, bool ONE>
__global__ void __launch_bounds__(MOST_WAVES * 64) k_scan_fwd(Args<T> a) {
    constexpr int V = Raw<T>::V, NG = SUMMARY ? 3 : 4;
    extern __shared__ float lds[];                           // two blocks' maps of every wave
    const int nw = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int per = a.H / V, total = a.B * per;
    const int id = min((int)blockIdx.x * 64 + lane, total - 1);            // (lanes past the end repeat the last units)
    const int b = id / per, u = (id - b * per) * V, k = blockIdx.y;
    const long su = (long)b * a.H + u, plane = (long)a.B * a.H;
    const int len = length_of(a, b), t0 = k * a.chunk, t1 = min(t0 + a.chunk, a.T_), live = min(t1, len);
    const T* g = a.gates + (size_t)b * a.sb + u;
    T* h = a.h + ((size_t)b * a.T_) * a.H + u;
    int phase = 0;
    float x[V], Pall[V];                                     // the state in front of the block; SUMMARY: the chunk's map
#pragma unroll
    for (int i = 0; i < V; ++i) {
        Pall[i] = 1.f;
        if (SUMMARY) x[i] = 0.f;
        else if (k > 0) x[i] = a.carry[k * plane + su + i];
        else x[i] = a.c0 ? a.c0[su + i] : 0.f;
    }
    Raw<T> nxt[SAVE][NG];
    auto fetch = [&](int t) {                                // steps behind the sequence request its last one
#pragma unroll
        for (int j = 0; j < SAVE; ++j) {
            const T* row = g + (size_t)max(min(t + j, live - 1), 0) * a.st;
#pragma unroll
            for (int q = 0; q < NG; ++q) nxt[j][q] = load_raw(row + (size_t)q * a.H);
        }
    };
    auto block = [&](int tb, bool whole) {
        const int t = tb + wave * SAVE;
        float f[SAVE][V], z[SAVE][V], so[SAVE][V], P[V], C[V], c[V];
#pragma unroll
        for (int i = 0; i < V; ++i) { P[i] = 1.f; C[i] = 0.f; }
#pragma unroll
        for (int j = 0; j < SAVE; ++j) {
            const bool on = t + j < live;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                f[j][i] = on ? sigm(value(nxt[j][1], i)) : 1.f;
                z[j][i] = on ? sigm(value(nxt[j][0], i)) * tanh_(value(nxt[j][2], i)) : 0.f;
                if (!SUMMARY) so[j][i] = on ? sigm(value(nxt[j][NG - 1], i)) : 0.f;
                C[i] = f[j][i] * C[i] + z[j][i];
                P[i] *= f[j][i];
            }
        }
        if (whole && !ONE) fetch(t + nw * SAVE);
        chain<V, false>(lds, phase, wave, nw, lane, P, C, x, c);
        if (SUMMARY) {
            // (the product of the block's forget gates: the chain applied to 1 without its added terms)
            const float* m = lds + (phase ^ 1) * nw * 2 * V * 64;
            for (int w = 0; w < nw; ++w)
#pragma unroll
                for (int i = 0; i < V; ++i) Pall[i] *= m[((w * 2) * V + i) * 64 + lane];
            return;
        }
        if (KEEP && (whole || t < t1)) {
#pragma unroll
            for (int i = 0; i < V; ++i) a.saved[(t / SAVE) * plane + su + i] = c[i];
        }
#pragma unroll
        for (int j = 0; j < SAVE; ++j) {
            float hv[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                c[i] = f[j][i] * c[i] + z[j][i];
                hv[i] = t + j < live ? so[j][i] * tanh_(c[i]) : 0.f;
            }
            if (whole || t + j < t1) store_values(h + (size_t)(t + j) * a.H, hv);
        }
    };
    const int step = nw * SAVE;
    int tb = t0;
    fetch(tb + wave * SAVE);
    if (ONE) block(tb, false);
    else {
        for (; tb + step <= t1; tb += step) block(tb, true);
        if (tb < t1) block(tb, false);
    }
    if (wave > 0) return;
    if (SUMMARY) {
#pragma unroll
        for (int i = 0; i < V; ++i) { a.prod[k * plane + su + i] = Pall[i]; a.add[k * plane + su + i] = x[i]; }
    } else if (a.c_last && (len > t0 || k == 0) && len <= t1) {
        // the state after a sample's last step leaves from the chunk that holds it (chunk 0 for an empty sample)
#pragma unroll
        for (int i = 0; i < V; ++i) a.c_last[su + i] = x[i];
    }
}

// carry[k] for k = 1 .. nchunk - 1 (FORWARD: from c0 on; otherwise from dc_last back, carry[k] is what reaches the END of
// chunk k).  A workgroup takes 32 (sample, unit) columns and cuts the chunks into 32 runs: every thread folds its run, the
// runs are chained through LDS, then every thread walks its run again from its true start.  Latency is all there is to
// it: 32 runs (8 chunks each for 16001 steps, read at once) take 5.4 us, 8 runs of 32 chunks 9.0.
constexpr int RUNS = 32;
template <typename T, bool FORWARD>
__global__ void __launch_bounds__(RUNS * 32) k_scan_chain(Args<T> a) {
    __shared__ float sp[RUNS][33], sa[RUNS][33];
    const int cx = threadIdx.x & 31, run = threadIdx.x >> 5;
    const long plane = (long)a.B * a.H, col = (long)blockIdx.x * 32 + cx;
    const bool on = col < plane;
    const int n = a.nchunk - 1;                              // maps applied: chunks 0 .. n-1, or n .. 1
    const int per = (n + RUNS - 1) / RUNS, lo = min(run * per, n), hi = min(lo + per, n);
    auto at = [&](int s) { return (FORWARD ? s : a.nchunk - 1 - s) * plane + col; };
    float p[8], q[8], P = 1.f, A = 0.f;
    auto fetch = [&](int s0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (s0 + j < hi) { p[j] = a.prod[at(s0 + j)]; q[j] = a.add[at(s0 + j)]; }
    };
    const float* first = FORWARD ? a.c0 : a.dc_last;
    float x = on && first ? first[col] : 0.f;
    if (on)
        for (int s0 = lo; s0 < hi; s0 += 8) {
            fetch(s0);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (s0 + j < hi) { A = p[j] * A + q[j]; P *= p[j]; }
        }
    sp[run][cx] = P;
    sa[run][cx] = A;
    __syncthreads();
    if (!on) return;
    if (!FORWARD && run == 0) a.carry[(a.nchunk - 1) * plane + col] = x;
    for (int r = 0; r < run; ++r) x = sp[r][cx] * x + sa[r][cx];
    for (int s0 = lo; s0 < hi; s0 += 8) {
        if (per > 8) fetch(s0);                              // (otherwise they are still there)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (s0 + j < hi) {
                x = p[j] * x + q[j];
                a.carry[(FORWARD ? s0 + j + 1 : a.nchunk - 2 - s0 - j) * plane + col] = x;
            }
    }
}

// Backward through chunk blockIdx.y, block by block from its end: a wave recomputes its 8 states from the saved one, then
// with dct = dh s(o) (1 - tanh^2 c) + dc
//   di = dct tanh(g) s(i)(1-s(i)), df = dct c_{t-1} s(f)(1-s(f)), dg = dct s(i)(1-tanh^2 g), do = dh tanh(c) s(o)(1-s(o)),
//   dc <- dct s(f):
// dc passes a step as x -> s(f) (x + dh s(o) (1 - tanh^2 c)), so the waves' maps are chained as in the forward.
// SUMMARY: only dc's map over the chunk (prod, add), for every chunk but the first.
template <typename T, bool SUMMARY, bool ONE>
__global__ void __launch_bounds__(MOST_WAVES * 64) k_scan_bwd(Args<T> a) {
    constexpr int V = Raw<T>::V;
    extern __shared__ float lds[];                           // two blocks' maps of every wave
    const int nw = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int per = a.H / V, total = a.B * per;
    const int id = min((int)blockIdx.x * 64 + lane, total - 1);
    const int b = id / per, u = (id - b * per) * V, k = blockIdx.y + (SUMMARY ? 1 : 0);
    const long su = (long)b * a.H + u, plane = (long)a.B * a.H;
    const int len = length_of(a, b), t0 = k * a.chunk, t1 = min(t0 + a.chunk, a.T_), live = min(t1, len);
    const T* g = a.gates + (size_t)b * a.sb + u;
    const T* dh = a.dh ? a.dh + ((size_t)b * a.T_) * a.H + u : g;          // (without dh the gates again, not used)
    const size_t dh_st = a.dh ? a.H : a.st;
    const bool has_dh = a.dh != nullptr;
    T* dg = a.dgates + ((size_t)b * a.T_) * 4 * a.H + u;
    int phase = 0;
    float x[V], Pall[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        Pall[i] = 1.f;
        if (SUMMARY) x[i] = 0.f;
        else if (a.nchunk > 1) x[i] = a.carry[k * plane + su + i];
        else x[i] = a.dc_last ? a.dc_last[su + i] : 0.f;
    }
    struct { Raw<T> r[SAVE][4], d[SAVE]; float c[V]; } nxt;
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < V; ++i) nxt.c[i] = a.saved[(max(min(t, live - 1), 0) / SAVE) * plane + su + i];
#pragma unroll
        for (int j = 0; j < SAVE; ++j) {
            const size_t row = max(min(t + j, live - 1), 0);
#pragma unroll
            for (int q = 0; q < 4; ++q) nxt.r[j][q] = load_raw(g + row * a.st + (size_t)q * a.H);
            nxt.d[j] = load_raw(dh + row * dh_st);
        }
    };
    auto block = [&](int tb, bool whole) {
        const int t = tb + wave * SAVE;
        // per step: s(f), the term added to dc, and what dct is multiplied with for each gate
        float sf[SAVE][V], e[SAVE][V], ki[SAVE][V], kf[SAVE][V], kg[SAVE][V], go[SAVE][V], P[V], D[V], dc[V], c[V];
#pragma unroll
        for (int i = 0; i < V; ++i) { P[i] = 1.f; D[i] = 0.f; c[i] = nxt.c[i]; }
#pragma unroll
        for (int j = 0; j < SAVE; ++j) {
            const bool on = t + j < live;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float si = sigm(value(nxt.r[j][0], i)), s = sigm(value(nxt.r[j][1], i)), tg = tanh_(value(nxt.r[j][2], i));
                const float so = sigm(value(nxt.r[j][3], i)), d = on && has_dh ? value(nxt.d[j], i) : 0.f;
                kf[j][i] = on ? c[i] * s * (1.f - s) : 0.f;
                c[i] = s * c[i] + si * tg;
                const float tc = tanh_(c[i]);
                sf[j][i] = on ? s : 1.f;
                ki[j][i] = on ? tg * si * (1.f - si) : 0.f;
                kg[j][i] = on ? si * (1.f - tg * tg) : 0.f;
                e[j][i] = on ? d * so * (1.f - tc * tc) : 0.f;
                go[j][i] = on ? d * tc * so * (1.f - so) : 0.f;
            }
        }
#pragma unroll
        for (int j = SAVE - 1; j >= 0; --j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                D[i] = sf[j][i] * (e[j][i] + D[i]);
                P[i] *= sf[j][i];
            }
        if (!ONE) fetch(t - nw * SAVE);                      // (in front of the chunk's first block: not used)
        chain<V, true>(lds, phase, wave, nw, lane, P, D, x, dc);
        if (SUMMARY) {
            const float* m = lds + (phase ^ 1) * nw * 2 * V * 64;
            for (int w = 0; w < nw; ++w)
#pragma unroll
                for (int i = 0; i < V; ++i) Pall[i] *= m[((w * 2) * V + i) * 64 + lane];
            return;
        }
#pragma unroll
        for (int j = SAVE - 1; j >= 0; --j) {
            float o4[4][V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float dct = e[j][i] + dc[i];
                o4[0][i] = dct * ki[j][i];
                o4[1][i] = dct * kf[j][i];
                o4[2][i] = dct * kg[j][i];
                o4[3][i] = go[j][i];
                dc[i] = dct * sf[j][i];
            }
            if (whole || t + j < t1) {
#pragma unroll
                for (int q = 0; q < 4; ++q) store_values(dg + ((size_t)(t + j) * 4 + q) * a.H, o4[q]);
            }
        }
    };
    const int step = nw * SAVE;
    int tb = t0 + (t1 - t0 - 1) / step * step;
    fetch(tb + wave * SAVE);
    if (ONE) block(tb, false);
    else {
        if (tb + step > t1) { block(tb, false); tb -= step; }
        for (; tb >= t0; tb -= step) block(tb, true);
    }
    if (wave > 0) return;
    if (SUMMARY) {
#pragma unroll
        for (int i = 0; i < V; ++i) { a.prod[k * plane + su + i] = Pall[i]; a.add[k * plane + su + i] = x[i]; }
    } else if (k == 0 && a.dc0) {
#pragma unroll
        for (int i = 0; i < V; ++i) a.dc0[su + i] = x[i];
    }
}

// Chunks of time: one where the units make 96 workgroups (which read as fast as the card does, one to a CU) or the sequence
// is a few blocks long; otherwise chunks of one block, which a workgroup's eight waves take at once (8 x as many single
// waves that each walk 64 steps: 6 % more for 16001 steps of 2048 units, forward and backward).
int chunk_of(int B, int T_, int H, int dtype) {
    const int v = dtype == VQA_BF16 ? 2 : 1, block = MOST_WAVES * SAVE;
    const long tiles = ((long)B * (H / v) + 63) / 64;
    return tiles >= 96 || T_ <= 4 * block ? (T_ + SAVE - 1) / SAVE * SAVE : block;
}
int chunks_of(int B, int T_, int H, int dtype) { const int c = chunk_of(B, T_, H, dtype); return (T_ + c - 1) / c; }

template <typename T> dim3 plan(Args<T>& a, float* ws, int dtype, int& threads) {
    a.chunk = chunk_of(a.B, a.T_, a.H, dtype);
    a.nchunk = chunks_of(a.B, a.T_, a.H, dtype);
    const size_t n = (size_t)a.nchunk * a.B * a.H;
    a.prod = ws; a.add = ws + n; a.carry = ws + 2 * n;
    const int shares = a.chunk / SAVE;
    threads = 64 * (shares < MOST_WAVES ? shares : MOST_WAVES);
    return dim3((unsigned)(((long)a.B * (a.H / Raw<T>::V) + 63) / 64), (unsigned)a.nchunk);
}

template <typename T> int fwd(Args<T> a, float* ws, int dtype, hipStream_t stream) {
    int threads;
    const dim3 grid = plan(a, ws, dtype, threads);
    const size_t lds = (size_t)threads * 4 * Raw<T>::V * sizeof(float);
    if (a.nchunk > 1) {
        k_scan_fwd<T, true, false, true><<<dim3(grid.x, grid.y - 1), threads, lds, stream>>>(a);
        k_scan_chain<T, true><<<(unsigned)(((long)a.B * a.H + 31) / 32), RUNS * 32, 0, stream>>>(a);
    }
    const bool one = a.chunk <= threads / 64 * SAVE;
    if (a.saved) {
        if (one) k_scan_fwd<T, false, true, true><<<grid, threads, lds, stream>>>(a);
        else k_scan_fwd<T, false, true, false><<<grid, threads, lds, stream>>>(a);
    } else {
        if (one) k_scan_fwd<T, false, false, true><<<grid, threads, lds, stream>>>(a);
        else k_scan_fwd<T, false, false, false><<<grid, threads, lds, stream>>>(a);
    }
    return vqa_check_launch("vqa_gated_scan_fwd");
}
template <typename T> int bwd(Args<T> a, float* ws, int dtype, hipStream_t stream) {
    int threads;
    const dim3 grid = plan(a, ws, dtype, threads);
    const size_t lds = (size_t)threads * 4 * Raw<T>::V * sizeof(float);
    if (a.nchunk > 1) {
        k_scan_bwd<T, true, true><<<dim3(grid.x, grid.y - 1), threads, lds, stream>>>(a);
        k_scan_chain<T, false><<<(unsigned)(((long)a.B * a.H + 31) / 32), RUNS * 32, 0, stream>>>(a);
    }
    if (a.chunk <= threads / 64 * SAVE) k_scan_bwd<T, false, true><<<grid, threads, lds, stream>>>(a);
    else k_scan_bwd<T, false, false><<<grid, threads, lds, stream>>>(a);
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
    VQA_REQUIRE(workspace || chunks_of(B, T, H, dtype) == 1, fn ": this size needs the workspace");

}  // namespace

extern "C" {

size_t vqa_gated_scan_workspace_floats(int B, int T, int H, int dtype) {
    if (B <= 0 || T <= 0 || H <= 0 || H % 8) return 0;
    const int n = chunks_of(B, T, H, dtype);
    return n > 1 ? (size_t)3 * n * B * H : 0;
}

size_t vqa_gated_scan_saved_floats(int B, int T, int H) {
    if (B <= 0 || T <= 0 || H <= 0) return 0;
    return (size_t)((T + SAVE - 1) / SAVE) * B * H;
}

int vqa_gated_scan_fwd(const void* gates, long sb, long st, const int32_t* lengths, const float* c0, void* h, float* c_last,
                       float* saved, float* workspace, int B, int T, int H, int dtype, hipStream_t stream) {
    SCAN_COMMON("vqa_gated_scan_fwd")
    VQA_REQUIRE(h && aligned16(h) && aligned16(c_last) && aligned16(saved), "vqa_gated_scan_fwd: h is needed, outputs must be 16-byte aligned");
    if (dtype == VQA_BF16) {
        Args<bf16_t> a = {(const bf16_t*)gates, sb, st, lengths, c0, (bf16_t*)h, c_last, saved};
        a.B = B; a.T_ = T; a.H = H;
        return fwd(a, workspace, dtype, stream);
    }
    Args<float> a = {(const float*)gates, sb, st, lengths, c0, (float*)h, c_last, saved};
    a.B = B; a.T_ = T; a.H = H;
    return fwd(a, workspace, dtype, stream);
}

int vqa_gated_scan_bwd(const void* dh, const float* dc_last, const void* gates, long sb, long st, const int32_t* lengths,
                       const float* c0, const float* saved, void* dgates, float* dc0, float* workspace, int B, int T, int H,
                       int dtype, hipStream_t stream) {
    SCAN_COMMON("vqa_gated_scan_bwd")
    VQA_REQUIRE(dh || dc_last, "vqa_gated_scan_bwd: one of dh, dc_last is needed");
    VQA_REQUIRE(saved, "vqa_gated_scan_bwd: the states that the forward saved are needed");
    VQA_REQUIRE(dgates && aligned16(dgates) && aligned16(dh) && aligned16(dc_last) && aligned16(dc0) && aligned16(saved),
                "vqa_gated_scan_bwd: dgates is needed, arrays must be 16-byte aligned");
    if (dtype == VQA_BF16) {
        Args<bf16_t> a = {(const bf16_t*)gates, sb, st, lengths, c0, nullptr, nullptr, (float*)saved,
                          (const bf16_t*)dh, dc_last, (bf16_t*)dgates, dc0};
        a.B = B; a.T_ = T; a.H = H;
        return bwd(a, workspace, dtype, stream);
    }
    Args<float> a = {(const float*)gates, sb, st, lengths, c0, nullptr, nullptr, (float*)saved,
                     (const float*)dh, dc_last, (float*)dgates, dc0};
    a.B = B; a.T_ = T; a.H = H;
    return bwd(a, workspace, dtype, stream);
}

}  // extern "C"
