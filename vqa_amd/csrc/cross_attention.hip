// Cross attention of token rows to an image's regions, forward and backward.
//
// For one (sample, key head) the Tq x G query rows that share its keys (G query heads per key head) are taken together:
// row m is token m / G, head m % G.  With z = scale q.k the forward keeps a running maximum and sum per row while it
// walks over the keys (p = exp(z - max) is rescaled when the maximum grows), so keys and values are read once and no
// score leaves the registers; the backward recomputes p = exp(z - lse) from the saved log-sum-exp.
//
// All products are 16 x 16 matrix-core tiles.  A FRAGMENT is 16 bytes per lane, 64 bytes of each of 16 matrix rows: lane l
// holds row l % 16, elements (l / 16) * E .. + E (E = 8 bf16 or 4 fp32); it serves as A operand (rows) or B operand
// (columns) alike, and a result tile has column l % 16 and rows 4 (l / 16) + 0..3 in the lane's four registers.  The
// contraction order is free as long as both operands agree, so a result tile P^T (keys x rows) IS the B operand of the next
// product over the same keys: lane l's four (twice four) values are the keys 4 (l / 16) + j (and 16 + 4 (l / 16) + j), and
// the other operand is read from LDS in that key order, transposed by ds_read_b64_tr_b16 for bf16.
#include "common.h"
#include "vqa_hip.h"
#include <math.h>

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

template <typename T> struct Ty;
template <> struct Ty<bf16_t> {
    typedef bf16x8_t frag;                       // contraction over 32
    typedef s16x4_t half;                        // contraction over 16
    static constexpr int E = 8, KC = 32, NS = 2; // elements per lane, contraction length, 16-row tiles per fragment's worth of rows
    static constexpr int PAD = 32;               // LDS pitch = row bytes + PAD: rows fall on different banks for both kinds of reads
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mma_half(half a, half b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0); }
    // four fp32 values rounded to storage: the probabilities and their gradients enter the products as bf16 (2^-9 each, random)
    static __device__ __forceinline__ half pack(f32x4 v) {
        const bf16x4_t b = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        return __builtin_bit_cast(half, b);
    }
    static __device__ __forceinline__ frag join(const half (&h)[2]) {
        const s16x8 v = {h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
        return __builtin_bit_cast(frag, v);
    }
    // four consecutive rows row0 .. + 3 (row0 may differ by 16-lane group) of the 16 columns at col, transposed: lane l gets
    // column l % 16
    static __device__ __forceinline__ half read_t(const char* lds, int pitch, int row0, int col, int li) {
        typedef s16x4_t __attribute__((address_space(3))) * lds_p;
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(lds + (row0 + (li >> 2)) * pitch + (col + 4 * (li & 3)) * 2));
    }
    static __device__ __forceinline__ float dot(frag a, frag b) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += (float)a[i] * (float)b[i];
        return s;
    }
};
template <> struct Ty<float> {
    typedef f32x4 frag;
    typedef f32x4 half;
    static constexpr int E = 4, KC = 16, NS = 1;
    static constexpr int PAD = 16;
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ f32x4 mma_half(half a, half b, f32x4 c) { return mma(a, b, c); }
    static __device__ __forceinline__ half pack(f32x4 v) { return v; }
    static __device__ __forceinline__ frag join(const half (&h)[1]) { return h[0]; }
    static __device__ __forceinline__ half read_t(const char* lds, int pitch, int row0, int col, int li) {
        half v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const float*>(lds + (row0 + i) * pitch + (col + li) * 4);
        return v;
    }
    static __device__ __forceinline__ float dot(frag a, frag b) { return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3]; }
};

// maximum / sum over the four 16-lane groups of a wave, for each l % 16, in all lanes
__device__ __forceinline__ float groups_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// LDS that one wave writes and reads for itself needs no barrier (its LDS operations execute in order), only the
// compiler to keep the order
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename T> struct Args {
    const T *q, *k, *v;
    long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
    const int32_t* kv_len; const uint8_t* mask; long mask_sb;
    T* o; float* lse;                                        // (B, Tq, H, D); (B, H, Tq)
    const T* dout; const float* delta; T *dq, *dk, *dv;      // dout (B, Tq, H, D); delta as lse; dq as o; dk, dv (B, Tk, Hkv, D)
    float* ws;
    int B, Tq, Tk, H, Hkv, G, D, M;                          // M = Tq * G rows per (sample, key head)
    float scale;
    int blocks, row_blocks, nsplit, tiles_split;             // work items; row blocks per pair; key ranges; key tiles per range
};

// Work items are handed out so that neighbours (row blocks of one pair, which read the same keys) run on one XCD and share
// its L2: workgroup i runs on XCD i % 8.
__device__ __forceinline__ int work_item(int blocks) {
    const int per = (blocks + 7) >> 3, w = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    return w;
}

// rows m .. of a pair as fragments: lane's row m (clamped rows give zeros)
template <typename T, int DF>
__device__ __forceinline__ void load_rows(const T* base, long st, long sh, int m, int M, int G, int D, int g, typename Ty<T>::frag (&r)[DF]) {
    typedef Ty<T> Y;
    const T* p = base;
    if (m < M) { const int t = m / G; p += (size_t)t * st + (size_t)(m - t * G) * sh; }
#pragma unroll
    for (int f = 0; f < DF; ++f) {
        const int c = f * Y::KC + g * Y::E;
        typename Y::frag z = {};
        r[f] = m < M && c < D ? *reinterpret_cast<const typename Y::frag*>(p + c) : z;
    }
}

// one tile of keys: which of its 16 x NS keys count (bit key of bits[ns]), and their rows as fragments (zeros for the others:
// what lies in a masked row, NaN included, never enters a product)
template <typename T> struct KeyBits { unsigned b[Ty<T>::NS]; };
template <typename T>
__device__ __forceinline__ KeyBits<T> key_bits(const Args<T>& a, const uint8_t* mask, int len, int key0, int li) {
    KeyBits<T> r;
#pragma unroll
    for (int ns = 0; ns < Ty<T>::NS; ++ns) {
        const int key = key0 + ns * 16 + li;
        const bool on = key < len && (!mask || mask[key] != 0);
        r.b[ns] = (unsigned)(__ballot(on) & 0xffffu);
    }
    return r;
}
template <typename T, int DF>
__device__ __forceinline__ void load_keys(const T* base, long st, const KeyBits<T>& bits, int key0, int D, int li, int g,
                                          typename Ty<T>::frag (&r)[Ty<T>::NS][DF]) {
    typedef Ty<T> Y;
#pragma unroll
    for (int ns = 0; ns < Y::NS; ++ns) {
        const bool on = (bits.b[ns] >> li) & 1;
        const T* p = base + (on ? (size_t)(key0 + ns * 16 + li) * st : 0);
#pragma unroll
        for (int f = 0; f < DF; ++f) {
            const int c = f * Y::KC + g * Y::E;
            typename Y::frag z = {};
            r[ns][f] = on && c < D ? *reinterpret_cast<const typename Y::frag*>(p + c) : z;
        }
    }
}
// fragments of NS x 16 rows to a row-major LDS tile
template <typename T, int DF>
__device__ __forceinline__ void rows_to_lds(char* lds, int pitch, const typename Ty<T>::frag (&r)[Ty<T>::NS][DF], int li, int g) {
#pragma unroll
    for (int ns = 0; ns < Ty<T>::NS; ++ns)
#pragma unroll
        for (int f = 0; f < DF; ++f)
            *reinterpret_cast<typename Ty<T>::frag*>(lds + (ns * 16 + li) * pitch + f * 64 + g * 16) = r[ns][f];
}
// transposed fragment of a KC-row LDS tile: 16 columns at col, contraction over its rows in result-tile order
template <typename T>
__device__ __forceinline__ typename Ty<T>::frag frag_t(const char* lds, int pitch, int col, int li, int g) {
    typename Ty<T>::half h[Ty<T>::NS];
#pragma unroll
    for (int ns = 0; ns < Ty<T>::NS; ++ns) h[ns] = Ty<T>::read_t(lds, pitch, ns * 16 + g * 4, col, li);
    return Ty<T>::join(h);
}

template <typename T> __device__ __forceinline__ void store4(T* p, f32x4 v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = v;
    else {
        u16x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = f32_to_bf16(v[i]);
        *reinterpret_cast<u16x4*>(p) = r;
    }
}

// element offset of row m of pair (b, hk) in a (B, Tq, H, D) array
template <typename T> __device__ __forceinline__ size_t row_at(const Args<T>& a, int b, int hk, int m) {
    const int t = m / a.G;
    return (((size_t)b * a.Tq + t) * a.H + hk * a.G + (m - t * a.G)) * a.D;
}
template <typename T> __device__ __forceinline__ size_t stat_at(const Args<T>& a, int b, int hk, int m) {
    const int t = m / a.G;
    return ((size_t)b * a.H + hk * a.G + (m - t * a.G)) * a.Tq + t;
}

// ---- forward --------------------------------------------------------------------------------
// A workgroup takes 16 MT rows of a pair and one range of key tiles, its four waves every fourth tile: each key is read
// by one wave, straight into fragments; the values pass through the wave's own LDS to be read transposed.  The four
// waves' (maximum, sum, output) are joined at the end, the key ranges by k_xattn_join.
template <typename T, int DF, int MT>
__global__ void __launch_bounds__(256) k_xattn_fwd(Args<T> a) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    constexpr int DP = DF * Y::KC, DT = DP / 16, PITCH = DP * (int)sizeof(T) + Y::PAD, OP = DP + 4;
    constexpr int TILE = Y::KC * PITCH, JOIN = 4 * 16 * OP * 4;
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE > JOIN ? 4 * TILE : JOIN];
    __shared__ float sm[4][16 * MT], sl[4][16 * MT];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int rb = wi % a.row_blocks, ps = wi / a.row_blocks, split = ps % a.nsplit, pair = ps / a.nsplit;
    const int b = pair / a.Hkv, hk = pair % a.Hkv, m0 = rb * 16 * MT;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const T* kb = a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh;
    const T* vb = a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh;
    const int first = split * a.tiles_split, last = min(first + a.tiles_split, (len + Y::KC - 1) / Y::KC);
    char* my = lds + wave * TILE;

    frag q[MT][DF];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        load_rows<T, DF>(a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh, a.q_st, a.q_sh, m0 + mt * 16 + li, a.M, a.G, a.D, g, q[mt]);
    f32x4 o[MT][DT];
    float mx[MT], sum[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        mx[mt] = -INFINITY;
        sum[mt] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float scale2 = a.scale * LOG2E;

    for (int tile = first + wave; tile < last; tile += 4) {
        const int key0 = tile * Y::KC;
        const KeyBits<T> bits = key_bits(a, mask, len, key0, li);
        unsigned any = 0;
#pragma unroll
        for (int ns = 0; ns < Y::NS; ++ns) any |= bits.b[ns];
        if (!any) continue;
        frag k[Y::NS][DF], v[Y::NS][DF];
        load_keys<T, DF>(kb, a.k_st, bits, key0, a.D, li, g, k);
        load_keys<T, DF>(vb, a.v_st, bits, key0, a.D, li, g, v);
        wave_lds_order();
        rows_to_lds<T, DF>(my, PITCH, v, li, g);
        wave_lds_order();
        typename Y::frag p[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            f32x4 s[Y::NS];
            float top = mx[mt];
#pragma unroll
            for (int ns = 0; ns < Y::NS; ++ns) {
                s[ns] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < DF; ++f) s[ns] = Y::mma(k[ns][f], q[mt][f], s[ns]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[ns][r] = (bits.b[ns] >> (g * 4 + r)) & 1 ? s[ns][r] * scale2 : -INFINITY;
                    top = fmaxf(top, s[ns][r]);
                }
            }
            top = groups_max(top);
            const float at = top == -INFINITY ? 0.f : top;
            const float shrink = __builtin_amdgcn_exp2f(mx[mt] - at);
            mx[mt] = top;
            sum[mt] *= shrink;
            typename Y::half h[Y::NS];
#pragma unroll
            for (int ns = 0; ns < Y::NS; ++ns) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[ns][r] = __builtin_amdgcn_exp2f(s[ns][r] - at);
                    sum[mt] += s[ns][r];
                }
                h[ns] = Y::pack(s[ns]);
            }
            p[mt] = Y::join(h);
            if (__any(shrink != 1.f)) {
#pragma unroll
                for (int d = 0; d < DT; ++d) o[mt][d] *= shrink;
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const frag vt = frag_t<T>(my, PITCH, d * 16, li, g);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) o[mt][d] = Y::mma(vt, p[mt], o[mt][d]);
        }
    }

    // join the four waves: row by row the common maximum, then the sums
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const float l = groups_sum(sum[mt]);
        if (g == 0) { sm[wave][mt * 16 + li] = mx[mt]; sl[wave][mt * 16 + li] = l; }
    }
    float* jo = reinterpret_cast<float*>(lds);
    const size_t rows = (size_t)a.B * a.Hkv * a.M;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DT; ++d)
            *reinterpret_cast<f32x4*>(jo + (wave * 16 + li) * OP + d * 16 + g * 4) = o[mt][d];
        __syncthreads();
        for (int c = threadIdx.x; c < 16 * (DP / 4); c += 256) {
            const int r = c / (DP / 4), col = (c % (DP / 4)) * 4, m = m0 + mt * 16 + r;
            if (m >= a.M) continue;
            float w[4], top = sm[0][mt * 16 + r];
#pragma unroll
            for (int i = 1; i < 4; ++i) top = fmaxf(top, sm[i][mt * 16 + r]);
            const float at = top == -INFINITY ? 0.f : top;
            float l = 0.f;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = __builtin_amdgcn_exp2f(sm[i][mt * 16 + r] - at);
                l += w[i] * sl[i][mt * 16 + r];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) v += w[i] * *reinterpret_cast<const f32x4*>(jo + (i * 16 + r) * OP + col);
            if (a.nsplit == 1) {
                const float inv = top == -INFINITY ? 0.f : 1.f / l;
                if (col < a.D) store4(a.o + row_at(a, b, hk, m) + col, v * inv);
                if (col == 0 && a.lse) a.lse[stat_at(a, b, hk, m)] = top == -INFINITY ? -INFINITY : (top + log2f(l)) * LN2;
            } else {
                const size_t at_row = (size_t)split * rows + (size_t)pair * a.M + m;
                if (col < a.D) *reinterpret_cast<f32x4*>(a.ws + at_row * a.D + col) = v;
                if (col == 0) {
                    float* st = a.ws + (size_t)a.nsplit * rows * a.D + at_row * 2;
                    st[0] = top;
                    st[1] = l;
                }
            }
        }
    }
}

// the key ranges of a row joined in range order; one thread per 4 columns
template <typename T>
__global__ void __launch_bounds__(256) k_xattn_join(Args<T> a) {
    const int chunks = a.D / 4;
    const size_t rows = (size_t)a.B * a.Hkv * a.M, id = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= rows * chunks) return;
    const size_t row = id / chunks;
    const int col = (int)(id % chunks) * 4, pair = (int)(row / a.M), m = (int)(row % a.M), b = pair / a.Hkv, hk = pair % a.Hkv;
    const float* st = a.ws + (size_t)a.nsplit * rows * a.D;
    float top = -INFINITY;
    for (int s = 0; s < a.nsplit; ++s) top = fmaxf(top, st[(s * rows + row) * 2]);
    const float at = top == -INFINITY ? 0.f : top;
    float l = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.nsplit; ++s) {
        const float w = __builtin_amdgcn_exp2f(st[(s * rows + row) * 2] - at);
        l += w * st[(s * rows + row) * 2 + 1];
        v += w * *reinterpret_cast<const f32x4*>(a.ws + (s * rows + row) * a.D + col);
    }
    store4(a.o + row_at(a, b, hk, m) + col, v * (top == -INFINITY ? 0.f : 1.f / l));
    if (col == 0 && a.lse) a.lse[stat_at(a, b, hk, m)] = top == -INFINITY ? -INFINITY : (top + log2f(l)) * LN2;
}

// ---- backward -------------------------------------------------------------------------------
// delta[row] = sum_d do * o, one 16-lane group per row
template <typename T>
__global__ void __launch_bounds__(256) k_xattn_delta(Args<T> a, float* delta) {
    const size_t rows = (size_t)a.B * a.Tq * a.H, row = (size_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int li = threadIdx.x & 15;
    if (row >= rows) return;
    float s = 0.f;
    for (int c = li * 4; c < a.D; c += 64) {
        const T *p = a.dout + row * a.D + c, *q = a.o + row * a.D + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) s += to_f32(p[i]) * to_f32(q[i]);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (li == 0) {
        const int h = (int)(row % a.H);
        const size_t bt = row / a.H;
        delta[((bt / a.Tq) * a.H + h) * a.Tq + bt % a.Tq] = s;
    }
}

// Rows of a pair all on the chip (M <= 16 MT): ONE pass over the keys for all three gradients.  Per 16 keys: S (rows x
// keys) and dP = dO V^T as result tiles, P and dS = P (dP - delta) from them; those are the B operands of dV^T = dO^T P and
// dK^T = Q^T dS, whose tiles are complete and leave at once; dS^T, through 16 x 16 of LDS, is the B operand of
// dQ^T += K^T dS^T, which stays in registers and is joined over waves (and key ranges) at the end.
template <typename T, int DF, int MT>
__global__ void __launch_bounds__(256) k_xattn_bwd(Args<T> a) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    typedef typename Y::half half;
    constexpr int DP = DF * Y::KC, DT = DP / 16, PITCH = DP * (int)sizeof(T) + Y::PAD, OP = DP + 4;
    constexpr int TILE = Y::KC * PITCH, JOIN = 4 * 16 * OP * 4, ROWS = MT * 16 * PITCH;
    constexpr int SP = sizeof(T) == 4 ? 80 : 40, DS = Y::KC * SP;      // dS^T: keys x 16 rows
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE > JOIN ? 4 * TILE : JOIN];
    __shared__ __attribute__((aligned(16))) char lq[ROWS], ldo[ROWS], lds_ds[4 * DS];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int split = wi % a.nsplit, pair = wi / a.nsplit, b = pair / a.Hkv, hk = pair % a.Hkv;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const T* kb = a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh;
    const T* vb = a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh;
    const int first = split * a.tiles_split, last = min(first + a.tiles_split, (a.Tk + Y::KC - 1) / Y::KC);
    char *my = lds + wave * TILE, *my_ds = lds_ds + wave * DS;
    const float scale2 = a.scale * LOG2E;

    frag q[MT][DF], d_o[MT][DF];
    float lse[MT][4], delta[MT][4];                          // of rows 4 g + r
    const size_t out0 = row_at(a, b, hk, 0);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = mt * 16 + li;
        load_rows<T, DF>(a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh, a.q_st, a.q_sh, m, a.M, a.G, a.D, g, q[mt]);
        load_rows<T, DF>(a.dout + out0, (long)a.H * a.D, a.D, m, a.M, a.G, a.D, g, d_o[mt]);
        frag o[DF];
        load_rows<T, DF>(a.o + out0, (long)a.H * a.D, a.D, m, a.M, a.G, a.D, g, o);
        float s = 0.f;
#pragma unroll
        for (int f = 0; f < DF; ++f) s += Y::dot(d_o[mt][f], o[f]);
        s = groups_sum(s);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int mr = mt * 16 + g * 4 + r;
            delta[mt][r] = __shfl(s, g * 4 + r, 64);
            lse[mt][r] = mr < a.M ? a.lse[stat_at(a, b, hk, mr)] * LOG2E : INFINITY;
        }
        if (wave == 0) {
#pragma unroll
            for (int f = 0; f < DF; ++f) {
                *reinterpret_cast<frag*>(lq + m * PITCH + f * 64 + g * 16) = q[mt][f];
                *reinterpret_cast<frag*>(ldo + m * PITCH + f * 64 + g * 16) = d_o[mt][f];
            }
        }
    }
    f32x4 dq[MT][DT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int d = 0; d < DT; ++d) dq[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();

    for (int tile = first + wave; tile < last; tile += 4) {
        const int key0 = tile * Y::KC;
        const KeyBits<T> bits = key_bits(a, mask, len, key0, li);
        frag k[Y::NS][DF], v[Y::NS][DF];
        load_keys<T, DF>(kb, a.k_st, bits, key0, a.D, li, g, k);
        load_keys<T, DF>(vb, a.v_st, bits, key0, a.D, li, g, v);
        wave_lds_order();
        rows_to_lds<T, DF>(my, PITCH, k, li, g);
        half dst[MT][Y::NS];
#pragma unroll
        for (int ns = 0; ns < Y::NS; ++ns) {
            half p[MT], ds[MT];
            const bool on = (bits.b[ns] >> li) & 1;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < DF; ++f) {
                    s = Y::mma(q[mt][f], k[ns][f], s);
                    dp = Y::mma(d_o[mt][f], v[ns][f], dp);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[r] = on ? __builtin_amdgcn_exp2f(s[r] * scale2 - lse[mt][r]) : 0.f;
                    dp[r] = on ? s[r] * (dp[r] - delta[mt][r]) : 0.f;
                }
                p[mt] = Y::pack(s);
                ds[mt] = Y::pack(dp);
            }
            f32x4 dk[DT], dv[DT];
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                dk[d] = f32x4{0.f, 0.f, 0.f, 0.f};
                dv[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    dv[d] = Y::mma_half(Y::read_t(ldo, PITCH, mt * 16 + g * 4, d * 16, li), p[mt], dv[d]);
                    dk[d] = Y::mma_half(Y::read_t(lq, PITCH, mt * 16 + g * 4, d * 16, li), ds[mt], dk[d]);
                }
            }
            const int key = key0 + ns * 16 + li;
            if (key < a.Tk) {
                const size_t at = (((size_t)b * a.Tk + key) * a.Hkv + hk) * a.D;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const int c = d * 16 + g * 4;
                    if (c < a.D) {
                        store4(a.dk + at + c, dk[d] * a.scale);
                        store4(a.dv + at + c, dv[d]);
                    }
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {                // dS^T by way of LDS: lane writes rows 4 g + r of key li
                wave_lds_order();
                *reinterpret_cast<half*>(my_ds + li * SP + g * (int)sizeof(half)) = ds[mt];
                wave_lds_order();
                dst[mt][ns] = Y::read_t(my_ds, SP, g * 4, 0, li);
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const frag kt = frag_t<T>(my, PITCH, d * 16, li, g);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) dq[mt][d] = Y::mma(kt, Y::join(dst[mt]), dq[mt][d]);
        }
    }

    float* jo = reinterpret_cast<float*>(lds);
    const size_t rows = (size_t)a.B * a.Hkv * a.M;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DT; ++d)
            *reinterpret_cast<f32x4*>(jo + (wave * 16 + li) * OP + d * 16 + g * 4) = dq[mt][d];
        __syncthreads();
        for (int c = threadIdx.x; c < 16 * (DP / 4); c += 256) {
            const int r = c / (DP / 4), col = (c % (DP / 4)) * 4, m = mt * 16 + r;
            if (m >= a.M || col >= a.D) continue;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) x += *reinterpret_cast<const f32x4*>(jo + (i * 16 + r) * OP + col);
            if (a.nsplit == 1) store4(a.dq + row_at(a, b, hk, m) + col, x * a.scale);
            else *reinterpret_cast<f32x4*>(a.ws + ((size_t)split * rows + (size_t)pair * a.M + m) * a.D + col) = x;
        }
    }
}

// dq's key ranges summed in range order
template <typename T>
__global__ void __launch_bounds__(256) k_xattn_dq_join(Args<T> a) {
    const int chunks = a.D / 4;
    const size_t rows = (size_t)a.B * a.Hkv * a.M, id = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= rows * chunks) return;
    const size_t row = id / chunks;
    const int col = (int)(id % chunks) * 4, pair = (int)(row / a.M), m = (int)(row % a.M);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.nsplit; ++s) v += *reinterpret_cast<const f32x4*>(a.ws + (s * rows + row) * a.D + col);
    store4(a.dq + row_at(a, pair / a.Hkv, pair % a.Hkv, m) + col, v * a.scale);
}

// More rows than fit: the rows' side (dq) as the forward does it, rows in registers, key tiles streamed ...
template <typename T, int DF, int MT>
__global__ void __launch_bounds__(256) k_xattn_bwd_q(Args<T> a) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    constexpr int DP = DF * Y::KC, DT = DP / 16, PITCH = DP * (int)sizeof(T) + Y::PAD, OP = DP + 4;
    constexpr int TILE = Y::KC * PITCH, JOIN = 4 * 16 * OP * 4;
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE > JOIN ? 4 * TILE : JOIN];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int rb = wi % a.row_blocks, pair = wi / a.row_blocks, b = pair / a.Hkv, hk = pair % a.Hkv, m0 = rb * 16 * MT;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const T* kb = a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh;
    const T* vb = a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh;
    const int last = (len + Y::KC - 1) / Y::KC;
    char* my = lds + wave * TILE;
    const float scale2 = a.scale * LOG2E;
    const size_t out0 = row_at(a, b, hk, 0);

    frag q[MT][DF], d_o[MT][DF];
    float lse[MT], delta[MT];                                // of row li
    f32x4 dq[MT][DT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 16 + li;
        load_rows<T, DF>(a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh, a.q_st, a.q_sh, m, a.M, a.G, a.D, g, q[mt]);
        load_rows<T, DF>(a.dout + out0, (long)a.H * a.D, a.D, m, a.M, a.G, a.D, g, d_o[mt]);
        lse[mt] = m < a.M ? a.lse[stat_at(a, b, hk, m)] * LOG2E : INFINITY;
        delta[mt] = m < a.M ? a.delta[stat_at(a, b, hk, m)] : 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) dq[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int tile = wave; tile < last; tile += 4) {
        const int key0 = tile * Y::KC;
        const KeyBits<T> bits = key_bits(a, mask, len, key0, li);
        unsigned any = 0;
#pragma unroll
        for (int ns = 0; ns < Y::NS; ++ns) any |= bits.b[ns];
        if (!any) continue;
        frag k[Y::NS][DF], v[Y::NS][DF];
        load_keys<T, DF>(kb, a.k_st, bits, key0, a.D, li, g, k);
        load_keys<T, DF>(vb, a.v_st, bits, key0, a.D, li, g, v);
        wave_lds_order();
        rows_to_lds<T, DF>(my, PITCH, k, li, g);
        wave_lds_order();
        frag ds[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            typename Y::half h[Y::NS];
#pragma unroll
            for (int ns = 0; ns < Y::NS; ++ns) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < DF; ++f) {
                    s = Y::mma(k[ns][f], q[mt][f], s);
                    dp = Y::mma(v[ns][f], d_o[mt][f], dp);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool on = (bits.b[ns] >> (g * 4 + r)) & 1;
                    const float p = on ? __builtin_amdgcn_exp2f(s[r] * scale2 - lse[mt]) : 0.f;
                    dp[r] = on ? p * (dp[r] - delta[mt]) : 0.f;
                }
                h[ns] = Y::pack(dp);
            }
            ds[mt] = Y::join(h);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const frag kt = frag_t<T>(my, PITCH, d * 16, li, g);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) dq[mt][d] = Y::mma(kt, ds[mt], dq[mt][d]);
        }
    }
    float* jo = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DT; ++d)
            *reinterpret_cast<f32x4*>(jo + (wave * 16 + li) * OP + d * 16 + g * 4) = dq[mt][d];
        __syncthreads();
        for (int c = threadIdx.x; c < 16 * (DP / 4); c += 256) {
            const int r = c / (DP / 4), col = (c % (DP / 4)) * 4, m = m0 + mt * 16 + r;
            if (m >= a.M || col >= a.D) continue;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) x += *reinterpret_cast<const f32x4*>(jo + (i * 16 + r) * OP + col);
            store4(a.dq + row_at(a, b, hk, m) + col, x * a.scale);
        }
    }
}

// ... and the keys' side (dk, dv): a wave keeps NS x 16 keys, their rows and both gradients in registers while the
// workgroup streams the rows through LDS, KC at a time.
template <typename T, int DF>
__global__ void __launch_bounds__(256) k_xattn_bwd_kv(Args<T> a) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    typedef typename Y::half half;
    constexpr int DP = DF * Y::KC, DT = DP / 16, PITCH = DP * (int)sizeof(T) + Y::PAD, TILE = Y::KC * PITCH;
    __shared__ __attribute__((aligned(16))) char lq[TILE], ldo[TILE];
    __shared__ __attribute__((aligned(16))) float l_lse[Y::KC], l_delta[Y::KC];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int kblocks = a.row_blocks, kbk = wi % kblocks, pair = wi / kblocks, b = pair / a.Hkv, hk = pair % a.Hkv;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const int key0 = (kbk * 4 + wave) * Y::KC;
    const float scale2 = a.scale * LOG2E;
    const size_t out0 = row_at(a, b, hk, 0);
    const T* qb = a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh;
    const T* dob = a.dout + out0;

    const KeyBits<T> bits = key_bits(a, mask, len, key0, li);
    frag k[Y::NS][DF], v[Y::NS][DF];
    load_keys<T, DF>(a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh, a.k_st, bits, key0, a.D, li, g, k);
    load_keys<T, DF>(a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh, a.v_st, bits, key0, a.D, li, g, v);
    f32x4 dk[Y::NS][DT], dv[Y::NS][DT];
#pragma unroll
    for (int ns = 0; ns < Y::NS; ++ns)
#pragma unroll
        for (int d = 0; d < DT; ++d) dk[ns][d] = dv[ns][d] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int wg_any = __syncthreads_or((int)(bits.b[0] | bits.b[Y::NS - 1]));
    if (wg_any) {
        for (int m0 = 0; m0 < a.M; m0 += Y::KC) {
            __syncthreads();
            // KC rows of q and dO, 16 bytes per thread at a time
            constexpr int CH = DP / Y::E;
            for (int c = threadIdx.x; c < Y::KC * CH; c += 256) {
                const int r = c / CH, col = (c % CH) * Y::E, m = m0 + r, t = m / a.G, hh = m - t * a.G;
                frag x = {}, y = {};
                if (m < a.M && col < a.D) {
                    x = *reinterpret_cast<const frag*>(qb + (size_t)t * a.q_st + (size_t)hh * a.q_sh + col);
                    y = *reinterpret_cast<const frag*>(dob + ((size_t)t * a.H + hh) * a.D + col);
                }
                *reinterpret_cast<frag*>(lq + r * PITCH + col * (int)sizeof(T)) = x;
                *reinterpret_cast<frag*>(ldo + r * PITCH + col * (int)sizeof(T)) = y;
            }
            if (threadIdx.x < Y::KC) {
                const int m = m0 + threadIdx.x;
                l_lse[threadIdx.x] = m < a.M ? a.lse[stat_at(a, b, hk, m)] * LOG2E : INFINITY;
                l_delta[threadIdx.x] = m < a.M ? a.delta[stat_at(a, b, hk, m)] : 0.f;
            }
            __syncthreads();
            half p[Y::NS][Y::NS], ds[Y::NS][Y::NS];          // [key tile][row tile]
#pragma unroll
            for (int qs = 0; qs < Y::NS; ++qs) {
                f32x4 s[Y::NS], dp[Y::NS];
#pragma unroll
                for (int ns = 0; ns < Y::NS; ++ns) s[ns] = dp[ns] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < DF; ++f) {
                    const frag qf = *reinterpret_cast<const frag*>(lq + (qs * 16 + li) * PITCH + f * 64 + g * 16);
                    const frag df = *reinterpret_cast<const frag*>(ldo + (qs * 16 + li) * PITCH + f * 64 + g * 16);
#pragma unroll
                    for (int ns = 0; ns < Y::NS; ++ns) {
                        s[ns] = Y::mma(qf, k[ns][f], s[ns]);
                        dp[ns] = Y::mma(df, v[ns][f], dp[ns]);
                    }
                }
                const f32x4 ls = *reinterpret_cast<const f32x4*>(l_lse + qs * 16 + g * 4);
                const f32x4 de = *reinterpret_cast<const f32x4*>(l_delta + qs * 16 + g * 4);
#pragma unroll
                for (int ns = 0; ns < Y::NS; ++ns) {
                    const bool on = (bits.b[ns] >> li) & 1;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[ns][r] = on ? __builtin_amdgcn_exp2f(s[ns][r] * scale2 - ls[r]) : 0.f;
                        dp[ns][r] = on ? s[ns][r] * (dp[ns][r] - de[r]) : 0.f;
                    }
                    p[ns][qs] = Y::pack(s[ns]);
                    ds[ns][qs] = Y::pack(dp[ns]);
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const frag dot_ = frag_t<T>(ldo, PITCH, d * 16, li, g), qt = frag_t<T>(lq, PITCH, d * 16, li, g);
#pragma unroll
                for (int ns = 0; ns < Y::NS; ++ns) {
                    dv[ns][d] = Y::mma(dot_, Y::join(p[ns]), dv[ns][d]);
                    dk[ns][d] = Y::mma(qt, Y::join(ds[ns]), dk[ns][d]);
                }
            }
        }
    }
#pragma unroll
    for (int ns = 0; ns < Y::NS; ++ns) {
        const int key = key0 + ns * 16 + li;
        if (key >= a.Tk) continue;
        const size_t at = (((size_t)b * a.Tk + key) * a.Hkv + hk) * a.D;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int c = d * 16 + g * 4;
            if (c < a.D) {
                store4(a.dk + at + c, dk[ns][d] * a.scale);
                store4(a.dv + at + c, dv[ns][d]);
            }
        }
    }
}

// ---- host -----------------------------------------------------------------------------------
int key_tile(int dtype) { return dtype == VQA_BF16 ? 32 : 16; }

// 16-row tiles a workgroup of the forward takes: all of a pair's rows up to 64 (each further tile re-reads the keys from
// the caches, not from registers); fp32 holds half as many
int row_tiles(long M, int dtype) {
    const int most = dtype == VQA_BF16 ? 4 : 2;
    int mt = 1;
    while (mt < most && 16L * mt < M) mt *= 2;
    return mt;
}
// Key ranges: one when the work items fill the chip; otherwise as many as bring 1024 of them, of at least 8 key tiles each
// (two per wave), and at most 32 (the join reads them one after the other).
int key_splits(long items, int Tk, int dtype) {
    const int tiles = (Tk + key_tile(dtype) - 1) / key_tile(dtype);
    if (items >= 512 || tiles < 16) return 1;
    long n = (1024 + items - 1) / items;
    if (n > tiles / 8) n = tiles / 8;
    if (n > 32) n = 32;
    const int per = (int)((tiles + n - 1) / n);
    return (tiles + per - 1) / per;                          // no empty range
}
bool one_pass(long M) { return M <= 32; }                    // the backward that keeps all rows of a pair on the chip

int fwd_splits(int B, int Tq, int Tk, int H, int Hkv, int dtype) {
    const long M = (long)Tq * (H / Hkv), mt = row_tiles(M, dtype);
    return key_splits((long)B * Hkv * ((M + 16 * mt - 1) / (16 * mt)), Tk, dtype);
}
int bwd_splits(int B, int Tq, int Tk, int H, int Hkv, int dtype) { return key_splits((long)B * Hkv, Tk, dtype); }

template <typename T, int DF, int MT> void launch_fwd(const Args<T>& a, hipStream_t s) {
    k_xattn_fwd<T, DF, MT><<<8 * ((a.blocks + 7) / 8), 256, 0, s>>>(a);
}
template <typename T, int DF> void launch_fwd_mt(const Args<T>& a, int mt, hipStream_t s) {
    if (mt == 1) launch_fwd<T, DF, 1>(a, s);
    else if (mt == 2) launch_fwd<T, DF, 2>(a, s);
    else if constexpr (sizeof(T) == 2) launch_fwd<T, DF, 4>(a, s);
}
template <typename T, int DF> void launch_bwd(const Args<T>& a, hipStream_t s) {
    const int grid = 8 * ((a.blocks + 7) / 8);
    if (a.M <= 16) k_xattn_bwd<T, DF, 1><<<grid, 256, 0, s>>>(a);
    else k_xattn_bwd<T, DF, 2><<<grid, 256, 0, s>>>(a);
}
template <typename T, int DF> void launch_bwd_two(Args<T> a, hipStream_t s) {
    constexpr int MT = 2;
    const long pairs = (long)a.B * a.Hkv;
    a.row_blocks = (a.M + 16 * MT - 1) / (16 * MT);
    a.blocks = (int)(pairs * a.row_blocks);
    k_xattn_bwd_q<T, DF, MT><<<8 * ((a.blocks + 7) / 8), 256, 0, s>>>(a);
    a.row_blocks = (a.Tk + 4 * Ty<T>::KC - 1) / (4 * Ty<T>::KC);
    a.blocks = (int)(pairs * a.row_blocks);
    k_xattn_bwd_kv<T, DF><<<8 * ((a.blocks + 7) / 8), 256, 0, s>>>(a);
}

// f<DF> with the number of fragments a row of D takes
#define BY_WIDTH(T, D, call)                                                                   \
    do {                                                                                       \
        if constexpr (sizeof(T) == 2) {                                                        \
            switch (((D) + 31) / 32) {                                                         \
                case 1: { constexpr int DF = 1; call; break; }                                 \
                case 2: { constexpr int DF = 2; call; break; }                                 \
                case 3: { constexpr int DF = 3; call; break; }                                 \
                default: { constexpr int DF = 4; call; break; }                                \
            }                                                                                  \
        } else {                                                                               \
            switch (((D) + 31) / 32) {                                                         \
                case 1: { constexpr int DF = 2; call; break; }                                 \
                case 2: { constexpr int DF = 4; call; break; }                                 \
                case 3: { constexpr int DF = 6; call; break; }                                 \
                default: { constexpr int DF = 8; call; break; }                                \
            }                                                                                  \
        }                                                                                      \
    } while (0)

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool view_ok(const VqaAttnView& v) { return v.data && aligned16(v.data) && v.sb % 8 == 0 && v.st % 8 == 0 && v.sh % 8 == 0 && v.sb >= 0 && v.st >= 0 && v.sh >= 0; }

template <typename T>
Args<T> args_of(const VqaAttnView& q, const VqaAttnView& k, const VqaAttnView& v, const int32_t* kv_len, const uint8_t* mask,
                long mask_sb, float scale, int B, int Tq, int Tk, int H, int Hkv, int D) {
    Args<T> a = {};
    a.q = (const T*)q.data; a.q_sb = q.sb; a.q_st = q.st; a.q_sh = q.sh;
    a.k = (const T*)k.data; a.k_sb = k.sb; a.k_st = k.st; a.k_sh = k.sh;
    a.v = (const T*)v.data; a.v_sb = v.sb; a.v_st = v.st; a.v_sh = v.sh;
    a.kv_len = kv_len; a.mask = mask; a.mask_sb = mask_sb;
    a.B = B; a.Tq = Tq; a.Tk = Tk; a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.D = D; a.M = Tq * a.G;
    a.scale = scale;
    return a;
}

template <typename T>
int fwd(Args<T> a, int nsplit, int dtype, hipStream_t stream) {
    const int mt = row_tiles(a.M, dtype);
    a.row_blocks = (a.M + 16 * mt - 1) / (16 * mt);
    a.nsplit = nsplit;
    const int tiles = (a.Tk + Ty<T>::KC - 1) / Ty<T>::KC;
    a.tiles_split = (tiles + nsplit - 1) / nsplit;
    a.blocks = a.B * a.Hkv * a.row_blocks * nsplit;
    BY_WIDTH(T, a.D, (launch_fwd_mt<T, DF>(a, mt, stream)));
    int rc = vqa_check_launch("vqa_cross_attn_fwd");
    if (rc || nsplit == 1) return rc;
    const size_t n = (size_t)a.B * a.Hkv * a.M * (a.D / 4);
    k_xattn_join<T><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a);
    return vqa_check_launch("vqa_cross_attn_fwd (join)");
}

template <typename T>
int bwd(Args<T> a, int nsplit, hipStream_t stream) {
    if (one_pass(a.M)) {
        a.nsplit = nsplit;
        const int tiles = (a.Tk + Ty<T>::KC - 1) / Ty<T>::KC;
        a.tiles_split = (tiles + nsplit - 1) / nsplit;
        a.blocks = a.B * a.Hkv * nsplit;
        BY_WIDTH(T, a.D, (launch_bwd<T, DF>(a, stream)));
        int rc = vqa_check_launch("vqa_cross_attn_bwd");
        if (rc || nsplit == 1) return rc;
        const size_t n = (size_t)a.B * a.Hkv * a.M * (a.D / 4);
        k_xattn_dq_join<T><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a);
        return vqa_check_launch("vqa_cross_attn_bwd (join)");
    }
    const size_t rows = (size_t)a.B * a.Tq * a.H;
    k_xattn_delta<T><<<(unsigned)((rows + 15) / 16), 256, 0, stream>>>(a, a.ws);
    a.delta = a.ws;
    BY_WIDTH(T, a.D, (launch_bwd_two<T, DF>(a, stream)));
    return vqa_check_launch("vqa_cross_attn_bwd");
}

bool sizes_ok(int B, int Tq, int Tk, int H, int Hkv, int D, int dtype) {
    return (dtype == VQA_F32 || dtype == VQA_BF16) && B > 0 && Tq > 0 && Tk > 0 && Hkv > 0 && H > 0 && H % Hkv == 0 && D > 0 &&
           D % 8 == 0 && D <= VQA_CROSS_ATTN_MAX_D && (long)B * Tq * H <= (1L << 27) && Tk <= (1 << 24) &&
           (long)B * Hkv * ((Tk + 63) / 64) <= (1L << 28);
}
#define XA_COMMON(fn)                                                                                                          \
    VQA_REQUIRE(sizes_ok(B, Tq, Tk, H, Hkv, D, dtype), fn ": dtype VQA_F32 or VQA_BF16, positive sizes, H a multiple of Hkv, " \
                "D a multiple of 8 up to 128, B * Tq * H <= 2^27, Tk <= 2^24");                                                 \
    VQA_REQUIRE(q && k && v && view_ok(*q) && view_ok(*k) && view_ok(*v),                                                      \
                fn ": q, k, v must be 16-byte aligned with strides that are multiples of 8");                                  \
    VQA_REQUIRE(!mask || B == 1 || mask_sb >= 0, fn ": the mask's stride must not be negative");

}  // namespace

extern "C" {

size_t vqa_cross_attn_fwd_workspace_floats(int B, int Tq, int Tk, int H, int Hkv, int D, int dtype) {
    if (!sizes_ok(B, Tq, Tk, H, Hkv, D, dtype)) return 0;
    const int n = fwd_splits(B, Tq, Tk, H, Hkv, dtype);
    return n > 1 ? (size_t)n * B * Tq * H * (D + 2) : 0;
}
size_t vqa_cross_attn_bwd_workspace_floats(int B, int Tq, int Tk, int H, int Hkv, int D, int dtype) {
    if (!sizes_ok(B, Tq, Tk, H, Hkv, D, dtype)) return 0;
    if (!one_pass((long)Tq * (H / Hkv))) return (size_t)B * Tq * H;
    const int n = bwd_splits(B, Tq, Tk, H, Hkv, dtype);
    return n > 1 ? (size_t)n * B * Tq * H * D : 0;
}

int vqa_cross_attn_fwd(const VqaAttnView* q, const VqaAttnView* k, const VqaAttnView* v, const int32_t* kv_len, const uint8_t* mask,
                       long mask_sb, float scale, void* o, float* lse, float* workspace, int B, int Tq, int Tk, int H, int Hkv,
                       int D, int dtype, hipStream_t stream) {
    XA_COMMON("vqa_cross_attn_fwd")
    const int n = fwd_splits(B, Tq, Tk, H, Hkv, dtype);
    VQA_REQUIRE(o && aligned16(o) && aligned16(workspace) && (workspace || n == 1),
                "vqa_cross_attn_fwd: o must be 16-byte aligned; this size needs the workspace");
    if (dtype == VQA_BF16) {
        Args<bf16_t> a = args_of<bf16_t>(*q, *k, *v, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D);
        a.o = (bf16_t*)o; a.lse = lse; a.ws = workspace;
        return fwd(a, n, dtype, stream);
    }
    Args<float> a = args_of<float>(*q, *k, *v, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D);
    a.o = (float*)o; a.lse = lse; a.ws = workspace;
    return fwd(a, n, dtype, stream);
}

int vqa_cross_attn_bwd(const void* d_o, const VqaAttnView* q, const VqaAttnView* k, const VqaAttnView* v, const void* o,
                       const float* lse, const int32_t* kv_len, const uint8_t* mask, long mask_sb, float scale, void* dq, void* dk,
                       void* dv, float* workspace, int B, int Tq, int Tk, int H, int Hkv, int D, int dtype, hipStream_t stream) {
    XA_COMMON("vqa_cross_attn_bwd")
    const int n = bwd_splits(B, Tq, Tk, H, Hkv, dtype);
    VQA_REQUIRE(d_o && o && lse && dq && dk && dv && aligned16(d_o) && aligned16(o) && aligned16(dq) && aligned16(dk) && aligned16(dv),
                "vqa_cross_attn_bwd: d_o, o, lse, dq, dk, dv are needed, 16-byte aligned");
    VQA_REQUIRE(aligned16(workspace) && (workspace || (n == 1 && one_pass((long)Tq * (H / Hkv)))), "vqa_cross_attn_bwd: this size needs the workspace");
    if (dtype == VQA_BF16) {
        Args<bf16_t> a = args_of<bf16_t>(*q, *k, *v, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D);
        a.dout = (const bf16_t*)d_o; a.o = (bf16_t*)o; a.lse = (float*)lse;
        a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv; a.ws = workspace;
        return bwd(a, n, stream);
    }
    Args<float> a = args_of<float>(*q, *k, *v, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D);
    a.dout = (const float*)d_o; a.o = (float*)o; a.lse = (float*)lse;
    a.dq = (float*)dq; a.dk = (float*)dk; a.dv = (float*)dv; a.ws = workspace;
    return bwd(a, n, stream);
}

}  // extern "C"
