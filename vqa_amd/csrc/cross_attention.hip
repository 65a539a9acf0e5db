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
//
// With few rows per key head the bound is HBM: K and V are read once (backward: and dK, dV written once).  Measured, bf16:
//   64 x 1 row x 8 key heads of 128 (4 query heads each) on 4096 regions, ragged: 156 us, at the copy rate (5.1 TB/s)
//   256 x 14 on 196 x 15 heads of 80, ragged: forward 62 us, backward 105 us
// with many rows and regions the matrix cores:
//   8 x 509 on 4096 x 8 key heads of 128 (2 each): forward 172 us (790 TFLOP/s), dq 208 us (three products, 990 TFLOP/s),
//   dk and dv 325 us (four products, 840 TFLOP/s), delta 11; a large library product reaches 1180 there
// and fp32 32 x 20 on 576 x 8 heads of 64: 22 and 44 us (medians under the profiler, whose short runs clock lower: these
// kernels take 3 - 12 % less in passes back to back).  The variants, by rules of two_plan(), few(), one_pass(), tiled():
// k_xattn_fwd / k_xattn_bwd stream the keys past up to 64 (32) rows in registers; k_xattn_bwd_q / _bwd_kv for more rows;
// k_xattn_*_tile for more than 64 rows on more than 256 keys; k_xattn_*_few for at most 32 keys.
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
    typedef s16x4_t half;                        // half of one: four values per lane
    static constexpr bool PARTS = true;          // a fp32 factor can be given in two parts
    static constexpr int E = 8, KC = 32, NS = 2; // elements per lane, contraction length, 16-row tiles per fragment's worth of rows
    static constexpr int PAD = 16;               // LDS pitch = row bytes + PAD: rows fall on different banks for both kinds of reads
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    // four fp32 values rounded to storage
    static __device__ __forceinline__ half pack(f32x4 v) {
        const bf16x4_t b = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        return __builtin_bit_cast(half, b);
    }
    // the part of v that pack leaves behind, rounded in its turn: value = pack(v) + rest(v) to 2^-17; of an infinite v
    // nothing is left (inf - inf would make its products NaN)
    static __device__ __forceinline__ half rest(f32x4 v, half h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] -= bf16_to_f32((bf16_t)h[i]);
            v[i] = fabsf(v[i]) < INFINITY ? v[i] : 0.f;
        }
        return pack(v);
    }
    // weights >= 0 in two parts, weight = hi + lo to 2^-16: cut off, not rounded, and lo at least a number that changes
    // nothing, so that both are above 0 where the weight is and their products with an infinite value agree
    static __device__ __forceinline__ void split(f32x4 v, half& hi, half& lo) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned cut = __float_as_uint(v[i]) & 0xffff0000u;
            hi[i] = (short)(cut >> 16);
            v[i] = fmaxf(v[i] - __uint_as_float(cut), 7.888609e-31f);
        }
        lo = pack(v);
    }
    // c + the four values
    static __device__ __forceinline__ float sum(half h, float c) {
        typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
        const bf16x2_t one = {(__bf16)1.f, (__bf16)1.f};
        const bf16x4_t b = __builtin_bit_cast(bf16x4_t, h);
        return __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{b[2], b[3]}, one, __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{b[0], b[1]}, one, c, false), false);
    }
    // product over 16 (contraction), the second factor in its two parts
    static __device__ __forceinline__ f32x4 mma_parts(half a, half hi, half lo, f32x4 c) {
        c = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, lo, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, hi, c, 0, 0, 0);
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
    // sum a (b + c): the two parts of an output are added first, an infinite a times each could be inf - inf
    static __device__ __forceinline__ float dot(frag a, frag b, frag c) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += (float)a[i] * ((float)b[i] + (float)c[i]);
        return s;
    }
};
template <> struct Ty<float> {
    typedef f32x4 frag;
    typedef f32x4 half;
    static constexpr bool PARTS = false;
    static constexpr int E = 4, KC = 16, NS = 1;
    static constexpr int PAD = 16;
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ half pack(f32x4 v) { return v; }
    static __device__ __forceinline__ half rest(f32x4, half) { return f32x4{0.f, 0.f, 0.f, 0.f}; }
    static __device__ __forceinline__ void split(f32x4 v, half& hi, half& lo) { hi = v; lo = f32x4{0.f, 0.f, 0.f, 0.f}; }
    static __device__ __forceinline__ f32x4 mma_parts(half a, half hi, half, f32x4 c) { return mma(a, hi, c); }
    static __device__ __forceinline__ frag join(const half (&h)[1]) { return h[0]; }
    static __device__ __forceinline__ half read_t(const char* lds, int pitch, int row0, int col, int li) {
        half v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const float*>(lds + (row0 + i) * pitch + (col + li) * 4);
        return v;
    }
    static __device__ __forceinline__ float dot(frag a, frag b, frag) { return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3]; }
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

// Waves per SIMD that a kernel of this file is compiled for: two, which leaves it 256 registers and products that add up in
// ordinary ones; with one it gets 512, but the products' sums move to the accumulation registers and back for every use
// (96-wide rows, 64 x 60 on 200 x 8 heads, bf16: dq 23.7 -> 18.6 us, dk / dv 43.8 -> 33.4; fp32 dq 56.7 -> 46.3).  One where
// 256 do not suffice and much of the rest would go to memory (dk / dv's few words cost less; 128-wide: dq 30.6, with two 40.2; 96-wide forward of 64 rows 23 and 46).
template <typename T> constexpr int waves_fwd(int df, int mt) { return sizeof(T) == 2 ? (df * mt > 8 ? 1 : 2) : (df * mt > 12 ? 1 : 2); }
template <typename T> constexpr int waves_bwd(int df, int mt) { return df * (mt + 1) > (sizeof(T) == 2 ? 6 : 8) ? 1 : 2; }
template <typename T> constexpr int waves_bwd_q(int df) { return df > (sizeof(T) == 2 ? 3 : 6) ? 1 : 2; }
template <typename T> constexpr int waves_bwd_few(int df, int nk) { return df * nk > (sizeof(T) == 2 ? 4 : 6) ? 1 : 2; }

template <typename T> struct Args {
    const T *q, *k, *v;
    long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
    const int32_t* kv_len; const uint8_t* mask; long mask_sb;
    T *o, *rest; float* lse;                                 // (B, Tq, H, D): the output, what rounding took from it; (B, H, Tq)
    const T* dout; const float* delta; T *dq, *dk, *dv;      // dout (B, Tq, H, D); delta as lse; dq as o; dk, dv (B, Tk, Hkv, D)
    float* ws;
    int B, Tq, Tk, H, Hkv, G, D, M;                          // M = Tq * G rows per (sample, key head)
    float scale;
    int items, blocks, row_blocks, nsplit, tiles_split;      // work items; workgroups; row blocks per pair; key ranges; key tiles per range
};

// Work items are handed out so that neighbours (row blocks of one pair, which read the same keys) run on one XCD and share
// its L2: workgroup i runs on XCD i % 8.
__device__ __forceinline__ int work_item(int blocks) {
    const int per = (blocks + 7) >> 3, w = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    return w;
}

// rows m .. of a pair as fragments: lane's row m (rows past the last one give zeros; no branches around the loads, see
// KeyTile)
template <typename T, int DF>
__device__ __forceinline__ void load_rows(const T* base, long st, long sh, int m, int M, int G, int D, int g, typename Ty<T>::frag (&r)[DF]) {
    typedef Ty<T> Y;
    const int mc = max(min(m, M - 1), 0), t = mc / G;
    const T* p = base + (size_t)t * st + (size_t)(mc - t * G) * sh;
#pragma unroll
    for (int f = 0; f < DF; ++f) {
        const int c = f * Y::KC + g * Y::E;
        const typename Y::frag x = *reinterpret_cast<const typename Y::frag*>(p + (c < D ? c : 0)), z = {};
        r[f] = m < M && c < D ? x : z;
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

// 16-byte accesses relative to a base that is the same for the whole wave, checked by the hardware: what starts outside
// [base, base + bytes) reads as zero or is not written
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
struct Window {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ Window(const void* base, unsigned bytes) {
        r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00027000);
    }
    __device__ __forceinline__ u32x4 load(unsigned at) const { return __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0); }
    __device__ __forceinline__ void store(unsigned at, u32x4 v) const { __builtin_amdgcn_raw_buffer_store_b128(v, r, (int)at, 0, 0); }
};

// A tile of keys on its way to LDS: neighbouring lanes read neighbouring 16-byte chunks of a row, and the next tile's chunks
// are in flight while the current tile is worked on.  For that no load (and no store in the loop) may stand under a
// branch: the counter that loads are waited for by must be known at compile time, or every wait is for everything in
// flight.  So the hardware checks the bounds, and the rows that do not count are cleared on the way into LDS: what lies
// in them, NaN included, never enters a product.
template <typename T, int NI> struct Spots {                 // lane's chunks: row | chunk << 8 (surplus ones repeat the last)
    int rc[NI];
    __device__ __forceinline__ void init(int lane, int D, int rows) {
        const unsigned per = D / Ty<T>::E, inv = (65536 + per - 1) / per;      // c / per, exact for c < 1024, per <= 32
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const unsigned c = min((unsigned)(i * 64 + lane), per * rows - 1), r = __umul24(c, inv) >> 16;
            rc[i] = (int)(r | (c - __umul24(r, per)) << 8);
        }
    }
    __device__ __forceinline__ unsigned row(int i) const { return rc[i] & 255; }
    __device__ __forceinline__ unsigned col(int i) const { return (rc[i] >> 8) * Ty<T>::E; }
    // (strides are multiples of 8 below 2^25: a product of 24 bits, which takes a quarter of a full one's time)
    __device__ __forceinline__ unsigned at(int i, unsigned st) const { return ((__umul24(row(i), st >> 3) << 3) + col(i)) * (unsigned)sizeof(T); }
};
template <typename T, int DF> struct KeyTile {
    typedef Ty<T> Y;
    static constexpr int NI = DF * Y::KC / 16;
    u32x4 k[NI], v[NI];
    unsigned m[Y::NS];                                       // mask bytes of keys ns * 16 + li
    static __device__ __forceinline__ void rows_of(u32x4 (&r)[NI], const Spots<T, NI>& sp, const T* base, long st, int len, int D, int key0) {
        const int rows = max(min(Y::KC, len - key0), 0);
        const Window w(base + (size_t)key0 * st, rows ? ((rows - 1) * (unsigned)st + D) * (unsigned)sizeof(T) : 0);
#pragma unroll
        for (int i = 0; i < NI; ++i) r[i] = w.load(sp.at(i, (unsigned)st));
    }
    __device__ __forceinline__ void load_k(const Args<T>& a, const Spots<T, NI>& sp, const uint8_t* mask, int len, const T* kb, int key0, int li) {
        // without a mask the bytes come from the keys and do not matter
        const uint8_t* mb = mask ? mask : reinterpret_cast<const uint8_t*>(kb);
#pragma unroll
        for (int ns = 0; ns < Y::NS; ++ns) m[ns] = mb[mask ? min(key0 + ns * 16 + li, a.Tk - 1) : 0];
        rows_of(k, sp, kb, a.k_st, len, a.D, key0);
    }
    __device__ __forceinline__ void load_v(const Args<T>& a, const Spots<T, NI>& sp, int len, const T* vb, int key0) {
        rows_of(v, sp, vb, a.v_st, len, a.D, key0);
    }
    __device__ __forceinline__ void load(const Args<T>& a, const Spots<T, NI>& sp, const uint8_t* mask, int len, const T* kb, const T* vb, int key0, int li) {
        load_k(a, sp, mask, len, kb, key0, li);
        load_v(a, sp, len, vb, key0);
    }
    __device__ __forceinline__ KeyBits<T> bits(bool masked, int len, int key0, int li) const {
        KeyBits<T> b;
#pragma unroll
        for (int ns = 0; ns < Y::NS; ++ns) b.b[ns] = (unsigned)(__ballot(key0 + ns * 16 + li < len && (!masked || m[ns] != 0)) & 0xffffu);
        return b;
    }
    static __device__ __forceinline__ void put(const u32x4 (&r)[NI], const Spots<T, NI>& sp, const KeyBits<T>& bits, char* lds, int pitch) {
        const unsigned on = bits.b[0] | bits.b[Y::NS - 1] << (16 * (Y::NS - 1));
        const u32x4 z = {};
        if (on == (Y::NS == 2 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
            for (int i = 0; i < NI; ++i) *reinterpret_cast<u32x4*>(lds + sp.row(i) * pitch + sp.col(i) * (int)sizeof(T)) = r[i];
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i)
                *reinterpret_cast<u32x4*>(lds + sp.row(i) * pitch + sp.col(i) * (int)sizeof(T)) = (on >> sp.row(i)) & 1 ? r[i] : z;
        }
    }
};
// a wave's part of LDS cleared: the columns between D and the fragments' width stay zero from then on
__device__ __forceinline__ void wave_clear(char* lds, int bytes, int lane) {
    const f32x4 z = {};
    for (int at = lane * 16; at < bytes; at += 1024) *reinterpret_cast<f32x4*>(lds + at) = z;
}
template <typename T> __device__ __forceinline__ typename Ty<T>::frag frag_at(const char* lds, int pitch, int row, int f, int g) {
    return *reinterpret_cast<const typename Ty<T>::frag*>(lds + row * pitch + f * 64 + g * 16);
}
// transposed fragment of a KC-row LDS tile: 16 columns at col, contraction over its rows in result-tile order
template <typename T>
__device__ __forceinline__ typename Ty<T>::frag frag_t(const char* lds, int pitch, int col, int li, int g) {
    typename Ty<T>::half h[Ty<T>::NS];
#pragma unroll
    for (int ns = 0; ns < Ty<T>::NS; ++ns) h[ns] = Ty<T>::read_t(lds, pitch, ns * 16 + g * 4, col, li);
    return Ty<T>::join(h);
}

// the same from a lane's own place (row g * 4 + li / 4, column 4 * (li % 4) of the tile's first 16 rows)
__device__ __forceinline__ bf16x8_t frag_tr(const char* at, int pitch) {
    typedef s16x4_t __attribute__((address_space(3))) * lds_p;
    const s16x4_t h[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)at), __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(at + 16 * pitch))};
    return Ty<bf16_t>::join(h);
}

// a value that all lanes hold, in a scalar register
__device__ __forceinline__ float uniform(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); }

// The forward finds a row's largest score before the scale's product (the exponential takes both in one instruction), which
// needs a positive one: a negative scale turns q's sign, and of a zero the least positive number makes the same weights.
__device__ __forceinline__ float positive_scale(float scale) { return uniform(fmaxf(fabsf(scale) * LOG2E, 1e-37f)); }

// the log-sum-exp of a row from its maximum (powers of two) and its sum of 2^(score - maximum): -inf where nothing counts (an
// empty sum), NaN where the scores are (no maximum either, but a sum that is NaN)
__device__ __forceinline__ float log_sum(float top, float l) { return l == 0.f ? -INFINITY : (top + log2f(l)) * LN2; }

// keeps a uniform branch a branch: the compiler would select, element by element, on every pass
__device__ __forceinline__ void rarely() { asm volatile(""); }

template <typename T> __device__ __forceinline__ void store4(T* p, f32x4 v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = v;
    else {
        u16x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = f32_to_bf16(v[i]);
        *reinterpret_cast<u16x4*>(p) = r;
    }
}

// four outputs, and what their rounding leaves for the backward's delta
template <typename T> __device__ __forceinline__ void store_out(const Args<T>& a, size_t at, f32x4 v) {
    store4(a.o + at, v);
    if constexpr (sizeof(T) == 2) {
        if (a.rest) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] -= bf16_to_f32(f32_to_bf16(v[i]));
                v[i] = fabsf(v[i]) < INFINITY ? v[i] : 0.f;  // (of an infinite output nothing)
            }
            store4(a.rest + at, v);
        }
    }
}

// element offset of pair (b, hk) in a (B, Tq, H, D) array, and the place n of its row m there: n D further on
template <typename T> __device__ __forceinline__ size_t pair_at(const Args<T>& a, int b, int hk) {
    return ((size_t)b * a.Tq * a.H + hk * a.G) * a.D;
}
template <typename T> __device__ __forceinline__ int place_of(const Args<T>& a, int m) {
    const int t = m / a.G;
    return t * a.H + (m - t * a.G);
}
template <typename T> __device__ __forceinline__ size_t row_at(const Args<T>& a, int b, int hk, int m) {
    return pair_at(a, b, hk) + (size_t)place_of(a, m) * a.D;
}
template <typename T> __device__ __forceinline__ size_t stat_at(const Args<T>& a, int b, int hk, int m) {
    const int t = m / a.G;
    return ((size_t)b * a.H + hk * a.G + (m - t * a.G)) * a.Tq + t;
}

// ---- forward --------------------------------------------------------------------------------
// W waves take 16 MT rows of a pair and one range of key tiles, each wave every W-th tile, through LDS of its own: no wave
// waits for another until their (maximum, sum, output) are joined at the end.  The key ranges are joined by k_xattn_join.
// The work is bound by reading the keys; p therefore enters its product in two bf16 parts, so that nothing but the output
// is rounded.
template <typename T, int DF, int MT, int W>
__global__ void __launch_bounds__(256, waves_fwd<T>(DF, MT)) k_xattn_fwd(Args<T> a) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    constexpr int DP = DF * Y::KC, DT = DP / 16, PITCH = DP * (int)sizeof(T) + Y::PAD, OP = DP + 4;
    constexpr int TILE = Y::KC * PITCH, JOIN = 4 * 16 * OP * 4;
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE > JOIN ? 4 * TILE : JOIN];
    __shared__ float sm[4][16 * MT], sl[4][16 * MT];
    __shared__ int places[4 / W][16 * MT];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4, w0 = wave % W;
    const int wi_ = work_item(a.blocks) * (4 / W) + wave / W;
    const bool idle = wi_ >= a.items;                        // an item past the last one: no keys, nothing stored
    const int wi = idle ? 0 : wi_;
    const int rb = wi % a.row_blocks, ps = wi / a.row_blocks, split = ps % a.nsplit, pair = ps / a.nsplit;
    const int b = pair / a.Hkv, hk = pair % a.Hkv, m0 = rb * 16 * MT, M = idle ? 0 : a.M;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const T* kb = a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh;
    const T* vb = a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh;
    const int first = split * a.tiles_split, last = idle ? 0 : min(first + a.tiles_split, (len + Y::KC - 1) / Y::KC);
    char* my = lds + wave * TILE;                            // the keys of a tile, then its values

    frag q[MT][DF];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        load_rows<T, DF>(a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh, a.q_st, a.q_sh, m0 + mt * 16 + li, M, a.G, a.D, g, q[mt]);
    Spots<T, DT> sp;
    sp.init(lane, a.D, Y::KC);
    KeyTile<T, DF> nxt;
    nxt.load(a, sp, mask, len, kb, vb, (first + w0) * Y::KC, li);
    f32x4 o[MT][DT];
    float mx[MT], sum[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        mx[mt] = -INFINITY;
        sum[mt] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float scale2 = positive_scale(a.scale);
    if (a.scale < 0.f) {
        rarely();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int f = 0; f < DF; ++f) q[mt][f] = -q[mt][f];
    }
    const bool spare = a.D <= DP - 16;                       // the last 16 columns are all padding
    if (a.D < DP) wave_clear(my, TILE, lane);

    for (int tile = first + w0; tile < last; tile += W) {
        wave_lds_order();
        const KeyBits<T> bits = nxt.bits(mask != nullptr, len, tile * Y::KC, li);
        nxt.put(nxt.k, sp, bits, my, PITCH);
        wave_lds_order();
        nxt.load_k(a, sp, mask, len, kb, (tile + W) * Y::KC, li);
        f32x4 s[MT][Y::NS];
#pragma unroll
        for (int ns = 0; ns < Y::NS; ++ns) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt][ns] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < DF; ++f) {
                const frag k = frag_at<T>(my, PITCH, ns * 16 + li, f, g);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][ns] = Y::mma(k, q[mt][f], s[mt][ns]);
            }
        }
        wave_lds_order();
        nxt.put(nxt.v, sp, bits, my, PITCH);
        wave_lds_order();
        nxt.load_v(a, sp, len, vb, (tile + W) * Y::KC);
        if ((bits.b[0] & bits.b[Y::NS - 1]) != 0xffffu) {
            rarely();
#pragma unroll
            for (int ns = 0; ns < Y::NS; ++ns)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!((bits.b[ns] >> (g * 4 + r)) & 1))
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) s[mt][ns][r] = -INFINITY;
        }
        frag p[MT], p_lo[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float top = -INFINITY;
#pragma unroll
            for (int ns = 0; ns < Y::NS; ++ns)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, s[mt][ns][r]);
            top = fmaxf(groups_max(top) * scale2, mx[mt]);
            const float at = top == -INFINITY ? 0.f : top;
            const float shrink = __builtin_amdgcn_exp2f(mx[mt] - at);
            mx[mt] = top;
            sum[mt] *= shrink;
            typename Y::half h[Y::NS], lo[Y::NS];
#pragma unroll
            for (int ns = 0; ns < Y::NS; ++ns) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[mt][ns][r] = __builtin_amdgcn_exp2f(s[mt][ns][r] * scale2 - at);
                    sum[mt] += s[mt][ns][r];
                }
                Y::split(s[mt][ns], h[ns], lo[ns]);
            }
            p[mt] = Y::join(h);
            p_lo[mt] = Y::join(lo);
            if (__any(shrink != 1.f)) {
#pragma unroll
                for (int d = 0; d < DT; ++d) o[mt][d] *= shrink;
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if (d == DT - 1 && spare) break;
            const frag vt = frag_t<T>(my, PITCH, d * 16, li, g);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                o[mt][d] = Y::mma(vt, p[mt], o[mt][d]);
                if constexpr (Y::PARTS) o[mt][d] = Y::mma(vt, p_lo[mt], o[mt][d]);
            }
        }
    }

    // join the item's waves: one thread per row finds the common maximum, the sum and what each wave's output counts for
    const size_t rows = (size_t)a.B * a.Hkv * a.M, row0 = (size_t)split * rows + (size_t)pair * a.M + m0;
    const int w1 = wave - w0, it = threadIdx.x % (64 * W);   // the item's first wave; the thread in the item
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const float l = groups_sum(sum[mt]);
        if (g == 0) { sm[wave][mt * 16 + li] = mx[mt]; sl[wave][mt * 16 + li] = l; }
    }
    __syncthreads();
    if (it < 16 * MT) {
        float top = sm[w1][it], l = 0.f, w[W];
#pragma unroll
        for (int i = 1; i < W; ++i) top = fmaxf(top, sm[w1 + i][it]);
        const float at = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            w[i] = __builtin_amdgcn_exp2f(sm[w1 + i][it] - at);
            l += w[i] * sl[w1 + i][it];
        }
        const float inv = a.nsplit > 1 ? 1.f : top == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < W; ++i) sm[w1 + i][it] = w[i] * inv;
        const int m = m0 + it;
        places[wave / W][it] = place_of(a, m);
        if (m < M) {
            if (a.nsplit > 1) {
                float* st = a.ws + ((size_t)a.nsplit * rows * a.D + (row0 + it) * 2);
                st[0] = top;
                st[1] = l;
            } else if (a.lse) a.lse[stat_at(a, b, hk, m)] = log_sum(top, l);
        }
    }
    float* jo = reinterpret_cast<float*>(lds);
    const size_t out0 = pair_at(a, b, hk);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (mt > 0) __syncthreads();
#pragma unroll
        for (int d = 0; d < DT; ++d)
            *reinterpret_cast<f32x4*>(jo + (wave * 16 + li) * OP + d * 16 + g * 4) = o[mt][d];
        __syncthreads();
#pragma unroll 2
        for (int c = it; c < 16 * (DP / 4); c += 64 * W) {
            const int r = c / (DP / 4), col = (c % (DP / 4)) * 4, row = mt * 16 + r;
            if (m0 + row >= M || col >= a.D) continue;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < W; ++i) v += sm[w1 + i][row] * *reinterpret_cast<const f32x4*>(jo + ((w1 + i) * 16 + r) * OP + col);
            if (a.nsplit == 1) store_out(a, out0 + (size_t)places[wave / W][row] * a.D + col, v);
            else *reinterpret_cast<f32x4*>(a.ws + (row0 + row) * a.D + col) = v;
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
    store_out(a, row_at(a, b, hk, m) + col, v * (top == -INFINITY ? 0.f : 1.f / l));
    if (col == 0 && a.lse) a.lse[stat_at(a, b, hk, m)] = log_sum(top, l);
}

// ---- backward -------------------------------------------------------------------------------
// delta[row] = sum_d do * o, one 16-lane group per row; o with what its rounding took (delta is subtracted from dO V^T, and
// where few regions count, or one region most of the weight, little is left of either)
template <typename T>
__global__ void __launch_bounds__(256) k_xattn_delta(Args<T> a, float* delta) {
    const size_t rows = (size_t)a.B * a.Tq * a.H, row = (size_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int li = threadIdx.x & 15;
    if (row >= rows) return;
    float s = 0.f;
    for (int c = li * 8; c < a.D; c += 128) {
        float x[8], y[8], z[8];
        Vec8<T>::load(a.dout + row * a.D + c, x);
        Vec8<T>::load(a.o + row * a.D + c, y);
        if (a.rest) {
            Vec8<T>::load(a.rest + row * a.D + c, z);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] += z[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) s += x[i] * y[i];
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (li == 0) {
        const int h = (int)(row % a.H);
        const size_t bt = row / a.H;
        delta[((bt / a.Tq) * a.H + h) * a.Tq + bt % a.Tq] = s;
    }
}

// four values of dq of row m, whose place is n: out, or to the key range's slab
template <typename T> __device__ __forceinline__ void leave_dq(const Args<T>& a, int split, int pair, int b, int hk, int m, int n, int col, f32x4 x) {
    if (a.nsplit == 1) store4(a.dq + pair_at(a, b, hk) + (size_t)n * a.D + col, x);
    else *reinterpret_cast<f32x4*>(a.ws + (((size_t)split * a.B * a.Hkv + pair) * a.M + m) * a.D + col) = x;
}
// four values of dk (which 0) or dv (1): out, or to the row range's slab [range][pair][dk | dv][key][D]
template <typename T> __device__ __forceinline__ void leave_dkv(const Args<T>& a, int split, int pair, int which, int key, int col, f32x4 x) {
    const int b = pair / a.Hkv, hk = pair % a.Hkv;
    if (a.nsplit == 1) store4((which ? a.dv : a.dk) + (((size_t)b * a.Tk + key) * a.Hkv + hk) * a.D + col, x);
    else *reinterpret_cast<f32x4*>(a.ws + (((size_t)split * a.B * a.Hkv + pair) * 2 * a.Tk + (size_t)which * a.Tk + key) * a.D + col) = x;
}

// Rows of a pair all on the chip (M <= 16 MT): ONE pass over the keys for all three gradients.  A tile's values pass
// through the wave's LDS for dP = dO V^T, then its keys for S = Q K^T (result tiles of 16 rows x 16 keys); P and
// dS = scale P (dP - delta) from them are the B operands of dV^T = dO^T P and dK^T = Q^T dS; dS^T, through 16 x 16 pieces of
// LDS, is the B operand of dQ^T += K^T dS^T, which stays in registers and is joined over waves (and key ranges) at the
// end.  dV and dK leave through the same LDS once the keys are done with, so that whole rows are written.  P and dS enter
// their products in two bf16 parts: the work is bound by reading the keys and writing their gradients, and only 16 of a
// matrix instruction's 32 contraction steps would be used otherwise.  Q^T and dO^T of up to 16 bf16 rows are held in
// registers (HELD); others are read, transposed, from LDS, one copy per item.
template <typename T, int DF, int MT, int W>
__global__ void __launch_bounds__(256, waves_bwd<T>(DF, MT)) k_xattn_bwd(Args<T> a) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    typedef typename Y::half half;
    constexpr bool HELD = MT == 1 && Y::PARTS;
    constexpr int DP = DF * Y::KC, DT = DP / 16, PITCH = DP * (int)sizeof(T) + Y::PAD, OP = DP + 4;
    constexpr int TILE = Y::KC * PITCH, JOIN = 4 * 16 * OP * 4, ROWS = HELD ? 0 : MT * 16 * PITCH;
    constexpr int PIECES = Y::NS * (Y::PARTS ? 2 : 1), SP = sizeof(T) == 4 ? 80 : 40, DS = PIECES * 16 * SP;     // dS^T: keys x 16 rows
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE > JOIN ? 4 * TILE : JOIN];
    __shared__ __attribute__((aligned(16))) char lds_ds[4 * DS], rows_lds[HELD ? 16 : (4 / W) * 2 * ROWS];
    __shared__ int places[4 / W][16 * MT];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4, w0 = wave % W;
    const int wi_ = work_item(a.blocks) * (4 / W) + wave / W;
    const bool idle = wi_ >= a.items;                        // an item past the last one: no keys, nothing stored
    const int wi = idle ? 0 : wi_;
    const int split = wi % a.nsplit, pair = wi / a.nsplit, b = pair / a.Hkv, hk = pair % a.Hkv, M = idle ? 0 : a.M;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const T* kb = a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh;
    const T* vb = a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh;
    const int first = split * a.tiles_split, last = idle ? 0 : min(first + a.tiles_split, (a.Tk + Y::KC - 1) / Y::KC);
    char *my = lds + wave * TILE, *my_ds = lds_ds + wave * DS;
    char *lq = rows_lds + (wave / W) * 2 * ROWS, *ldo = lq + ROWS;
    const float scale2 = a.scale * LOG2E;
    const unsigned out_st = a.Hkv * a.D;
    const bool spare = a.D <= DP - 16;                       // the last 16 columns are all padding

    // everything that the first tile waits for is requested at once: rows, outputs, statistics, then the tile itself
    frag q[MT][DF], d_o[MT][DF], o[MT][DF], rest[MT][DF];
    float row_lse[MT], lse[MT][4], delta[MT][4];             // of row li; of rows 4 g + r
    const size_t out0 = row_at(a, b, hk, 0);
    const T* rest_from = a.rest ? a.rest : a.o;              // (without a rest the outputs again, not used)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = mt * 16 + li;
        load_rows<T, DF>(a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh, a.q_st, a.q_sh, m, M, a.G, a.D, g, q[mt]);
        load_rows<T, DF>(a.dout + out0, (long)a.H * a.D, a.D, m, M, a.G, a.D, g, d_o[mt]);
        load_rows<T, DF>(a.o + out0, (long)a.H * a.D, a.D, m, M, a.G, a.D, g, o[mt]);
        if constexpr (Y::PARTS) load_rows<T, DF>(rest_from + out0, (long)a.H * a.D, a.D, m, M, a.G, a.D, g, rest[mt]);
        row_lse[mt] = a.lse[stat_at(a, b, hk, min(m, a.M - 1))];
    }
    Spots<T, DT> sp;
    sp.init(lane, a.D, Y::KC);
    KeyTile<T, DF> nxt;
    nxt.load(a, sp, mask, len, kb, vb, (first + w0) * Y::KC, li);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float s = 0.f;
        const frag none = {};
#pragma unroll
        for (int f = 0; f < DF; ++f) s += Y::dot(d_o[mt][f], o[mt][f], Y::PARTS && a.rest ? rest[mt][f] : none);
        s = groups_sum(s);
        const float l = mt * 16 + li < M ? row_lse[mt] * LOG2E : INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            delta[mt][r] = __shfl(s, g * 4 + r, 64);
            lse[mt][r] = __shfl(l, g * 4 + r, 64);
        }
    }
    half q_t[HELD ? DT : 1], do_t[HELD ? DT : 1];
    auto rows_to = [&](char* to, const frag (&r)[MT][DF]) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int f = 0; f < DF; ++f) *reinterpret_cast<frag*>(to + (mt * 16 + li) * PITCH + f * 64 + g * 16) = r[mt][f];
    };
    if constexpr (HELD) {
        rows_to(my, q);
        wave_lds_order();
#pragma unroll
        for (int d = 0; d < DT; ++d) q_t[d] = Y::read_t(my, PITCH, g * 4, d * 16, li);
        wave_lds_order();
        rows_to(my, d_o);
        wave_lds_order();
#pragma unroll
        for (int d = 0; d < DT; ++d) do_t[d] = Y::read_t(my, PITCH, g * 4, d * 16, li);
        wave_lds_order();
    } else {
        if (w0 == 0) { rows_to(lq, q); rows_to(ldo, d_o); }
        __syncthreads();
    }
    if (a.D < DP) wave_clear(my, TILE, lane);
    f32x4 dq[MT][DT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int d = 0; d < DT; ++d) dq[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int tile = first + w0; tile < last; tile += W) {
        const int key0 = tile * Y::KC;
        const KeyBits<T> bits = nxt.bits(mask != nullptr, len, key0, li);
        wave_lds_order();
        nxt.put(nxt.v, sp, bits, my, PITCH);
        wave_lds_order();
        nxt.load_v(a, sp, len, vb, key0 + W * Y::KC);
        f32x4 s[Y::NS][MT], dp[Y::NS][MT];
#pragma unroll
        for (int ns = 0; ns < Y::NS; ++ns) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[ns][mt] = dp[ns][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < DF; ++f) {
                const frag v = frag_at<T>(my, PITCH, ns * 16 + li, f, g);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) dp[ns][mt] = Y::mma(d_o[mt][f], v, dp[ns][mt]);
            }
        }
        wave_lds_order();
        nxt.put(nxt.k, sp, bits, my, PITCH);
        wave_lds_order();
        nxt.load_k(a, sp, mask, len, kb, key0 + W * Y::KC, li);
        half p[Y::NS][MT], p_lo[Y::NS][MT], ds[Y::NS][MT], ds_lo[Y::NS][MT];
#pragma unroll
        for (int ns = 0; ns < Y::NS; ++ns) {
#pragma unroll
            for (int f = 0; f < DF; ++f) {
                const frag k = frag_at<T>(my, PITCH, ns * 16 + li, f, g);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[ns][mt] = Y::mma(q[mt][f], k, s[ns][mt]);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[ns][mt][r] = __builtin_amdgcn_exp2f(s[ns][mt][r] * scale2 - lse[mt][r]);
                    dp[ns][mt][r] = s[ns][mt][r] * (dp[ns][mt][r] - delta[mt][r]) * a.scale;
                }
            if (bits.b[ns] != 0xffffu) {
                rarely();
                const bool on = (bits.b[ns] >> li) & 1;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[ns][mt][r] = on ? s[ns][mt][r] : 0.f;
                        dp[ns][mt][r] = on ? dp[ns][mt][r] : 0.f;
                    }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                Y::split(s[ns][mt], p[ns][mt], p_lo[ns][mt]);
                ds[ns][mt] = Y::pack(dp[ns][mt]);
                ds_lo[ns][mt] = Y::rest(dp[ns][mt], ds[ns][mt]);
            }
        }
        half dst[MT][Y::NS], dst_lo[MT][Y::NS];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {                    // dS^T by way of LDS: lane writes rows 4 g + r of key li
            wave_lds_order();
#pragma unroll
            for (int ns = 0; ns < Y::NS; ++ns) {
                *reinterpret_cast<half*>(my_ds + (ns * 16 + li) * SP + g * (int)sizeof(half)) = ds[ns][mt];
                if constexpr (Y::PARTS) *reinterpret_cast<half*>(my_ds + ((Y::NS + ns) * 16 + li) * SP + g * (int)sizeof(half)) = ds_lo[ns][mt];
            }
            wave_lds_order();
#pragma unroll
            for (int ns = 0; ns < Y::NS; ++ns) {
                dst[mt][ns] = Y::read_t(my_ds, SP, ns * 16 + g * 4, 0, li);
                if constexpr (Y::PARTS) dst_lo[mt][ns] = Y::read_t(my_ds, SP, (Y::NS + ns) * 16 + g * 4, 0, li);
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if (d == DT - 1 && spare) break;
            const frag kt = frag_t<T>(my, PITCH, d * 16, li, g);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                dq[mt][d] = Y::mma(kt, Y::join(dst[mt]), dq[mt][d]);
                if constexpr (Y::PARTS) dq[mt][d] = Y::mma(kt, Y::join(dst_lo[mt]), dq[mt][d]);
            }
        }
        // the tile's gradients: result tiles to LDS (over the keys), rows to memory
        auto leave = [&](T* to, const half (&held)[HELD ? DT : 1], const char* from, const half (&x)[Y::NS][MT], const half (&x_lo)[Y::NS][MT]) {
            wave_lds_order();
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                if (d == DT - 1 && spare) break;
#pragma unroll
                for (int ns = 0; ns < Y::NS; ++ns) {
                    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        if constexpr (HELD) y = Y::mma_parts(held[d], x[ns][mt], x_lo[ns][mt], y);
                        else y = Y::mma_parts(Y::read_t(from, PITCH, mt * 16 + g * 4, d * 16, li), x[ns][mt], x_lo[ns][mt], y);
                    }
                    store4(reinterpret_cast<T*>(my + (ns * 16 + li) * PITCH) + d * 16 + g * 4, y);
                }
            }
            wave_lds_order();
            const int n = min(Y::KC, a.Tk - key0);
            const Window w(to + (((size_t)b * a.Tk + key0) * a.Hkv + hk) * a.D, ((n - 1) * out_st + a.D) * (unsigned)sizeof(T));
            u32x4 out[DT];
#pragma unroll
            for (int i = 0; i < DT; ++i) out[i] = *reinterpret_cast<const u32x4*>(my + sp.row(i) * PITCH + sp.col(i) * (int)sizeof(T));
            const unsigned on = bits.b[0] | bits.b[Y::NS - 1] << (16 * (Y::NS - 1));
            if (on != (Y::NS == 2 ? 0xffffffffu : 0xffffu)) {            // keys that do not count: 0, whatever dO holds
                rarely();
#pragma unroll
                for (int i = 0; i < DT; ++i)
                    if (!((on >> sp.row(i)) & 1)) out[i] = u32x4{};
            }
#pragma unroll
            for (int i = 0; i < DT; ++i) w.store(sp.at(i, out_st), out[i]);
        };
        leave(a.dv, do_t, ldo, p, p_lo);
        leave(a.dk, q_t, lq, ds, ds_lo);
        if (a.D & 8) {
            // the result tiles wrote 8 columns behind D too: zero again, as all rows' next products run over them and a NaN
            // of one row left there would reach every other (a guard on the stores instead: fp32 32 x 20 on 576, 43.5 -> 47 us)
            constexpr int CH = 8 * (int)sizeof(T) / 16;
            wave_lds_order();
            if (lane < Y::KC * CH) *reinterpret_cast<u32x4*>(my + (lane / CH) * PITCH + a.D * (int)sizeof(T) + (lane % CH) * 16) = u32x4{};
        }
    }

    float* jo = reinterpret_cast<float*>(lds);
    const int it = threadIdx.x % (64 * W);                   // the thread in the item
    if (it < 16 * MT) places[wave / W][it] = place_of(a, it);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DT; ++d)
            *reinterpret_cast<f32x4*>(jo + (wave * 16 + li) * OP + d * 16 + g * 4) = dq[mt][d];
        __syncthreads();
#pragma unroll 2
        for (int c = it; c < 16 * (DP / 4); c += 64 * W) {
            const int r = c / (DP / 4), col = (c % (DP / 4)) * 4, m = mt * 16 + r;
            if (m >= M || col >= a.D) continue;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < W; ++i) x += *reinterpret_cast<const f32x4*>(jo + ((wave - w0 + i) * 16 + r) * OP + col);
            leave_dq(a, split, pair, b, hk, m, places[wave / W][m], col, x);
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
    store4(a.dq + row_at(a, pair / a.Hkv, pair % a.Hkv, m) + col, v);
}

// More rows than fit: the rows' side (dq) as the forward does it, rows in registers, key tiles streamed ...
template <typename T, int DF, int MT, int W>
__global__ void __launch_bounds__(256, waves_bwd_q<T>(DF)) k_xattn_bwd_q(Args<T> a) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    constexpr int DP = DF * Y::KC, DT = DP / 16, PITCH = DP * (int)sizeof(T) + Y::PAD, OP = DP + 4;
    constexpr int TILE = Y::KC * PITCH, JOIN = 4 * 16 * OP * 4;
    __shared__ __attribute__((aligned(16))) char lds[8 * TILE > JOIN ? 8 * TILE : JOIN];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4, w0 = wave % W;
    const int wi_ = work_item(a.blocks) * (4 / W) + wave / W;
    const bool idle = wi_ >= a.items;                        // an item past the last one: no keys, nothing stored
    const int wi = idle ? 0 : wi_, M = idle ? 0 : a.M;
    const int rb = wi % a.row_blocks, ps = wi / a.row_blocks, split = ps % a.nsplit, pair = ps / a.nsplit;
    const int b = pair / a.Hkv, hk = pair % a.Hkv, m0 = rb * 16 * MT;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const T* kb = a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh;
    const T* vb = a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh;
    const int first = split * a.tiles_split, last = idle ? 0 : min(first + a.tiles_split, (len + Y::KC - 1) / Y::KC);
    char *lk = lds + wave * 2 * TILE, *lv = lk + TILE;
    const float scale2 = a.scale * LOG2E;
    const size_t out0 = row_at(a, b, hk, 0);

    frag q[MT][DF], d_o[MT][DF];
    float lse[MT], delta[MT];                                // of row li
    f32x4 dq[MT][DT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 16 + li;
        load_rows<T, DF>(a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh, a.q_st, a.q_sh, m, M, a.G, a.D, g, q[mt]);
        load_rows<T, DF>(a.dout + out0, (long)a.H * a.D, a.D, m, M, a.G, a.D, g, d_o[mt]);
        const size_t at = stat_at(a, b, hk, min(m, a.M - 1));
        const float l = a.lse[at];
        delta[mt] = a.delta[at];
        lse[mt] = m < M ? l * LOG2E : INFINITY;
#pragma unroll
        for (int d = 0; d < DT; ++d) dq[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    Spots<T, DT> sp;
    sp.init(lane, a.D, Y::KC);
    KeyTile<T, DF> nxt;
    nxt.load(a, sp, mask, len, kb, vb, (first + w0) * Y::KC, li);
    if (a.D < DP) wave_clear(lk, 2 * TILE, lane);
    for (int tile = first + w0; tile < last; tile += W) {
        wave_lds_order();
        const KeyBits<T> bits = nxt.bits(mask != nullptr, len, tile * Y::KC, li);
        nxt.put(nxt.k, sp, bits, lk, PITCH);
        nxt.put(nxt.v, sp, bits, lv, PITCH);
        wave_lds_order();
        nxt.load(a, sp, mask, len, kb, vb, (tile + W) * Y::KC, li);
        if (!(bits.b[0] | bits.b[Y::NS - 1])) continue;
        typename Y::half h[MT][Y::NS], lo[MT][Y::NS];
#pragma unroll
        for (int ns = 0; ns < Y::NS; ++ns) {
            f32x4 s[MT], dp[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt] = dp[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < DF; ++f) {
                const frag k = frag_at<T>(lk, PITCH, ns * 16 + li, f, g), v = frag_at<T>(lv, PITCH, ns * 16 + li, f, g);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    s[mt] = Y::mma(k, q[mt][f], s[mt]);
                    dp[mt] = Y::mma(v, d_o[mt][f], dp[mt]);
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool on = (bits.b[ns] >> (g * 4 + r)) & 1;
                    const float p = on ? __builtin_amdgcn_exp2f(s[mt][r] * scale2 - lse[mt]) : 0.f;
                    dp[mt][r] = on ? p * (dp[mt][r] - delta[mt]) : 0.f;
                }
                h[mt][ns] = Y::pack(dp[mt]);
                lo[mt][ns] = Y::rest(dp[mt], h[mt][ns]);
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const frag kt = frag_t<T>(lk, PITCH, d * 16, li, g);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                dq[mt][d] = Y::mma(kt, Y::join(h[mt]), dq[mt][d]);
                if constexpr (Y::PARTS) dq[mt][d] = Y::mma(kt, Y::join(lo[mt]), dq[mt][d]);
            }
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
        for (int c = threadIdx.x % (64 * W); c < 16 * (DP / 4); c += 64 * W) {
            const int r = c / (DP / 4), col = (c % (DP / 4)) * 4, m = m0 + mt * 16 + r;
            if (m >= M || col >= a.D) continue;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < W; ++i) x += *reinterpret_cast<const f32x4*>(jo + ((wave - w0 + i) * 16 + r) * OP + col);
            leave_dq(a, split, pair, b, hk, m, place_of(a, m), col, x * a.scale);
        }
    }
}

// ... and the keys' side (dk, dv): a wave keeps NS x 16 keys, their rows and both gradients in registers while the
// workgroup streams the rows through LDS, KC at a time.
template <typename T, int DF>
__global__ void __launch_bounds__(256, 2) k_xattn_bwd_kv(Args<T> a) {
    typedef Ty<T> Y;
    typedef typename Y::frag frag;
    typedef typename Y::half half;
    constexpr int DP = DF * Y::KC, DT = DP / 16, PITCH = DP * (int)sizeof(T) + Y::PAD, TILE = Y::KC * PITCH;
    __shared__ __attribute__((aligned(16))) char lq[TILE], ldo[TILE];
    __shared__ __attribute__((aligned(16))) float l_lse[Y::KC], l_delta[Y::KC];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int kblocks = a.row_blocks, kbk = wi % kblocks, ps = wi / kblocks, split = ps % a.nsplit, pair = ps / a.nsplit;
    const int b = pair / a.Hkv, hk = pair % a.Hkv, m_first = split * a.tiles_split * Y::KC, m_last = min(m_first + a.tiles_split * Y::KC, a.M);
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
        for (int m0 = m_first; m0 < m_last; m0 += Y::KC) {
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
            half p[Y::NS][Y::NS], ds[Y::NS][Y::NS], p_lo[Y::NS][Y::NS], ds_lo[Y::NS][Y::NS];         // [key tile][row tile]
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
                    Y::split(s[ns], p[ns][qs], p_lo[ns][qs]);
                    ds[ns][qs] = Y::pack(dp[ns]);
                    ds_lo[ns][qs] = Y::rest(dp[ns], ds[ns][qs]);
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const frag dot_ = frag_t<T>(ldo, PITCH, d * 16, li, g), qt = frag_t<T>(lq, PITCH, d * 16, li, g);
#pragma unroll
                for (int ns = 0; ns < Y::NS; ++ns) {
                    dv[ns][d] = Y::mma(dot_, Y::join(p[ns]), dv[ns][d]);
                    dk[ns][d] = Y::mma(qt, Y::join(ds[ns]), dk[ns][d]);
                    if constexpr (Y::PARTS) {
                        dv[ns][d] = Y::mma(dot_, Y::join(p_lo[ns]), dv[ns][d]);
                        dk[ns][d] = Y::mma(qt, Y::join(ds_lo[ns]), dk[ns][d]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int ns = 0; ns < Y::NS; ++ns) {
        const int key = key0 + ns * 16 + li;
        if (key >= a.Tk) continue;
        const bool on = (bits.b[ns] >> li) & 1;              // (a key that does not count: 0, whatever dO holds)
        const f32x4 z = {};
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int c = d * 16 + g * 4;
            if (c < a.D) {
                leave_dkv(a, split, pair, 0, key, c, on ? dk[ns][d] * a.scale : z);
                leave_dkv(a, split, pair, 1, key, c, on ? dv[ns][d] : z);
            }
        }
    }
}

// ---- few keys -------------------------------------------------------------------------------
// At most 32 keys under more than 16 rows: the roles change.  The keys and values of a pair (NK tiles of 16) stay in every
// wave's registers, the rows stream past, 16 at a time and each read once; scores of a row are complete at once, so the
// softmax needs no second look; dq leaves with its rows, dk and dv are summed in registers over a wave's rows and joined
// over waves and row ranges at the end.
template <typename T, int DF, int NK> struct FewKeys {
    typedef Ty<T> Y;
    static constexpr int DP = DF * Y::KC, DT = DP / 16, PITCH = DP * (int)sizeof(T) + Y::PAD, TILE = 16 * PITCH;
    // one operand's keys to LDS (zeros for those that do not count)
    static __device__ __forceinline__ void stage(char* lds, const T* base, long st, unsigned on, int Tk, int D) {
        constexpr int CH = DP / Y::E;
        for (int c = threadIdx.x; c < 16 * NK * CH; c += blockDim.x) {
            const int r = c / CH, col = (c % CH) * Y::E;
            typename Y::frag x = {};
            if (((on >> r) & 1) && col < D) x = *reinterpret_cast<const typename Y::frag*>(base + (size_t)r * st + col);
            *reinterpret_cast<typename Y::frag*>(lds + r * PITCH + col * (int)sizeof(T)) = x;
        }
    }
    static __device__ __forceinline__ unsigned live(const Args<T>& a, const uint8_t* mask, int len, int lane) {
        const int key = lane & 31;
        return (unsigned)(__ballot(key < 16 * NK && key < len && (!mask || mask[key] != 0)) & 0xffffffffu);
    }
};

template <typename T, int DF, int NK>
__global__ void __launch_bounds__(256, 2) k_xattn_fwd_few(Args<T> a) {
    typedef Ty<T> Y;
    typedef FewKeys<T, DF, NK> F;
    typedef typename Y::frag frag;
    typedef typename Y::half half;
    constexpr int DT = F::DT, PITCH = F::PITCH;
    __shared__ __attribute__((aligned(16))) char lds[2 * NK * F::TILE];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int split = wi % a.nsplit, pair = wi / a.nsplit, b = pair / a.Hkv, hk = pair % a.Hkv;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const unsigned on = F::live(a, a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr, len, lane);
    const T* qb = a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh;
    const int first = split * a.tiles_split, last = min(first + a.tiles_split, (a.M + 15) / 16);
    frag nxt[DF];
    load_rows<T, DF>(qb, a.q_st, a.q_sh, (first + wave) * 16 + li, a.M, a.G, a.D, g, nxt);
    F::stage(lds, a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh, a.k_st, on, a.Tk, a.D);
    F::stage(lds + NK * F::TILE, a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh, a.v_st, on, a.Tk, a.D);
    __syncthreads();
    frag k[NK][DF];
    half vt[NK][DT];
#pragma unroll
    for (int n = 0; n < NK; ++n) {
#pragma unroll
        for (int f = 0; f < DF; ++f) k[n][f] = frag_at<T>(lds, PITCH, n * 16 + li, f, g);
#pragma unroll
        for (int d = 0; d < DT; ++d) vt[n][d] = Y::read_t(lds + NK * F::TILE, PITCH, n * 16 + g * 4, d * 16, li);
    }
    const float scale2 = a.scale * LOG2E;
    for (int tile = first + wave; tile < last; tile += 4) {
        frag q[DF];
#pragma unroll
        for (int f = 0; f < DF; ++f) q[f] = nxt[f];
        load_rows<T, DF>(qb, a.q_st, a.q_sh, (tile + 4) * 16 + li, a.M, a.G, a.D, g, nxt);
        f32x4 s[NK];
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < DF; ++f) s[n] = Y::mma(k[n][f], q[f], s[n]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[n][r] = (on >> (n * 16 + g * 4 + r)) & 1 ? s[n][r] * scale2 : -INFINITY;
                top = fmaxf(top, s[n][r]);
            }
        }
        top = groups_max(top);
        const float at = top == -INFINITY ? 0.f : top;
        half hi[NK], lo[NK];
#pragma unroll
        for (int n = 0; n < NK; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[n][r] = __builtin_amdgcn_exp2f(s[n][r] - at);
                sum += s[n][r];
            }
            Y::split(s[n], hi[n], lo[n]);
        }
        sum = groups_sum(sum);
        const float inv = top == -INFINITY ? 0.f : 1.f / sum;
        const int m = tile * 16 + li;
        const size_t at_row = row_at(a, b, hk, min(m, a.M - 1));
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = 0; n < NK; ++n) o = Y::mma_parts(vt[n][d], hi[n], lo[n], o);
            const int col = d * 16 + g * 4;
            if (m < a.M && col < a.D) store_out(a, at_row + col, o * inv);
        }
        if (g == 0 && m < a.M && a.lse) a.lse[stat_at(a, b, hk, m)] = log_sum(top, sum);
    }
}

template <typename T, int DF, int NK>
__global__ void __launch_bounds__(256, waves_bwd_few<T>(DF, NK)) k_xattn_bwd_few(Args<T> a) {
    typedef Ty<T> Y;
    typedef FewKeys<T, DF, NK> F;
    typedef typename Y::frag frag;
    typedef typename Y::half half;
    constexpr int DT = F::DT, PITCH = F::PITCH, DP = F::DP, OP = DP + 4;
    constexpr int PIECES = Y::PARTS ? 2 : 1, SP = sizeof(T) == 4 ? 80 : 40, DS = NK * PIECES * 16 * SP;
    constexpr int WAVE = 2 * F::TILE + DS, KEYS = 2 * NK * F::TILE, JOIN = 4 * 16 * OP * 4;
    constexpr int LDS = KEYS > 4 * WAVE ? KEYS : 4 * WAVE;
    __shared__ __attribute__((aligned(16))) char lds[LDS > JOIN ? LDS : JOIN];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int split = wi % a.nsplit, pair = wi / a.nsplit, b = pair / a.Hkv, hk = pair % a.Hkv;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const unsigned on = F::live(a, a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr, len, lane);
    const T* qb = a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh;
    const size_t out0 = row_at(a, b, hk, 0);
    const T* rest_from = a.rest ? a.rest : a.o;              // (without a rest the outputs again, not used)
    const int first = split * a.tiles_split, last = min(first + a.tiles_split, (a.M + 15) / 16);
    const float scale2 = a.scale * LOG2E;

    struct { frag q[DF], d_o[DF], o[DF], rest[DF]; float lse; } nxt;
    auto fetch = [&](int tile) {
        const int m = tile * 16 + li;
        load_rows<T, DF>(qb, a.q_st, a.q_sh, m, a.M, a.G, a.D, g, nxt.q);
        load_rows<T, DF>(a.dout + out0, (long)a.H * a.D, a.D, m, a.M, a.G, a.D, g, nxt.d_o);
        load_rows<T, DF>(a.o + out0, (long)a.H * a.D, a.D, m, a.M, a.G, a.D, g, nxt.o);
        if constexpr (Y::PARTS) load_rows<T, DF>(rest_from + out0, (long)a.H * a.D, a.D, m, a.M, a.G, a.D, g, nxt.rest);
        nxt.lse = a.lse[stat_at(a, b, hk, min(m, a.M - 1))];
    };
    fetch(first + wave);
    F::stage(lds, a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh, a.k_st, on, a.Tk, a.D);
    F::stage(lds + NK * F::TILE, a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh, a.v_st, on, a.Tk, a.D);
    __syncthreads();
    frag k[NK][DF], v[NK][DF];
    half kt[NK][DT];
    f32x4 dk[NK][DT], dv[NK][DT];
#pragma unroll
    for (int n = 0; n < NK; ++n) {
#pragma unroll
        for (int f = 0; f < DF; ++f) {
            k[n][f] = frag_at<T>(lds, PITCH, n * 16 + li, f, g);
            v[n][f] = frag_at<T>(lds + NK * F::TILE, PITCH, n * 16 + li, f, g);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            kt[n][d] = Y::read_t(lds, PITCH, n * 16 + g * 4, d * 16, li);
            dk[n][d] = dv[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    __syncthreads();
    char *lq = lds + wave * WAVE, *ldo = lq + F::TILE, *my_ds = ldo + F::TILE;

    for (int tile = first + wave; tile < last; tile += 4) {
        const int m = tile * 16 + li;
        frag q[DF], d_o[DF];
        float s0 = 0.f;
        const frag none = {};
#pragma unroll
        for (int f = 0; f < DF; ++f) {
            q[f] = nxt.q[f];
            d_o[f] = nxt.d_o[f];
            s0 += Y::dot(d_o[f], nxt.o[f], Y::PARTS && a.rest ? nxt.rest[f] : none);
        }
        s0 = groups_sum(s0);
        const float l = m < a.M ? nxt.lse * LOG2E : INFINITY;
        fetch(tile + 4);
        wave_lds_order();
#pragma unroll
        for (int f = 0; f < DF; ++f) {
            *reinterpret_cast<frag*>(lq + li * PITCH + f * 64 + g * 16) = q[f];
            *reinterpret_cast<frag*>(ldo + li * PITCH + f * 64 + g * 16) = d_o[f];
        }
        float lse[4], delta[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            delta[r] = __shfl(s0, g * 4 + r, 64);
            lse[r] = __shfl(l, g * 4 + r, 64);
        }
        half p[NK], p_lo[NK], ds[NK], ds_lo[NK];
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            f32x4 s = {0.f, 0.f, 0.f, 0.f}, dp = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < DF; ++f) {
                s = Y::mma(q[f], k[n][f], s);
                dp = Y::mma(d_o[f], v[n][f], dp);
            }
            const bool live = (on >> (n * 16 + li)) & 1;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[r] = live ? __builtin_amdgcn_exp2f(s[r] * scale2 - lse[r]) : 0.f;
                dp[r] = live ? s[r] * (dp[r] - delta[r]) * a.scale : 0.f;
            }
            Y::split(s, p[n], p_lo[n]);
            ds[n] = Y::pack(dp);
            ds_lo[n] = Y::rest(dp, ds[n]);
            *reinterpret_cast<half*>(my_ds + (n * 16 + li) * SP + g * (int)sizeof(half)) = ds[n];
            if constexpr (Y::PARTS) *reinterpret_cast<half*>(my_ds + ((NK + n) * 16 + li) * SP + g * (int)sizeof(half)) = ds_lo[n];
        }
        wave_lds_order();
        half dst[NK], dst_lo[NK];
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            dst[n] = Y::read_t(my_ds, SP, n * 16 + g * 4, 0, li);
            dst_lo[n] = Y::PARTS ? Y::read_t(my_ds, SP, (NK + n) * 16 + g * 4, 0, li) : dst[n];
        }
        const size_t at_row = row_at(a, b, hk, min(m, a.M - 1));
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const half do_t = Y::read_t(ldo, PITCH, g * 4, d * 16, li), q_t = Y::read_t(lq, PITCH, g * 4, d * 16, li);
            f32x4 dq = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                dv[n][d] = Y::mma_parts(do_t, p[n], p_lo[n], dv[n][d]);
                dk[n][d] = Y::mma_parts(q_t, ds[n], ds_lo[n], dk[n][d]);
                dq = Y::mma_parts(kt[n][d], dst[n], dst_lo[n], dq);
            }
            const int col = d * 16 + g * 4;
            if (m < a.M && col < a.D) store4(a.dq + at_row + col, dq);
        }
    }

    // the waves' sums joined
    float* jo = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int d = 0; d < DT; ++d)
                *reinterpret_cast<f32x4*>(jo + (wave * 16 + li) * OP + d * 16 + g * 4) = which ? dv[n][d] : dk[n][d];
            __syncthreads();
            for (int c = threadIdx.x; c < 16 * (DP / 4); c += 256) {
                const int r = c / (DP / 4), col = (c % (DP / 4)) * 4, key = n * 16 + r;
                if (key >= a.Tk || col >= a.D) continue;
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 4; ++i) x += *reinterpret_cast<const f32x4*>(jo + (i * 16 + r) * OP + col);
                leave_dkv(a, split, pair, which, key, col, (on >> key) & 1 ? x : f32x4{0.f, 0.f, 0.f, 0.f});
            }
        }
}

// the row ranges of dk and dv summed in range order
template <typename T>
__global__ void __launch_bounds__(256) k_xattn_dkv_join(Args<T> a) {
    const int chunks = a.D / 4;
    const size_t pairs = (size_t)a.B * a.Hkv, per = (size_t)2 * a.Tk * chunks, id = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= pairs * per) return;
    const size_t pair = id / per;
    const int in = (int)(id % per), col = (in % chunks) * 4, kk = in / chunks, which = kk / a.Tk, key = kk % a.Tk;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.nsplit; ++s) x += *reinterpret_cast<const f32x4*>(a.ws + ((s * pairs + pair) * 2 * a.Tk + kk) * a.D + col);
    store4((which ? a.dv : a.dk) + ((((pair / a.Hkv) * a.Tk + key) * a.Hkv) + pair % a.Hkv) * a.D + col, x);
}

// ---- many rows and many keys ------------------------------------------------------------------
// Beyond 64 rows and 256 keys the matrix cores are the bound (14 M Tk / (M + Tk) flops per byte and 16-bit element, against
// 230 that the card does per byte it reads), and what feeds them is LDS: a wave that reads a 16 x 16 key fragment once for
// two row tiles keeps LDS as busy as the matrix core.  Keys (rows, in the keys' backward) lie in LDS, two tiles of 64, for
// eight waves of 32 rows each; the next tile is in flight in registers.  P and dS are rounded to bf16 for their products:
// each term moves by 2^-8 of itself at most, whatever the number of regions that count, which for terms of either sign is
// about as much noise as the rounding of the result, sqrt(2) of its error together; in two parts they would cost half as
// many products again.  dq alone has more where rows are short: its terms dS k cancel down to dS (k - k'), k' the keys' weighted mean, whose share of k is 1 / D with
// independent keys, while the noise is that of dS k (1.5 of the rounding's error at D <= 32, 1.43 from 64 on).  Up to 64 its
// dS therefore comes in two parts (8 x 509 on 2000 x 8 heads of 64: 56 us instead of 46).

// R rows (64 or 32) of two operands on their way to LDS, NW waves together
template <int DF, int NW, int R = 64> struct RowTile {
    static constexpr int DP = DF * 32, PITCH = DP * 2 + 16, TILE = R * PITCH, NI = (4 * DF * R + NW * 64 - 1) / (NW * 64);
    u32x4 x[NI], y[NI];
    int rc[NI];                                              // row | chunk << 8
    __device__ __forceinline__ void init(int D) {
        const unsigned per = D / 8, inv = (65536 + per - 1) / per;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const unsigned c = min((unsigned)(i * NW * 64 + threadIdx.x), per * R - 1), r = __umul24(c, inv) >> 16;
            rc[i] = (int)(r | (c - __umul24(r, per)) << 8);
        }
    }
    __device__ __forceinline__ unsigned row(int i) const { return rc[i] & 255; }
    __device__ __forceinline__ unsigned col(int i) const { return (rc[i] >> 8) * 8; }
    // rows of one stride (keys)
    static __device__ __forceinline__ Window window(const bf16_t* base, long st, long row0, int rows, int D) {
        return Window(base + (size_t)row0 * st, rows > 0 ? ((rows - 1) * (unsigned)st + D) * 2u : 0u);
    }
    __device__ __forceinline__ void put(char* lx, char* ly, unsigned long long on) {
        if (on != ~0ull) {
            rarely();
#pragma unroll
            for (int i = 0; i < NI; ++i)
                if (!((on >> row(i)) & 1)) x[i] = y[i] = u32x4{};
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int at = row(i) * PITCH + col(i) * 2;
            *reinterpret_cast<u32x4*>(lx + at) = x[i];
            *reinterpret_cast<u32x4*>(ly + at) = y[i];
        }
    }
};

// which of 64 keys count, one bit per key; the mask's bytes are requested with the tile
struct Live64 {
    unsigned m;
    __device__ __forceinline__ void load(const uint8_t* mask, const void* any, int key0, int Tk, int lane) {
        const uint8_t* p = mask ? mask : reinterpret_cast<const uint8_t*>(any);
        m = p[mask ? min(key0 + lane, Tk - 1) : 0];
    }
    __device__ __forceinline__ unsigned long long bits(bool masked, int len, int key0, int lane) const {
        return __ballot(key0 + lane < len && (!masked || m != 0));
    }
};

// the workgroup's LDS cleared (pad columns stay zero)
__device__ __forceinline__ void group_clear(char* lds, int bytes) {
    const f32x4 z = {};
    for (int at = threadIdx.x * 16; at < bytes; at += blockDim.x * 16) *reinterpret_cast<f32x4*>(lds + at) = z;
}

template <int DF, int NW>
__global__ void __launch_bounds__(NW * 64) k_xattn_fwd_tile(Args<bf16_t> a) {
    typedef Ty<bf16_t> Y;
    typedef RowTile<DF, NW> Tile;
    constexpr int DT = DF * 2, PITCH = Tile::PITCH, MT = 2;
    __shared__ __attribute__((aligned(16))) char lds[4 * Tile::TILE];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int rb = wi % a.row_blocks, ps = wi / a.row_blocks, split = ps % a.nsplit, pair = ps / a.nsplit;
    const int b = pair / a.Hkv, hk = pair % a.Hkv, m0 = (rb * NW + wave) * 16 * MT;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const bf16_t* kb = a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh;
    const bf16_t* vb = a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh;
    const int first = split * a.tiles_split, last = min(first + a.tiles_split, (len + 63) / 64);

    bf16x8_t q[MT][DF];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        load_rows<bf16_t, DF>(a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh, a.q_st, a.q_sh, m0 + mt * 16 + li, a.M, a.G, a.D, g, q[mt]);
    Tile nxt;
    Live64 live;
    nxt.init(a.D);
    auto load = [&](int tile) {
        const int key0 = tile * 64, rows = min(64, len - key0);
        live.load(mask, kb, key0, a.Tk, lane);
        const Window kw = Tile::window(kb, a.k_st, key0, rows, a.D), vw = Tile::window(vb, a.v_st, key0, rows, a.D);
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            nxt.x[i] = kw.load(((__umul24(nxt.row(i), (unsigned)a.k_st >> 3) << 3) + nxt.col(i)) * 2u);
            nxt.y[i] = vw.load(((__umul24(nxt.row(i), (unsigned)a.v_st >> 3) << 3) + nxt.col(i)) * 2u);
        }
    };
    load(first);
    f32x4 o[MT][DT];
    float mx[MT], sum[MT], weight[MT];                       // mx: scaled, in powers of two; sums of p, of the rounded p
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        mx[mt] = -INFINITY;
        sum[mt] = 0.f;
        weight[mt] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float scale2 = positive_scale(a.scale);
    // o is divided by the sum of the weights that its products take, p ROUNDED: it stays a weighted mean of the values, off by
    // 2^-8 of sum p |v - o| at most, and so does the backward's delta = dO o, which is subtracted from dO v.  Divided by
    // the sum of the exact p it would be off by up to 2^-8 of o where one region has most of the weight, however little
    // dO (v - o) is there.  The weights' sum costs an instruction for two p (8 x 509 on 4096: 184 -> 187 us; as matrix products
    // with ones 192).  The log-sum-exp is of the exact p.
    if (a.scale < 0.f) {
        rarely();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int f = 0; f < DF; ++f) q[mt][f] = -q[mt][f];
    }
    if (a.D < Tile::DP) { group_clear(lds, 4 * Tile::TILE); __syncthreads(); }
    unsigned long long on = live.bits(mask != nullptr, len, first * 64, lane), on_next = 0;
    nxt.put(lds, lds + Tile::TILE, on);
    load(first + 1);
    __syncthreads();

    int cur = 0;
    for (int tile = first; tile < last; ++tile) {
        const char *lk = lds + cur * 2 * Tile::TILE, *lv = lk + Tile::TILE;
        f32x4 s[MT][4];
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt][sub] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < DF; ++f) {
                const bf16x8_t k = frag_at<bf16_t>(lk, PITCH, sub * 16 + li, f, g);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][sub] = Y::mma(k, q[mt][f], s[mt][sub]);
            }
        }
        bf16x8_t p[MT][2];
        if (on != ~0ull) {
            rarely();
#pragma unroll
            for (int sub = 0; sub < 4; ++sub)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!((on >> (sub * 16 + g * 4 + r)) & 1))
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) s[mt][sub][r] = -INFINITY;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float top = -INFINITY;
#pragma unroll
            for (int sub = 0; sub < 4; ++sub)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, s[mt][sub][r]);
            top = groups_max(top) * scale2;
            // the maximum follows only when a row's has grown by more than 2^8: until then p stays below 256 and the
            // output need not be rescaled
            if (__any(top > mx[mt] + 8.f)) {
                const float up = fmaxf(top, mx[mt]), at = up == -INFINITY ? 0.f : up, shrink = __builtin_amdgcn_exp2f(mx[mt] - at);
                mx[mt] = up;
                sum[mt] *= shrink;
                weight[mt] *= shrink;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[mt][d] *= shrink;
            }
            const float at = mx[mt] == -INFINITY ? 0.f : mx[mt];
            Y::half h[4];
#pragma unroll
            for (int sub = 0; sub < 4; ++sub) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[mt][sub][r] = __builtin_amdgcn_exp2f(s[mt][sub][r] * scale2 - at);
                    sum[mt] += s[mt][sub][r];
                }
                h[sub] = Y::pack(s[mt][sub]);
            }
            const Y::half h0[2] = {h[0], h[1]}, h1[2] = {h[2], h[3]};
            p[mt][0] = Y::join(h0);
            p[mt][1] = Y::join(h1);
#pragma unroll
            for (int sub = 0; sub < 4; ++sub) weight[mt] = Y::sum(h[sub], weight[mt]);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const bf16x8_t vt = frag_t<bf16_t>(lv + kk * 32 * PITCH, PITCH, d * 16, li, g);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) o[mt][d] = Y::mma(vt, p[mt][kk], o[mt][d]);
            }
        cur ^= 1;
        on_next = live.bits(mask != nullptr, len, (tile + 1) * 64, lane);
        nxt.put(lds + cur * 2 * Tile::TILE, lds + cur * 2 * Tile::TILE + Tile::TILE, on_next);
        on = on_next;
        load(tile + 2);
        __syncthreads();
    }

    const size_t rows = (size_t)a.B * a.Hkv * a.M;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const float l = groups_sum(sum[mt]), l_rounded = groups_sum(weight[mt]), top = mx[mt];
        const int m = m0 + mt * 16 + li;
        if (m >= a.M) continue;
        const size_t at_row = (size_t)split * rows + (size_t)pair * a.M + m;
        // a key range's share of o leaves as its mean times its exact sum, which is what the join takes it for
        const float inv = top == -INFINITY ? 0.f : (a.nsplit > 1 ? l : 1.f) / l_rounded;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int col = d * 16 + g * 4;
            if (col >= a.D) continue;
            if (a.nsplit == 1) store_out(a, row_at(a, b, hk, m) + col, o[mt][d] * inv);
            else *reinterpret_cast<f32x4*>(a.ws + at_row * a.D + col) = o[mt][d] * inv;
        }
        if (g == 0) {
            if (a.nsplit > 1) {
                float* st = a.ws + (size_t)a.nsplit * rows * a.D + at_row * 2;
                st[0] = top;
                st[1] = l;
            } else if (a.lse) a.lse[stat_at(a, b, hk, m)] = log_sum(top, l);
        }
    }
}

// the rows' side of the backward, the same way
template <int DF, int NW>
__global__ void __launch_bounds__(NW * 64) k_xattn_bwd_q_tile(Args<bf16_t> a) {
    typedef Ty<bf16_t> Y;
    typedef RowTile<DF, NW> Tile;
    constexpr int DT = DF * 2, PITCH = Tile::PITCH, MT = 2;
    constexpr bool TWO = DF <= 2;                            // dS in two parts
    __shared__ __attribute__((aligned(16))) char lds[4 * Tile::TILE];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int rb = wi % a.row_blocks, ps = wi / a.row_blocks, split = ps % a.nsplit, pair = ps / a.nsplit, b = pair / a.Hkv, hk = pair % a.Hkv, m0 = (rb * NW + wave) * 16 * MT;
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const bf16_t* kb = a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh;
    const bf16_t* vb = a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh;
    const int first = split * a.tiles_split, last = min(first + a.tiles_split, (len + 63) / 64);
    const size_t out0 = row_at(a, b, hk, 0);

    bf16x8_t q[MT][DF], d_o[MT][DF];
    float lse[MT], delta[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 16 + li;
        load_rows<bf16_t, DF>(a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh, a.q_st, a.q_sh, m, a.M, a.G, a.D, g, q[mt]);
        load_rows<bf16_t, DF>(a.dout + out0, (long)a.H * a.D, a.D, m, a.M, a.G, a.D, g, d_o[mt]);
        const size_t at = stat_at(a, b, hk, min(m, a.M - 1));
        const float l = a.lse[at];
        delta[mt] = a.delta[at];
        lse[mt] = m < a.M && l != -INFINITY ? l * LOG2E : INFINITY;        // (nothing attended: p = 0)
    }
    Tile nxt;
    Live64 live;
    nxt.init(a.D);
    auto load = [&](int tile) {
        const int key0 = tile * 64, rows = min(64, len - key0);
        live.load(mask, kb, key0, a.Tk, lane);
        const Window kw = Tile::window(kb, a.k_st, key0, rows, a.D), vw = Tile::window(vb, a.v_st, key0, rows, a.D);
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            nxt.x[i] = kw.load(((__umul24(nxt.row(i), (unsigned)a.k_st >> 3) << 3) + nxt.col(i)) * 2u);
            nxt.y[i] = vw.load(((__umul24(nxt.row(i), (unsigned)a.v_st >> 3) << 3) + nxt.col(i)) * 2u);
        }
    };
    load(first);
    f32x4 dq[MT][DT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int d = 0; d < DT; ++d) dq[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float scale2 = uniform(a.scale * LOG2E);
    if (a.D < Tile::DP) { group_clear(lds, 4 * Tile::TILE); __syncthreads(); }
    unsigned long long on = live.bits(mask != nullptr, len, first * 64, lane);
    nxt.put(lds, lds + Tile::TILE, on);
    load(first + 1);
    __syncthreads();

    int cur = 0;
    for (int tile = first; tile < last; ++tile) {
        const char *lk = lds + cur * 2 * Tile::TILE, *lv = lk + Tile::TILE;
        if (on)                                              // (a tile that is masked throughout adds nothing)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            Y::half h[MT][2], lo[MT][2];
#pragma unroll
            for (int ns = 0; ns < 2; ++ns) {
                const int sub = kk * 2 + ns;
                f32x4 s[MT], dp[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt] = dp[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < DF; ++f) {
                    const bf16x8_t k = frag_at<bf16_t>(lk, PITCH, sub * 16 + li, f, g), v = frag_at<bf16_t>(lv, PITCH, sub * 16 + li, f, g);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        s[mt] = Y::mma(k, q[mt][f], s[mt]);
                        dp[mt] = Y::mma(v, d_o[mt][f], dp[mt]);
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)              // (a key that does not count is a row of zeros: its ds need only be finite)
                        dp[mt][r] = __builtin_amdgcn_exp2f(fminf(s[mt][r] * scale2 - lse[mt], 1.f)) * (dp[mt][r] - delta[mt]);
                    h[mt][ns] = Y::pack(dp[mt]);
                    if (TWO) lo[mt][ns] = Y::rest(dp[mt], h[mt][ns]);
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const bf16x8_t kt = frag_t<bf16_t>(lk + kk * 32 * PITCH, PITCH, d * 16, li, g);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    dq[mt][d] = Y::mma(kt, Y::join(h[mt]), dq[mt][d]);
                    if (TWO) dq[mt][d] = Y::mma(kt, Y::join(lo[mt]), dq[mt][d]);
                }
            }
        }
        cur ^= 1;
        on = live.bits(mask != nullptr, len, (tile + 1) * 64, lane);
        nxt.put(lds + cur * 2 * Tile::TILE, lds + cur * 2 * Tile::TILE + Tile::TILE, on);
        load(tile + 2);
        __syncthreads();
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 16 + li;
        if (m >= a.M) continue;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int col = d * 16 + g * 4;
            if (col < a.D) leave_dq(a, split, pair, b, hk, m, place_of(a, m), col, dq[mt][d] * a.scale);
        }
    }
}

// the keys' side: a wave keeps 32 keys, their rows and both gradients in registers, q and dO pass through LDS R
// rows at a time
template <int DF, int NW>
__global__ void __launch_bounds__(NW * 64) k_xattn_bwd_kv_tile(Args<bf16_t> a) {
    typedef Ty<bf16_t> Y;
    constexpr int R = DF == 4 ? 32 : 64;                     // (at the widest rows a prefetch of 64 would not fit the registers)
    typedef RowTile<DF, NW, R> Tile;
    constexpr int DT = DF * 2, PITCH = Tile::PITCH;
    // two tiles of q and dO rows, then the rows' lse and delta of each: [tile][lse | delta][row]
    __shared__ __attribute__((aligned(16))) char lds[4 * Tile::TILE + 4 * R * 4];
    const int wi = work_item(a.blocks);
    if (wi >= a.blocks) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int kblocks = a.row_blocks, kbk = wi % kblocks, ps = wi / kblocks, split = ps % a.nsplit, pair = ps / a.nsplit;
    const int b = pair / a.Hkv, hk = pair % a.Hkv, m_first = split * a.tiles_split * R, m_last = min(m_first + a.tiles_split * R, a.M);
    const int len = a.kv_len ? max(0, min(a.kv_len[b], a.Tk)) : a.Tk;
    const uint8_t* mask = a.mask ? a.mask + (size_t)b * a.mask_sb : nullptr;
    const int key0 = (kbk * NW + wave) * 32, block0 = kbk * NW * 32;
    const float scale2 = uniform(a.scale * LOG2E);
    const bf16_t* qb = a.q + (size_t)b * a.q_sb + (size_t)hk * a.G * a.q_sh;
    const bf16_t* dob = a.dout + row_at(a, b, hk, 0);

    const KeyBits<bf16_t> bits = key_bits(a, mask, len, key0, li);
    bf16x8_t k[2][DF], v[2][DF];
    load_keys<bf16_t, DF>(a.k + (size_t)b * a.k_sb + (size_t)hk * a.k_sh, a.k_st, bits, key0, a.D, li, g, k);
    load_keys<bf16_t, DF>(a.v + (size_t)b * a.v_sb + (size_t)hk * a.v_sh, a.v_st, bits, key0, a.D, li, g, v);
    f32x4 dk[2][DT], dv[2][DT];
#pragma unroll
    for (int ns = 0; ns < 2; ++ns)
#pragma unroll
        for (int d = 0; d < DT; ++d) dk[ns][d] = dv[ns][d] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (block0 < len) {                                      // (a block behind the regions: its gradients are zero)
        Tile nxt;
        float n_lse, n_delta;
        nxt.init(a.D);
        // the tile's rows as (token, head of the group): stepped from tile to tile, a division each would cost as much as
        // the exponentials
        const int dt = R / a.G, dh = R % a.G;
        struct Row { int t, h; };
        auto at_row = [&](int m) { Row r; r.t = m / a.G; r.h = m - r.t * a.G; return r; };
        auto next = [&](Row& r) { r.t += dt; r.h += dh; if (r.h >= a.G) { r.h -= a.G; ++r.t; } };
        Row rows[Tile::NI], stat = at_row(m_first + (lane & (R - 1)));
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) rows[i] = at_row(m_first + (int)nxt.row(i));
        auto load = [&]() {                                  // rows past the last one read it again (cleared before their use)
#pragma unroll
            for (int i = 0; i < Tile::NI; ++i) {
                const int t = min(rows[i].t, a.Tq - 1), hh = rows[i].h;
                nxt.x[i] = *reinterpret_cast<const u32x4*>(qb + (size_t)t * a.q_st + (size_t)hh * a.q_sh + nxt.col(i));
                nxt.y[i] = *reinterpret_cast<const u32x4*>(dob + ((size_t)t * a.H + hh) * a.D + nxt.col(i));
                next(rows[i]);
            }
            const size_t at = ((size_t)b * a.H + hk * a.G + stat.h) * a.Tq + min(stat.t, a.Tq - 1);
            const float l = a.lse[at], de = a.delta[at];
            n_delta = stat.t < a.Tq ? de : 0.f;
            n_lse = stat.t < a.Tq ? l * LOG2E : INFINITY;
            next(stat);
        };
        auto put = [&](int buf) {
            nxt.put(lds + buf * 2 * Tile::TILE, lds + buf * 2 * Tile::TILE + Tile::TILE, ~0ull);
            if (wave == 0 && lane < R) {
                float* st = reinterpret_cast<float*>(lds + 4 * Tile::TILE) + buf * 2 * R + lane;
                st[0] = n_lse;
                st[R] = n_delta;
            }
        };
        load();
        if (a.D < Tile::DP) { group_clear(lds, 4 * Tile::TILE); __syncthreads(); }
        put(0);
        load();
        __syncthreads();
        // a lane's places in a tile, as one number each (the compiler would keep their parts)
        int at_frag = li * PITCH + g * 16, at_t = (g * 4 + (li >> 2)) * PITCH + (li & 3) * 8;
        asm volatile("" : "+v"(at_frag), "+v"(at_t));
        int cur = 0;
        auto step = [&]() {
            const char* lq = lds + cur * 2 * Tile::TILE;         // q rows; dO rows a TILE behind
            const float* lst = reinterpret_cast<const float*>(lds + 4 * Tile::TILE) + cur * 2 * R;
#pragma unroll
            for (int hf = 0; hf < R / 32; ++hf) {
                Y::half p[2][2], ds[2][2];                   // [key tile][row tile]
#pragma unroll
                for (int qs = 0; qs < 2; ++qs) {
                    const int row = hf * 32 + qs * 16;
                    f32x4 s[2], dp[2];
#pragma unroll
                    for (int ns = 0; ns < 2; ++ns) s[ns] = dp[ns] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int f = 0; f < DF; ++f) {
                        const char* at = lq + at_frag + row * PITCH + f * 64;
                        const bf16x8_t qf = *reinterpret_cast<const bf16x8_t*>(at), df = *reinterpret_cast<const bf16x8_t*>(at + Tile::TILE);
#pragma unroll
                        for (int ns = 0; ns < 2; ++ns) {
                            s[ns] = Y::mma(qf, k[ns][f], s[ns]);
                            dp[ns] = Y::mma(df, v[ns][f], dp[ns]);
                        }
                    }
                    const f32x4 ls = *reinterpret_cast<const f32x4*>(lst + row + g * 4);
                    const f32x4 de = *reinterpret_cast<const f32x4*>(lst + R + row + g * 4);
#pragma unroll
                    for (int ns = 0; ns < 2; ++ns) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {        // (a key that does not count: its own sums, dropped at the end)
                            s[ns][r] = __builtin_amdgcn_exp2f(s[ns][r] * scale2 - ls[r]);
                            dp[ns][r] = s[ns][r] * (dp[ns][r] - de[r]);
                        }
                        p[ns][qs] = Y::pack(s[ns]);
                        ds[ns][qs] = Y::pack(dp[ns]);
                        asm volatile("" : "+v"(p[ns][qs]), "+v"(ds[ns][qs]));
                    }
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const char* at = lq + at_t + hf * 32 * PITCH + d * 32;
                    const bf16x8_t qt = frag_tr(at, PITCH), dot_ = frag_tr(at + Tile::TILE, PITCH);
#pragma unroll
                    for (int ns = 0; ns < 2; ++ns) {
                        dv[ns][d] = Y::mma(dot_, Y::join(p[ns]), dv[ns][d]);
                        dk[ns][d] = Y::mma(qt, Y::join(ds[ns]), dk[ns][d]);
                    }
                }
            }
        };
        int m0 = m_first;
        for (; m0 + R <= m_last; m0 += R) {
            step();
            cur ^= 1;
            put(cur);
            load();
            __syncthreads();
        }
        if (m0 < m_last) {                                   // rows past the last one: zeros (their p of 0 would make NaN of an infinite dO)
            for (int at = (m_last - m0) * PITCH + threadIdx.x * 16; at < Tile::TILE; at += NW * 64 * 16)
                *reinterpret_cast<u32x4*>(lds + cur * 2 * Tile::TILE + Tile::TILE + at) = u32x4{};
            __syncthreads();
            step();
        }
    }
#pragma unroll
    for (int ns = 0; ns < 2; ++ns) {
        const int key = key0 + ns * 16 + li;
        if (key >= a.Tk) continue;
        const bool on = (bits.b[ns] >> li) & 1;
        const f32x4 z = {};
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int c = d * 16 + g * 4;
            if (c < a.D) {
                leave_dkv(a, split, pair, 0, key, c, on ? dk[ns][d] * a.scale : z);
                leave_dkv(a, split, pair, 1, key, c, on ? dv[ns][d] : z);
            }
        }
    }
}

// ---- host -----------------------------------------------------------------------------------
int key_tile(int dtype) { return dtype == VQA_BF16 ? 32 : 16; }

// 16-row tiles a workgroup of the forward takes: all of a pair's rows up to 64 (each further tile re-reads the keys from
// the caches, not from registers); fp32, and rows wider than 96,
// leave registers for half as many
int row_tiles(long M, int D, int dtype) {
    const int most = dtype == VQA_BF16 && D <= 96 ? 4 : 2;
    int mt = 1;
    while (mt < most && 16L * mt < M) mt *= 2;
    return mt;
}
// Key ranges: one when the work items give every CU one; otherwise as many as bring two to a CU, of at least 256 keys each
// (bf16; 128 fp32), and at most 32 (the join reads them one after the other).
int key_splits(long items, int Tk, int dtype, bool tiled) {
    const int tile = tiled ? 64 : key_tile(dtype), tiles = (Tk + tile - 1) / tile, least = tiled ? 4 : 8;
    if (items >= 256 || tiles < 2 * least) return 1;
    long n = (512 + items - 1) / items;
    if (n > tiles / least) n = tiles / least;
    if (n > 32) n = 32;
    const int per = (int)((tiles + n - 1) / n);
    return (tiles + per - 1) / per;                          // no empty range
}
bool one_pass(long M) { return M <= 32; }                    // the backward that keeps all rows of a pair on the chip
bool tiled(long M, int Tk, int dtype) { return dtype == VQA_BF16 && M > 64 && Tk > 256; }        // k_xattn_*_tile
// k_xattn_*_few (bf16, forward and backward: 256 x 20 rows on 20 x 8 heads 39 us, the streaming pair 48; 100 x 16 on 1 x 15
// heads, two rows a head, 51 against 65; up to 16 rows both take one pass over as much)
bool few(long M, int Tk) { return Tk <= 32 && M > 16; }
// Row ranges of the few-keys kernels: two workgroups to a CU, of at least two row tiles per wave, at most 64 slabs
int row_splits(long pairs, long M) {
    const long tiles = (M + 15) / 16;
    long n = (512 + pairs - 1) / pairs;
    if (n > tiles / 8) n = tiles / 8;
    if (n > 64) n = 64;
    if (n < 1) n = 1;
    const long per = (tiles + n - 1) / n;
    return (int)((tiles + per - 1) / per);
}
// Waves of a tiled workgroup: eight share a key tile; four for so few rows that they take no more
int tile_waves(long M) { return M <= 128 ? 4 : 8; }

int fwd_splits(int B, int Tq, int Tk, int H, int Hkv, int D, int dtype) {
    const long M = (long)Tq * (H / Hkv);
    if (few(M, Tk)) return 1;                                // (its row ranges join nothing)
    const long mt = row_tiles(M, D, dtype), rows = tiled(M, Tk, dtype) ? 32 * tile_waves(M) : 16 * mt;
    return key_splits((long)B * Hkv * ((M + rows - 1) / rows), Tk, dtype, tiled(M, Tk, dtype));
}
int bwd_splits(int B, int Tq, int Tk, int H, int Hkv, int dtype) { return key_splits((long)B * Hkv, Tk, dtype, false); }

// Waves per work item: two, so that an item's end (the join) and the next one's beginning overlap with other items (64 x 8
// rows on 700 x 8 heads: 17 against 21 us); four where the items are fewer than two to a CU and only their own length counts
// (one image of 196 regions: 5.6 against 7.2), and where two would fill a last round of CUs (512 items) by less than half, if
// an item is `least` tiles long.  Time with four over time with two, 520 - 4100 items, both types, widths 64 and 128:
//   one row tile a wave, forward, last round less than half full: 0.87 - 1.04 from 5 tiles on, 0.85 - 0.97 from 16; others 0.96 -
//     1.10 from 16, up to 1.2 below; one-pass backward: 0.85 - 1.03 and 0.84 - 0.97, others 0.91 - 1.11, below 9 tiles up to 1.5;
//   several row tiles a wave, forward: 1.0 - 1.25 below 16 tiles, 0.88 - 1.07 from 16 on, others 0.95 - 1.17; dq with dk, dv the
//     same to a third of it: 0.93 - 1.05 from 16 tiles on;
//   from the sixth round on (2816 items) nothing is left to gain: 0.94 - 1.04.
int waves_of(const int items, const int tiles, const int least) {
    return items < 512 || (tiles >= least && (items - 1) % 512 < 256 && items <= 2816) ? 4 : 2;
}
constexpr int least_fwd(int row_tiles) { return row_tiles == 1 ? 5 : 16; }
constexpr int LEAST_BWD = 9, LEAST_Q = 16;                    // one-pass backward, dq of many rows

// The two-kernel backward: blocks, key ranges of the dq kernel, row ranges of the dk / dv kernel.  Ranges only where the
// blocks alone leave CUs idle; row ranges of at least 4 tiles, at most 16 (slabs of dk and dv are as large as they are).
// Forward and backward of bf16 2 x 509 rows on 2000 x 4 heads of 64: 75 us, 119 without ranges; fp32 2 x 200 on 200: 47, 56.
size_t delta_floats(size_t rows) { return (rows + 3) / 4 * 4; }             // (the slabs behind it start at 16 bytes)
struct TwoPlan { int row_blocks, key_splits, key_tiles, key_blocks, row_splits, row_tiles; };
TwoPlan two_plan(int B, int Hkv, long M, int Tk, int D, int dtype) {
    const bool tile = tiled(M, Tk, dtype);
    const long pairs = (long)B * Hkv;
    TwoPlan p;
    const int rows = tile ? 32 * tile_waves(M) : 32, ktile = tile ? 64 : key_tile(dtype), ktiles = (Tk + ktile - 1) / ktile;
    p.row_blocks = (int)((M + rows - 1) / rows);
    p.key_splits = key_splits(pairs * p.row_blocks, Tk, dtype, tile);
    p.key_tiles = (ktiles + p.key_splits - 1) / p.key_splits;
    const int keys = tile ? 256 : 4 * key_tile(dtype), rtile = tile ? (D > 96 ? 32 : 64) : key_tile(dtype);
    p.key_blocks = (Tk + keys - 1) / keys;
    const long rtiles = (M + rtile - 1) / rtile, blocks = pairs * p.key_blocks;
    long n = blocks >= 256 ? 1 : (512 + blocks - 1) / blocks;
    if (n > rtiles / 4) n = rtiles / 4;
    if (n > 16) n = 16;
    if (n < 1) n = 1;
    p.row_tiles = (int)((rtiles + n - 1) / n);
    p.row_splits = (int)((rtiles + p.row_tiles - 1) / p.row_tiles);
    return p;
}

template <typename T, int DF, int MT> void launch_fwd(const Args<T>& a, hipStream_t s) {
    const int grid = 8 * ((a.blocks + 7) / 8);
    if (waves_of(a.items, a.tiles_split, least_fwd(MT)) == 2) k_xattn_fwd<T, DF, MT, 2><<<grid, 256, 0, s>>>(a);
    else k_xattn_fwd<T, DF, MT, 4><<<grid, 256, 0, s>>>(a);
}
template <typename T, int DF> void launch_fwd_mt(const Args<T>& a, int mt, hipStream_t s) {
    if (mt == 1) launch_fwd<T, DF, 1>(a, s);
    else if (mt == 2) launch_fwd<T, DF, 2>(a, s);
    else if constexpr (sizeof(T) == 2 && DF < 4) launch_fwd<T, DF, 4>(a, s);
}
template <typename T, int DF> void launch_bwd(const Args<T>& a, hipStream_t s) {
    const int grid = 8 * ((a.blocks + 7) / 8);
    if (waves_of(a.items, a.tiles_split, LEAST_BWD) == 2) {
        if (a.M > 16) k_xattn_bwd<T, DF, 2, 2><<<grid, 256, 0, s>>>(a);
        else k_xattn_bwd<T, DF, 1, 2><<<grid, 256, 0, s>>>(a);
    } else {
        if (a.M > 16) k_xattn_bwd<T, DF, 2, 4><<<grid, 256, 0, s>>>(a);
        else k_xattn_bwd<T, DF, 1, 4><<<grid, 256, 0, s>>>(a);
    }
}
template <typename T, int DF> void launch_bwd_q(const Args<T>& a, hipStream_t s) {
    const int grid = 8 * ((a.blocks + 7) / 8);
    if (waves_of(a.items, a.tiles_split, LEAST_Q) == 2) k_xattn_bwd_q<T, DF, 2, 2><<<grid, 256, 0, s>>>(a);
    else k_xattn_bwd_q<T, DF, 2, 4><<<grid, 256, 0, s>>>(a);
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
bool view_ok(const VqaAttnView& v) { return v.data && aligned16(v.data) && v.sb % 8 == 0 && v.st % 8 == 0 && v.sh % 8 == 0 && v.sb >= 0 && v.st >= 0 && v.sh >= 0 && v.st < (1L << 25); }

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

// f<DF> for the tiled kernels
#define TILED(D, call)                                                                         \
    switch (((D) + 31) / 32) {                                                                 \
        case 1: { constexpr int DF = 1; call; break; }                                         \
        case 2: { constexpr int DF = 2; call; break; }                                         \
        case 3: { constexpr int DF = 3; call; break; }                                         \
        default: { constexpr int DF = 4; call; break; }                                        \
    }

template <typename T> void few_plan(Args<T>& a) {
    a.nsplit = row_splits((long)a.B * a.Hkv, a.M);
    const int tiles = (a.M + 15) / 16;
    a.tiles_split = (tiles + a.nsplit - 1) / a.nsplit;
    a.blocks = a.B * a.Hkv * a.nsplit;
}

template <typename T>
int fwd(Args<T> a, int nsplit, int dtype, hipStream_t stream) {
    a.nsplit = nsplit;
    bool done = few(a.M, a.Tk);
    if (done) {
        few_plan(a);
        const int grid = 8 * ((a.blocks + 7) / 8);
        if (a.Tk <= 16) BY_WIDTH(T, a.D, (k_xattn_fwd_few<T, DF, 1><<<grid, 256, 0, stream>>>(a)));
        else BY_WIDTH(T, a.D, (k_xattn_fwd_few<T, DF, 2><<<grid, 256, 0, stream>>>(a)));
    }
    if constexpr (sizeof(T) == 2) {
        if (tiled(a.M, a.Tk, dtype)) {
            const int nw = tile_waves(a.M), tiles = (a.Tk + 63) / 64;
            a.row_blocks = (a.M + 32 * nw - 1) / (32 * nw);
            a.tiles_split = (tiles + nsplit - 1) / nsplit;
            a.blocks = a.B * a.Hkv * a.row_blocks * nsplit;
            const int grid = 8 * ((a.blocks + 7) / 8);
            if (nw == 8) { TILED(a.D, (k_xattn_fwd_tile<DF, 8><<<grid, 512, 0, stream>>>(a))) }
            else { TILED(a.D, (k_xattn_fwd_tile<DF, 4><<<grid, 256, 0, stream>>>(a))) }
            done = true;
        }
    }
    if (!done) {
        const int mt = row_tiles(a.M, a.D, dtype);
        a.row_blocks = (a.M + 16 * mt - 1) / (16 * mt);
        const int tiles = (a.Tk + Ty<T>::KC - 1) / Ty<T>::KC;
        a.tiles_split = (tiles + nsplit - 1) / nsplit;
        a.items = a.B * a.Hkv * a.row_blocks * nsplit;
        a.blocks = waves_of(a.items, a.tiles_split, least_fwd(mt)) == 2 ? (a.items + 1) / 2 : a.items;
        BY_WIDTH(T, a.D, (launch_fwd_mt<T, DF>(a, mt, stream)));
    }
    int rc = vqa_check_launch("vqa_cross_attn_fwd");
    if (rc || nsplit == 1) return rc;
    const size_t n = (size_t)a.B * a.Hkv * a.M * (a.D / 4);
    k_xattn_join<T><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a);
    return vqa_check_launch("vqa_cross_attn_fwd (join)");
}

template <typename T>
int bwd(Args<T> a, int nsplit, int dtype, hipStream_t stream) {
    if (one_pass(a.M) && !few(a.M, a.Tk)) {
        a.nsplit = nsplit;
        const int tiles = (a.Tk + Ty<T>::KC - 1) / Ty<T>::KC;
        a.tiles_split = (tiles + nsplit - 1) / nsplit;
        a.items = a.B * a.Hkv * nsplit;
        a.blocks = waves_of(a.items, a.tiles_split, LEAST_BWD) == 2 ? (a.items + 1) / 2 : a.items;
        BY_WIDTH(T, a.D, (launch_bwd<T, DF>(a, stream)));
        int rc = vqa_check_launch("vqa_cross_attn_bwd");
        if (rc || nsplit == 1) return rc;
        const size_t n = (size_t)a.B * a.Hkv * a.M * (a.D / 4);
        k_xattn_dq_join<T><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a);
        return vqa_check_launch("vqa_cross_attn_bwd (join)");
    }
    if (few(a.M, a.Tk)) {
        few_plan(a);
        const int grid = 8 * ((a.blocks + 7) / 8);
        if (a.Tk <= 16) BY_WIDTH(T, a.D, (k_xattn_bwd_few<T, DF, 1><<<grid, 256, 0, stream>>>(a)));
        else BY_WIDTH(T, a.D, (k_xattn_bwd_few<T, DF, 2><<<grid, 256, 0, stream>>>(a)));
        int rc = vqa_check_launch("vqa_cross_attn_bwd");
        if (rc || a.nsplit == 1) return rc;
        const size_t n = (size_t)a.B * a.Hkv * 2 * a.Tk * (a.D / 4);
        k_xattn_dkv_join<T><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a);
        return vqa_check_launch("vqa_cross_attn_bwd (join)");
    }
    const size_t rows = (size_t)a.B * a.Tq * a.H;
    const TwoPlan p = two_plan(a.B, a.Hkv, a.M, a.Tk, a.D, dtype);
    float* const ws = a.ws;
    k_xattn_delta<T><<<(unsigned)((rows + 15) / 16), 256, 0, stream>>>(a, ws);
    a.delta = ws;
    // dq
    a.row_blocks = p.row_blocks; a.nsplit = p.key_splits; a.tiles_split = p.key_tiles;
    a.items = a.B * a.Hkv * a.row_blocks * a.nsplit;
    float* const slabs = ws + delta_floats(rows);
    a.ws = slabs;
    const bool tile = tiled(a.M, a.Tk, dtype);
    if constexpr (sizeof(T) == 2) {
        if (tile) {
            a.blocks = a.items;
            const int grid = 8 * ((a.blocks + 7) / 8);
            if (tile_waves(a.M) == 8) { TILED(a.D, (k_xattn_bwd_q_tile<DF, 8><<<grid, 512, 0, stream>>>(a))) }
            else { TILED(a.D, (k_xattn_bwd_q_tile<DF, 4><<<grid, 256, 0, stream>>>(a))) }
        }
    }
    if (!tile) {
        a.blocks = waves_of(a.items, a.tiles_split, LEAST_Q) == 2 ? (a.items + 1) / 2 : a.items;
        BY_WIDTH(T, a.D, (launch_bwd_q<T, DF>(a, stream)));
    }
    int rc = vqa_check_launch("vqa_cross_attn_bwd (dq)");
    if (rc) return rc;
    if (a.nsplit > 1) {
        const size_t n = rows * (a.D / 4);
        k_xattn_dq_join<T><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a);
    }
    // dk, dv
    a.ws = slabs + (p.key_splits > 1 ? p.key_splits * rows * a.D : 0);
    a.row_blocks = p.key_blocks; a.nsplit = p.row_splits; a.tiles_split = p.row_tiles;
    a.blocks = a.B * a.Hkv * a.row_blocks * a.nsplit;
    const int grid = 8 * ((a.blocks + 7) / 8);
    if constexpr (sizeof(T) == 2) {
        if (tile) { TILED(a.D, (k_xattn_bwd_kv_tile<DF, 8><<<grid, 512, 0, stream>>>(a))) }
    }
    if (!tile) BY_WIDTH(T, a.D, (k_xattn_bwd_kv<T, DF><<<grid, 256, 0, stream>>>(a)));
    rc = vqa_check_launch("vqa_cross_attn_bwd (dk, dv)");
    if (rc || a.nsplit == 1) return rc;
    const size_t n = (size_t)a.B * a.Hkv * 2 * a.Tk * (a.D / 4);
    k_xattn_dkv_join<T><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a);
    return vqa_check_launch("vqa_cross_attn_bwd (join)");
}

bool sizes_ok(int B, int Tq, int Tk, int H, int Hkv, int D, int dtype) {
    return (dtype == VQA_F32 || dtype == VQA_BF16) && B > 0 && Tq > 0 && Tk > 0 && Hkv > 0 && H > 0 && H % Hkv == 0 && D > 0 &&
           D % 8 == 0 && D <= VQA_CROSS_ATTN_MAX_D && (long)B * Tq * H <= (1L << 27) && Tk <= (1 << 24) &&
           (long)Hkv * D < (1L << 25) &&
           // (a launch has fewer than 2^32 threads; the largest grids are these blocks, of 256)
           (long)B * Hkv * (((long)Tq * (H / Hkv) + 15) / 16) <= (1L << 23) && (long)B * Hkv * ((Tk + 63) / 64) <= (1L << 23);
}
#define XA_COMMON(fn)                                                                                                          \
    VQA_REQUIRE(sizes_ok(B, Tq, Tk, H, Hkv, D, dtype), fn ": dtype VQA_F32 or VQA_BF16, positive sizes, H a multiple of Hkv, " \
                "D a multiple of 8 up to 128, B * Tq * H <= 2^27, Tk <= 2^24, at most 2^23 blocks of 16 rows or 64 keys");      \
    VQA_REQUIRE(q && k && v && view_ok(*q) && view_ok(*k) && view_ok(*v),                                                      \
                fn ": q, k, v must be 16-byte aligned with strides that are multiples of 8");                                  \
    VQA_REQUIRE(!mask || B == 1 || mask_sb >= 0, fn ": the mask's stride must not be negative");                               \
    VQA_REQUIRE(isfinite(scale), fn ": scale must be finite");

}  // namespace

extern "C" {

size_t vqa_cross_attn_fwd_workspace_floats(int B, int Tq, int Tk, int H, int Hkv, int D, int dtype) {
    if (!sizes_ok(B, Tq, Tk, H, Hkv, D, dtype)) return 0;
    const int n = fwd_splits(B, Tq, Tk, H, Hkv, D, dtype);
    return n > 1 ? (size_t)n * B * Tq * H * (D + 2) : 0;
}
size_t vqa_cross_attn_bwd_workspace_floats(int B, int Tq, int Tk, int H, int Hkv, int D, int dtype) {
    if (!sizes_ok(B, Tq, Tk, H, Hkv, D, dtype)) return 0;
    const long M = (long)Tq * (H / Hkv);
    if (few(M, Tk)) {
        const int s = row_splits((long)B * Hkv, M);
        return s > 1 ? (size_t)s * B * Hkv * 2 * Tk * D : 0;
    }
    if (!one_pass(M)) {
        const TwoPlan p = two_plan(B, Hkv, M, Tk, D, dtype);
        const size_t rows = (size_t)B * Tq * H;
        return delta_floats(rows) + (p.key_splits > 1 ? p.key_splits * rows * D : 0) + (p.row_splits > 1 ? (size_t)p.row_splits * B * Hkv * 2 * Tk * D : 0);
    }
    const int n = bwd_splits(B, Tq, Tk, H, Hkv, dtype);
    return n > 1 ? (size_t)n * B * Tq * H * D : 0;
}

int vqa_cross_attn_fwd(const VqaAttnView* q, const VqaAttnView* k, const VqaAttnView* v, const int32_t* kv_len, const uint8_t* mask,
                       long mask_sb, float scale, void* o, void* o_rest, float* lse, float* workspace, int B, int Tq, int Tk, int H, int Hkv,
                       int D, int dtype, hipStream_t stream) {
    XA_COMMON("vqa_cross_attn_fwd")
    const int n = fwd_splits(B, Tq, Tk, H, Hkv, D, dtype);
    VQA_REQUIRE(o && aligned16(o) && aligned16(o_rest) && aligned16(workspace) && (workspace || n == 1),
                "vqa_cross_attn_fwd: o must be 16-byte aligned; this size needs the workspace");
    if (dtype == VQA_BF16) {
        Args<bf16_t> a = args_of<bf16_t>(*q, *k, *v, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D);
        a.o = (bf16_t*)o; a.rest = (bf16_t*)o_rest; a.lse = lse; a.ws = workspace;
        return fwd(a, n, dtype, stream);
    }
    Args<float> a = args_of<float>(*q, *k, *v, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D);
    a.o = (float*)o; a.lse = lse; a.ws = workspace;
    return fwd(a, n, dtype, stream);
}

int vqa_cross_attn_bwd(const void* d_o, const VqaAttnView* q, const VqaAttnView* k, const VqaAttnView* v, const void* o, const void* o_rest,
                       const float* lse, const int32_t* kv_len, const uint8_t* mask, long mask_sb, float scale, void* dq, void* dk,
                       void* dv, float* workspace, int B, int Tq, int Tk, int H, int Hkv, int D, int dtype, hipStream_t stream) {
    XA_COMMON("vqa_cross_attn_bwd")
    const int n = bwd_splits(B, Tq, Tk, H, Hkv, dtype);
    VQA_REQUIRE(d_o && o && lse && dq && dk && dv && aligned16(d_o) && aligned16(o) && aligned16(o_rest) && aligned16(dq) && aligned16(dk) && aligned16(dv),
                "vqa_cross_attn_bwd: d_o, o, lse, dq, dk, dv are needed, 16-byte aligned");
    VQA_REQUIRE(aligned16(workspace) && (workspace || vqa_cross_attn_bwd_workspace_floats(B, Tq, Tk, H, Hkv, D, dtype) == 0),
                "vqa_cross_attn_bwd: this size needs the workspace");
    if (dtype == VQA_BF16) {
        Args<bf16_t> a = args_of<bf16_t>(*q, *k, *v, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D);
        a.dout = (const bf16_t*)d_o; a.o = (bf16_t*)o; a.rest = (bf16_t*)o_rest; a.lse = (float*)lse;
        a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv; a.ws = workspace;
        return bwd(a, n, dtype, stream);
    }
    Args<float> a = args_of<float>(*q, *k, *v, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D);
    a.dout = (const float*)d_o; a.o = (float*)o; a.lse = (float*)lse;
    a.dq = (float*)dq; a.dk = (float*)dk; a.dv = (float*)dv; a.ws = workspace;
    return bwd(a, n, dtype, stream);
}

}  // extern "C"
