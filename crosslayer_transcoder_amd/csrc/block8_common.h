// 8-bit block-scaled matrices: the held form shared by quant8.hip, gemm8.hip and rows8.hip.
//
// A matrix [R, C] is held as codes [R][up128(C)] bytes (zero behind C) and scale bytes [up128(C) / 128][up128(R)]: the byte
// e + 127 is the scale 2^e of a row's block of 128 columns, rows contiguous.  Powers of two because (a) the scaling is then
// exact, so a code is the input rounded ONCE and is defined bit for bit, (b) the matrix instruction takes the scale as an
// operand (E8M0) and applies it for nothing, (c) 2^e x code is exact in bf16.  One granularity for every operand: a 128 x 128
// weight tile repeats its byte for 128 rows (1/128 byte an element).
#pragma once
#include "common.h"

constexpr int B8 = 128;                              // block: columns that share a scale
constexpr int B8_MIN_EXP = -112;                     // smallest scale exponent: 2^-e stays a normal fp32 number, and code x 2^e one of e4m3
// (e5m2's smallest codes, 2^-16 .. 3 x 2^-16, are subnormal numbers there, in fp32 and bf16: exact as long as subnormals are kept, which
// the conversions and the bf16 matrix instructions do; tested.)  At the other end 1.9375 x 2^127 (e5m2: 1.875) and more rounds to code x 2^e =
// 2^128, an infinity in fp32 and bf16.

// a launch's threads are counted in 32 bits
static inline bool b8_fits(long blocks, int threads) { return blocks <= 0xffffffffL / threads; }

__host__ __device__ static inline long up128(long n) { return (n + 127) / 128 * 128; }

// Scale exponent of a block from the bits of its largest finite magnitude: the smallest e >= -112 with amax <= largest * 2^e.
// largest = 1.75 * 2^8 (e4m3) or 1.75 * 2^15 (e5m2), so e follows from amax's exponent and whether its mantissa exceeds 1.75.
template <int FMT> __device__ __forceinline__ int block_exponent(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23) - 127 - (FMT ? 15 : 8) + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < B8_MIN_EXP ? B8_MIN_EXP : e;          // (zero and subnormal fp32 maxima land here too)
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// |x| as bits, 0 for inf and NaN: they take no part in the scale (and become NaN, or e5m2's infinity, as codes)
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
// four values / 2^e -> four codes (nearest, ties to even; the conversion takes the scale)
template <int FMT> __device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d, float scale) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    s16x2 r = {0, 0};
    if constexpr (FMT) {
        r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, a, b, scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, c, d, scale, true);
    } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
    }
    return __builtin_bit_cast(uint32_t, r);
}
// four codes -> four values (unscaled, exact)
typedef float b8_f32x2 __attribute__((ext_vector_type(2)));
typedef float b8_f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ b8_f32x4 unpack_codes(int fmt, uint32_t u) {
    const b8_f32x2 lo = fmt ? __builtin_amdgcn_cvt_pk_f32_bf8((int)u, false) : __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false);
    const b8_f32x2 hi = fmt ? __builtin_amdgcn_cvt_pk_f32_bf8((int)u, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
    return b8_f32x4{lo[0], lo[1], hi[0], hi[1]};
}

// element types of unpacked tensors (CLT_DT_*): fp32, bf16, fp16
template <int DT> struct Elem { typedef uint16_t type; };
template <> struct Elem<CLT_DT_F32> { typedef float type; };
template <int DT> __device__ __forceinline__ float elem_to_f32(typename Elem<DT>::type v) {
    if constexpr (DT == CLT_DT_F32) return v;
    else if constexpr (DT == CLT_DT_BF16) return bf16_to_f32(v);
    else return f16_to_f32(v);
}
// 16-byte accesses to rows that are aligned to their element only (unaligned vector accesses are legal here)
typedef uint32_t b8_u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef float b8_f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
// 8 consecutive elements of a row as fp32; `n` valid, the rest 0
template <int DT> __device__ __forceinline__ void b8_load8(const typename Elem<DT>::type* p, int n, float v[8]) {
    if (n >= 8) {
        if constexpr (DT == CLT_DT_F32) {
            const b8_f32x4_u a = reinterpret_cast<const b8_f32x4_u*>(p)[0], b = reinterpret_cast<const b8_f32x4_u*>(p + 4)[0];
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[k] = a[k]; v[k + 4] = b[k]; }
        } else {
            const b8_u32x4_u u = *reinterpret_cast<const b8_u32x4_u*>(p);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[2 * k] = elem_to_f32<DT>((uint16_t)(u[k] & 0xffffu));
                v[2 * k + 1] = elem_to_f32<DT>((uint16_t)(u[k] >> 16));
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k < n ? elem_to_f32<DT>(p[k]) : 0.0f;
    }
}
// two fp32 -> one dword of 16-bit results, nearest even (fp16: overflow gives inf; the loss scaler's flag is not touched here)
template <int DT> __device__ __forceinline__ uint32_t pack_out16(float lo, float hi) {
    if constexpr (DT == CLT_DT_BF16) return pack_bf16x2(lo, hi);
    else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const b8_f32x2 v = {lo, hi};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
    }
}
template <int DT> __device__ __forceinline__ typename Elem<DT>::type f32_to_elem(float v) {
    if constexpr (DT == CLT_DT_F32) return v;
    else return (uint16_t)pack_out16<DT>(v, 0.0f);
}

// ---- products (gemm8.hip, gemm8_large.hip) ----
typedef int b8_i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8_bf16x8 __attribute__((ext_vector_type(8)));
struct Gemm8Args {
    const uint8_t *a, *as, *b, *bs;          // codes and scale bytes
    void* c; const float* bias;
    long lda, ldas, ldb, ldbs, ldc;          // pitches: code rows, scale-byte rows (one per block of 128), C rows
    long ba, bas, bb, bbs, bc, bbias;        // batch strides
    int M, N, KB, tilesA, tilesB;
    int accumulate, batch;
    uint32_t inv_tiles, inv_panel, inv_rem;  // reciprocals of the large form's tile order (fast_div)
    int slices, slice_kb; float* part;       // K in slices: partial sums [slice][batch][M][N], else nullptr
    long slice_stride;                       // of the results (large form)
    int first;                               // small tiles: the large form has done this many of its tiles (0: none of them)
};

// n / d for n < 2^31 with inv = (2^32 - 1) / d from the host: the estimate is at most one too small.  (A division in a kernel costs a
// few hundred cycles of dependent vector instructions, and a lone wave per SIMD has nothing to put under them.)
__device__ __forceinline__ int fast_div(int n, int d, uint32_t inv) {
    int q = (int)__umulhi((uint32_t)n, inv);
    if (n - q * d >= d) ++q;
    return q;
}

constexpr int B8_PANEL = 4;                          // A tiles of a panel
struct B8Tile { int batch, slice, a0, b0; };
// 256 x 256 tile of index vb: every XCD (index mod 8) works on a contiguous range of tiles, walked in panels of 4 A tiles with the A tile
// fastest, so that the blocks an XCD runs together share operand tiles in its L2
__device__ __forceinline__ B8Tile b8_tile(const Gemm8Args& g, int vb) {
    const int nwg = g.tilesA * g.tilesB;
    B8Tile t;
    t.batch = fast_div(vb, nwg, g.inv_tiles);
    int lid = vb - t.batch * nwg;
    t.slice = 0;
    if (g.slices > 1) { t.slice = t.batch / g.slices; t.slice = t.batch - t.slice * g.slices; t.batch = (t.batch - t.slice) / g.slices; }
    const int xcd = lid & 7, q = nwg >> 3, r = nwg & 7;
    lid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (lid >> 3);
    const int full = g.tilesA / B8_PANEL, rem = g.tilesA - full * B8_PANEL, per = B8_PANEL * g.tilesB;
    int ta, tb;
    if (lid < full * per) { const int pn = fast_div(lid, per, g.inv_panel), x = lid - pn * per; tb = x / B8_PANEL; ta = pn * B8_PANEL + (x - tb * B8_PANEL); }
    else { const int x = lid - full * per; tb = fast_div(x, rem, g.inv_rem); ta = full * B8_PANEL + (x - tb * rem); }
    t.a0 = ta * 256; t.b0 = tb * 256;
    return t;
}
// for 256 x 256 tiles
inline void b8_tile_order(Gemm8Args& g) {
    g.tilesA = (g.M - 1) / 256 + 1; g.tilesB = (g.N - 1) / 256 + 1;
    const int rem = g.tilesA % B8_PANEL;
    g.inv_tiles = 0xffffffffu / (uint32_t)(g.tilesA * g.tilesB);
    g.inv_panel = 0xffffffffu / (uint32_t)(B8_PANEL * g.tilesB);
    g.inv_rem = rem ? 0xffffffffu / (uint32_t)rem : 0u;
}
int clt_internal_gemm8_large(const Gemm8Args& g, int fa, int fb, int dtype, int tiles, hipStream_t st);      // gemm8_large.hip

// Four consecutive columns of a row of C (`valid` of them): one store, aligned to the element only
typedef uint32_t b8_u32x2_u __attribute__((ext_vector_type(2), aligned(2)));
template <int DT> __device__ __forceinline__ void b8_store4(void* c, long at, b8_f32x4 v, int valid, int accumulate) {
    typename Elem<DT>::type* p = static_cast<typename Elem<DT>::type*>(c) + at;
    if constexpr (DT == CLT_DT_F32) {
        if (valid >= 4) {
            b8_f32x4_u* q = reinterpret_cast<b8_f32x4_u*>(p);
            *q = accumulate ? *q + v : v;
        } else
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i < valid) p[i] = accumulate ? p[i] + v[i] : v[i];
    } else {
        if (valid >= 4) *reinterpret_cast<b8_u32x2_u*>(p) = b8_u32x2_u{pack_out16<DT>(v[0], v[1]), pack_out16<DT>(v[2], v[3])};
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i < valid) p[i] = f32_to_elem<DT>(v[i]);
    }
}

// eight codes (two dwords) x 2^e -> eight bf16
template <int FMT> __device__ __forceinline__ b8_bf16x8 widen8(uint32_t lo, uint32_t hi, float scale) {
    b8_bf16x2 p[4];
    if constexpr (FMT) {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, false); p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, true);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, false); p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, true);
    } else {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false); p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false); p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    }
    return b8_bf16x8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}

