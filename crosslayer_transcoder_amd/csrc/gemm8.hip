// C[M][N] (+)= A[M][K] * B[N][K]^T + bias[N] for 8-bit block-scaled operands (held form: block8_common.h), batched.
//
//   C[m][n] = sum over blocks kb of 2^(ea[kb][m] + eb[kb][n]) * (sum over the block's 128 k of a * b)
//
// Two inner products, by the type of the result (gfx950's 8-bit matrix instructions align the products of a group of 16 at the
// largest one and keep about 14 bits below it — measured 1.0e-5 .. 1.5e-5 relative on normal data, whichever 8-bit instruction
// and shape; their sums over groups and blocks are fp32):
//   16-bit results: v_mfma_scale_f32_16x16x128_f8f6f4, one instruction per 16 x 16 tile and block of 128, scales as operands —
//     the alignment loss is far below the result's own rounding (2^-9 bf16, 2^-12 fp16).
//   32-bit results: the codes become bf16 in registers (2^e x code is exact in bf16) and go through v_mfma_f32_16x16x32_bf16:
//     exact products, fp32 sums, at the 16-bit rate.
// B rows ride the instruction's "M" index and A rows its "N" index, so a lane's four accumulators are four consecutive columns
// of one row of C.
#include "block8_common.h"

namespace {
typedef b8_f32x4 f32x4;

// Four consecutive columns of a row of C: 16- or 8-byte store where the row's alignment allows it (vec), else element by element
template <int DT> __device__ __forceinline__ void store4(void* c, long at, f32x4 v, int valid, bool vec, int accumulate) {
    typename Elem<DT>::type* p = static_cast<typename Elem<DT>::type*>(c) + at;
    if constexpr (DT == CLT_DT_F32) {
        if (vec && valid >= 4) {
            f32x4* q = reinterpret_cast<f32x4*>(p);
            *q = accumulate ? *q + v : v;
        } else
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i < valid) p[i] = accumulate ? p[i] + v[i] : v[i];
    } else {
        if (vec && valid >= 4) *reinterpret_cast<uint2*>(p) = make_uint2(pack_out16<DT>(v[0], v[1]), pack_out16<DT>(v[2], v[3]));
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i < valid) p[i] = f32_to_elem<DT>(v[i]);
    }
}

// 128 x 128 tile, 4 waves of 64 x 64, one k-block (128 bytes a row) staged through registers into LDS while the next is loaded.
// LDS rows are 128 bytes whose 16-byte chunks are XOR-swizzled with bits 1..3 of the row (conflict-free fragment reads).
template <int DT, int FA, int FB> __global__ __launch_bounds__(256) void gemm8_kernel(Gemm8Args g) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * 128 * 128];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, fr = lane & 15, fq = lane >> 4;
    const int wb = w >> 1, wa = w & 1;
    const long per = (long)g.tilesA * g.tilesB, batch = blockIdx.x / per;
    const int t = (int)(blockIdx.x - batch * per), ta = t % g.tilesA, tb = t / g.tilesA;
    const int a0 = ta * 128, b0 = tb * 128;
    const uint8_t *A = g.a + batch * g.ba, *B = g.b + batch * g.bb, *As = g.as + batch * g.bas, *Bs = g.bs + batch * g.bbs;

    const uint8_t *pa[4], *pb[4];
    int at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int id = i * 256 + tid, row = id >> 3, ch = id & 7;
        pa[i] = A + (long)min(a0 + row, g.M - 1) * g.lda + ch * 16;          // rows past the edge: loaded, never stored
        pb[i] = B + (long)min(b0 + row, g.N - 1) * g.ldb + ch * 16;
        at[i] = row * 128 + ((ch ^ ((row >> 1) & 7)) << 4);
    }
    int ra[4], rb[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        ra[n] = min(a0 + wa * 64 + n * 16 + fr, g.M - 1);
        rb[n] = min(b0 + wb * 64 + n * 16 + fr, g.N - 1);
    }
    f32x4 acc[4][4];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    uint4 va[4], vb[4];
    int sa[4], sb[4];
    auto load = [&](int kb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            va[i] = *reinterpret_cast<const uint4*>(pa[i] + (long)kb * 128);
            vb[i] = *reinterpret_cast<const uint4*>(pb[i] + (long)kb * 128);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) { sa[n] = As[kb * g.ldas + ra[n]]; sb[n] = Bs[kb * g.ldbs + rb[n]]; }
    };
    if (g.KB > 0) load(0);
    for (int kb = 0; kb < g.KB; ++kb) {
        __syncthreads();                                   // every wave has read the previous block
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            *reinterpret_cast<uint4*>(lds + at[i]) = va[i];
            *reinterpret_cast<uint4*>(lds + 16384 + at[i]) = vb[i];
        }
        int ca[4], cb[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) { ca[n] = sa[n]; cb[n] = sb[n]; }
        if (kb + 1 < g.KB) load(kb + 1);
        __syncthreads();
        // a lane's 32 codes of a row: 16-byte chunks fq and fq + 4 (the same k for both operands; the order inside a block is free)
        b8_i32x8 fa[4], fb[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int x = fr >> 1, rowa = (wa * 64 + n * 16 + fr) * 128, rowb = 16384 + (wb * 64 + n * 16 + fr) * 128;
            const int4 a_lo = *reinterpret_cast<const int4*>(lds + rowa + ((fq ^ x) << 4)), a_hi = *reinterpret_cast<const int4*>(lds + rowa + (((fq + 4) ^ x) << 4));
            const int4 b_lo = *reinterpret_cast<const int4*>(lds + rowb + ((fq ^ x) << 4)), b_hi = *reinterpret_cast<const int4*>(lds + rowb + (((fq + 4) ^ x) << 4));
            fa[n] = b8_i32x8{a_lo.x, a_lo.y, a_lo.z, a_lo.w, a_hi.x, a_hi.y, a_hi.z, a_hi.w};
            fb[n] = b8_i32x8{b_lo.x, b_lo.y, b_lo.z, b_lo.w, b_hi.x, b_hi.y, b_hi.z, b_hi.w};
        }
        if constexpr (DT != CLT_DT_F32) {
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    acc[m][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[m], fa[n], acc[m][n], FB, FA, 0, cb[m], 0, ca[n]);
        } else {
            float xa[4], xb[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) { xa[n] = exp2_int(ca[n] - 127); xb[n] = exp2_int(cb[n] - 127); }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                b8_bf16x8 ha[4], hb[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    ha[n] = widen8<FA>((uint32_t)fa[n][2 * s], (uint32_t)fa[n][2 * s + 1], xa[n]);
                    hb[n] = widen8<FB>((uint32_t)fb[n][2 * s], (uint32_t)fb[n][2 * s + 1], xb[n]);
                }
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int n = 0; n < 4; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hb[m], ha[n], acc[m][n], 0, 0, 0);
            }
        }
    }
    constexpr int VEC = 4;
    const size_t es = DT == CLT_DT_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)g.c % (VEC * es)) == 0 && g.ldc % VEC == 0 && g.bc % VEC == 0;
    const float* bias = g.bias ? g.bias + batch * g.bbias : nullptr;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const int col = b0 + wb * 64 + m * 16 + fq * 4, valid = g.N - col;
        f32x4 bv = {0.0f, 0.0f, 0.0f, 0.0f};
        if (bias)
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i < valid) bv[i] = bias[col + i];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int row = a0 + wa * 64 + n * 16 + fr;
            if (row < g.M && valid > 0) store4<DT>(g.c, batch * g.bc + (long)row * g.ldc + col, acc[m][n] + bv, valid, vec, g.accumulate);
        }
    }
}

template <int DT> int launch(const Gemm8Args& g, int fa, int fb, long blocks, hipStream_t st) {
    const dim3 gr((unsigned)blocks), t(256);
    if (fa == 0 && fb == 0) gemm8_kernel<DT, 0, 0><<<gr, t, 0, st>>>(g);
    else if (fa == 1 && fb == 0) gemm8_kernel<DT, 1, 0><<<gr, t, 0, st>>>(g);
    else if (fa == 0) gemm8_kernel<DT, 0, 1><<<gr, t, 0, st>>>(g);
    else gemm8_kernel<DT, 1, 1><<<gr, t, 0, st>>>(g);
    CLT_LAUNCH_CHECK();
    return CLT_OK;
}
}  // namespace

extern "C" int clt_gemm8(const void* a, const void* a_scale, int a_format, long lda, long ldas, long a_batch, long as_batch,
                         const void* b, const void* b_scale, int b_format, long ldb, long ldbs, long b_batch, long bs_batch,
                         void* c, int c_dtype, long ldc, long c_batch, const float* bias, long bias_batch, int M, int N, int K,
                         int batch, int accumulate, void* stream) {
    if (M <= 0 || N <= 0 || K < 0 || batch <= 0 || c_dtype < 0 || c_dtype > 2 || (a_format & ~1) || (b_format & ~1) || !c) return CLT_ERR_SHAPE;
    if (accumulate && c_dtype != CLT_DT_F32) return CLT_ERR_SHAPE;                 // (a 16-bit sum would round at every call)
    const int KB = (int)(up128(K) / 128);
    if (KB && (!a || !a_scale || !b || !b_scale || lda < up128(K) || ldb < up128(K) || ldas < M || ldbs < N || ldc < N)) return CLT_ERR_SHAPE;
    if (KB && (!aligned16(a) || !aligned16(b) || lda % 16 || ldb % 16 || a_batch % 16 || b_batch % 16)) return CLT_ERR_ALIGN;
    if (((uintptr_t)c & (c_dtype == CLT_DT_F32 ? 3 : 1)) || ((uintptr_t)bias & 3)) return CLT_ERR_ALIGN;
    Gemm8Args g = {static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(a_scale), static_cast<const uint8_t*>(b),
                   static_cast<const uint8_t*>(b_scale), c, bias, lda, ldas, ldb, ldbs, ldc, a_batch, as_batch, b_batch, bs_batch,
                   c_batch, bias_batch, M, N, KB, (M - 1) / 128 + 1, (N - 1) / 128 + 1, accumulate};
    const hipStream_t st = as_stream(stream);
    const int rc = clt_internal_gemm8_large(g, a_format, b_format, c_dtype, batch, st);
    if (rc <= 0) return rc;                                  // (1: the shape is the small tiles')
    const long blocks = (long)g.tilesA * g.tilesB * batch;
    if (blocks > 0x7fffffffL) return CLT_ERR_RANGE;
    return c_dtype == CLT_DT_F32 ? launch<CLT_DT_F32>(g, a_format, b_format, blocks, st)
           : c_dtype == CLT_DT_BF16 ? launch<CLT_DT_BF16>(g, a_format, b_format, blocks, st)
                                    : launch<CLT_DT_F16>(g, a_format, b_format, blocks, st);
}
