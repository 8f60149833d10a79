// C[M][N] (+)= A[M][K] * B[N][K]^T + bias[N] for 8-bit block-scaled operands (held form: block8_common.h), batched.
//
//   C[m][n] = sum over blocks kb of 2^(ea[kb][m] + eb[kb][n]) * (sum over the block's 128 k of a * b)
//
// Two inner products, by the type of the result (gfx950's 8-bit matrix instructions align the products of a group of 16 at the
// largest one and keep about 14 bits below it, whichever 8-bit instruction and shape; their sums over groups and blocks are fp32):
//   bf16 results: v_mfma_scale_f32_16x16x128_f8f6f4, one instruction per 16 x 16 tile and block of 128, scales as operands.  A group is
//     off by less than 16 * 2^-13 of its largest product, which is less than 2^-9 of the sum of |a b| over all of them.  Against 64 bits,
//     2048 x 768 x 4096: on normal data 1.1e-5 of the result's norm (rounding to bf16: 1.66e-3), 1 % of the values are the neighbour of
//     the rounded sum and a near-cancelled one may be off by many of its own places; with two columns 100 times larger than the rest that
//     cancel each other 2.2e-4 of the norm, 9 % neighbours.
//   fp16 and fp32 results: the codes become bf16 in registers (2^e x code is exact in bf16) and go through v_mfma_f32_16x16x32_bf16:
//     exact products, fp32 sums, at the 16-bit rate.  fp16 too: its rounding is 2e-4 of the norm, no more than the alignment may lose
//     (the cancelling columns: 3.1e-4 in all, 35 % of the values neighbours).
// B rows ride the instruction's "M" index and A rows its "N" index, so a lane's accumulators are consecutive columns of a row of C.
//
// This file: the entry point and the form for everything that does not fill the chip with 256 x 256 tiles (gemm8_large.hip): 128 x 128
// tiles, K cut into slices where tiles are few (partial sums in fp32, added in order by a second launch).
#include <type_traits>
#include "block8_common.h"

namespace {
typedef b8_f32x4 f32x4;
typedef b8_i32x8 i32x8;
typedef b8_bf16x8 bf16x8;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

// One block of 4 waves of 64 x 64.  Blocks of k (16 KB of A, 16 KB of B, their scale bytes) arrive by DMA in a ring of DEPTH LDS
// buffers; a block's fragments are read while the previous block's products run, one barrier a block.  DEPTH 4 where a CU has one
// tile, 2 (two tiles a CU, one's loads and stores under the other's products) where there are more than 256: 2048 x 4096 x 4096 with fp32
// results 73 / 62 us, 12 x (64 x 768 x 32768) 125 / 100, but 1536 x 4096 x 1792 (168 tiles) 24 / 34.
// LDS rows of 128 bytes, 16-byte chunks XOR-swizzled with bits 1..3 of the row.  Row p of a 64-row half is matrix row
// (p % 16) * 4 + p / 16 (A) or c(p % 16) * 4 + p / 16 (B, c(4 q + i) = 4 i + q): a lane's four fragments are four consecutive rows,
// so their scales are one dword, and its accumulators of the four B fragments are four consecutive columns.
// Bound: a block of k is 64 instructions of 32 cycles (four waves: 512 cycles of each SIMD; exact products 1024) against 96 KB through
// LDS (768 cycles); with every CU busy it takes 0.6 us (exact products: 1.0), two together 0.85 (1.6).  2048 x 4096 x 4096: 39 us = 1760
// TFLOP/s.
constexpr int OPB = 128 * 128, STG = 2 * OPB + 512;
constexpr int PIECES = 9;                            // DMA instructions of a wave per block of k
extern __shared__ __attribute__((aligned(1024))) unsigned char t8_smem[];

template <int DT, int FA, int FB, int DEPTH> __global__ __launch_bounds__(256, DEPTH == 2 ? 2 : 1) void gemm8_kernel(Gemm8Args g) {
    constexpr bool WIDE = DT != CLT_DT_BF16;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
    const int wb = w >> 1, wa = w & 1;
    // every XCD (block index mod 8) works on a contiguous range of tiles, so that its L2 holds their operands once (12 x (768 x 4096 x 768):
    // 61 -> 39 us); not where K is cut: the columns of one slice lie in a few of an L2's channels (512 x 8192 x 768: 18 -> 21 us)
    const int xcd = blockIdx.x & 7, per = gridDim.x >> 3, more = gridDim.x & 7;
    const int lid = g.slices > 1 ? blockIdx.x : (xcd < more ? xcd * (per + 1) : more + xcd * per) + (blockIdx.x >> 3);
    int a0, b0, slice = 0, batch;
    if (g.first) {                                       // a quarter of one of the large tiles that are left
        const B8Tile t = b8_tile(g, g.first + (lid >> 2));
        a0 = t.a0 + (lid & 1) * 128; b0 = t.b0 + (lid >> 1 & 1) * 128;
        batch = t.batch;
        if (a0 >= g.M || b0 >= g.N) return;
    } else {
        const int nwg = g.tilesA * g.tilesB, tile = lid % nwg, id = lid / nwg;
        slice = id % g.slices; batch = id / g.slices;
        a0 = tile % g.tilesA * 128; b0 = tile / g.tilesA * 128;
    }
    const int k0 = slice * g.slice_kb, nk = min(g.slice_kb, g.KB - k0);

    // DMA: piece i of wave w fills LDS rows (4 i + w) * 8 .. + 7 of an operand.  Ranges end behind the tile's last row: rows past the
    // matrix arrive as zeros (the range check counts the scalar offset, here the block of k, too).
    auto rsrc = [](const void* p, long records) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)records, 0x00020000); };
    __amdgpu_buffer_rsrc_t rA = rsrc(g.a + batch * g.ba + (long)a0 * g.lda, (long)min(g.M - a0, 128) * g.lda);
    __amdgpu_buffer_rsrc_t rB = rsrc(g.b + batch * g.bb + (long)b0 * g.ldb, (long)min(g.N - b0, 128) * g.ldb);
    const int srow = (int)(w & 1 ? g.ldbs : g.ldas);     // even waves bring A's scale bytes, odd waves B's
    __amdgpu_buffer_rsrc_t rS = rsrc(w & 1 ? g.bs + batch * g.bbs + b0 : g.as + batch * g.bas + a0,
                                     (long)(g.KB - 1) * srow + min(((w & 1 ? g.N - b0 : g.M - a0) + 3) & ~3, 128));
    const __amdgpu_buffer_rsrc_t none = rsrc(g.a, 0);
    const int q8 = (w & 1) * 8 + (lane >> 3), ch = (lane & 7) ^ ((q8 >> 1) & 7);
    const int vA = (q8 * 4 + (w >> 1)) * (int)g.lda + ch * 16;
    const int vB = ((((q8 & 3) << 2) | (q8 >> 2)) * 4 + (w >> 1)) * (int)g.ldb + ch * 16;
    auto stage = [&](int k) {                            // block k of the slice (behind the end: nothing, zeros arrive)
        unsigned char* base = t8_smem + (k & (DEPTH - 1)) * STG;
        const bool live = k < nk;
        const __amdgpu_buffer_rsrc_t pa = live ? rA : none, pb = live ? rB : none, ps = live ? rS : none;
        const int kb = k0 + k;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int rows = (i & 1) * 2 + (i >> 1) * 64;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(pa, (lds_void*)(base + (i * 4 + w) * 1024), 16, vA + rows * (int)g.lda, kb * 128, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(pb, (lds_void*)(base + OPB + (i * 4 + w) * 1024), 16, vB + rows * (int)g.ldb, kb * 128, 0, 0);
        }
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ps, (lds_void*)(base + 2 * OPB + (w & 1) * 256), 4, lane * 4, kb * srow, 0, 0);
    };
#pragma unroll
    for (int k = 0; k < DEPTH; ++k) stage(k);

    f32x4 acc[4][4];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int x = fr >> 1, lo = (fq ^ x) << 4;
    const int rowA = (wa * 64 + fr) * 128, rowB = OPB + (wb * 64 + fr) * 128;
    const int scA = 2 * OPB + wa * 64 + fr * 4, scB = 2 * OPB + 256 + wb * 64 + (((fr & 3) << 2) | (fr >> 2)) * 4;
    i32x8 fa[2][4], fb[2][4];
    int sa[2], sb[2];
    auto ld = [&](const unsigned char* p) {              // chunks fq and fq + 4: any split of the block's k that both operands share
        const i32x4 u = *reinterpret_cast<const i32x4*>(p + lo), v = *reinterpret_cast<const i32x4*>(p + (lo ^ 64));
        return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto fragments = [&](int k, int s) {
        const unsigned char* base = t8_smem + (k & (DEPTH - 1)) * STG;
        sa[s] = *reinterpret_cast<const int*>(base + scA);
        sb[s] = *reinterpret_cast<const int*>(base + scB);
#pragma unroll
        for (int n = 0; n < 4; ++n) { fa[s][n] = ld(base + rowA + n * 2048); fb[s][n] = ld(base + rowB + n * 2048); }
    };
    auto products = [&](int s) {
        if constexpr (!WIDE) {
#define G8_MFMA(M_, N_) acc[M_][N_] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[s][M_], fa[s][N_], acc[M_][N_], FB, FA, M_, sb[s], N_, sa[s]);
#define G8_ROW(M_) G8_MFMA(M_, 0) G8_MFMA(M_, 1) G8_MFMA(M_, 2) G8_MFMA(M_, 3)
            G8_ROW(0) G8_ROW(1) G8_ROW(2) G8_ROW(3)
#undef G8_ROW
#undef G8_MFMA
        } else {
            float xa[4], xb[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                xa[n] = __uint_as_float((((uint32_t)sa[s] >> (8 * n)) & 0xffu) << 23);
                xb[n] = __uint_as_float((((uint32_t)sb[s] >> (8 * n)) & 0xffu) << 23);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bf16x8 ha[4], hb[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    ha[n] = widen8<FA>((uint32_t)fa[s][n][2 * j], (uint32_t)fa[s][n][2 * j + 1], xa[n]);
                    hb[n] = widen8<FB>((uint32_t)fb[s][n][2 * j], (uint32_t)fb[s][n][2 * j + 1], xb[n]);
                }
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int n = 0; n < 4; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hb[m], ha[n], acc[m][n], 0, 0, 0);
            }
        }
    };
    // this wave's pieces of the next block have landed (the blocks behind it may be on their way) and its reads are complete
#define G8_NEXT() asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"((DEPTH - 2) * PIECES) : "memory")
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"((DEPTH - 1) * PIECES) : "memory");
    fragments(0, 0);
    int k = 0;
    for (; k + 1 < nk; k += 2) {
        G8_NEXT();
        fragments(k + 1, 1);
        stage(k + DEPTH);
        products(0);
        G8_NEXT();
        fragments(k + 2, 0);
        stage(k + 1 + DEPTH);
        products(1);
    }
    if (k < nk) products(0);
#undef G8_NEXT
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // no DMA into this block's LDS outlives it

    // for (n, i) a lane has row 4 fr + n and four columns 4 (4 i + fq) ..
    const bool part = g.part != nullptr;
    const float* bias = g.bias && !part ? g.bias + batch * g.bbias : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int col = b0 + wb * 64 + (i * 4 + fq) * 4, valid = g.N - col;
        f32x4 bv = {0.0f, 0.0f, 0.0f, 0.0f};
        if (bias)
#pragma unroll
            for (int j = 0; j < 4; ++j) bv[j] = bias[min(col + j, g.N - 1)];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int row = a0 + wa * 64 + fr * 4 + n;
            if (row >= g.M || valid <= 0) continue;
            const f32x4 v = f32x4{acc[0][n][i], acc[1][n][i], acc[2][n][i], acc[3][n][i]} + bv;
            if (part) b8_store4<CLT_DT_F32>(g.part, (((long)slice * g.batch + batch) * g.M + row) * g.N + col, v, valid, 0);
            else b8_store4<DT>(g.c, batch * g.bc + (long)row * g.ldc + col, v, valid, g.accumulate);
        }
    }
}

// partial sums of the slices -> C, slices in order; four columns a thread
template <int DT> __global__ __launch_bounds__(256) void gemm8_fold_kernel(Gemm8Args g, int quads, long total) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    const long r = id / quads;                           // row of the whole batch
    const int col = (int)(id - r * quads) * 4, valid = g.N - col, batch = (int)(r / g.M), row = (int)(r - (long)batch * g.M);
    const long step = (long)g.batch * g.M * g.N;
    const float* p = g.part + r * g.N + col;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    // (a row's last columns: each element by itself, the ones past the end repeated and dropped)
    const bool whole = valid >= 4;
    const int c1 = min(1, valid - 1), c2 = min(2, valid - 1);
    auto sum = [&](int k, auto n) {                      // n requests at a time, added in order
        constexpr int R = decltype(n)::value;
        f32x4 v[R];
        if (whole) {
#pragma unroll
            for (int j = 0; j < R; ++j) v[j] = *reinterpret_cast<const b8_f32x4_u*>(p + (k + j) * step);
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j) { const float* q = p + (k + j) * step; v[j] = f32x4{q[0], q[c1], q[c2], 0.0f}; }
        }
#pragma unroll
        for (int j = 0; j < R; ++j) s += v[j];
    };
    int k = 0;
    for (; k + 8 <= g.slices; k += 8) sum(k, std::integral_constant<int, 8>{});
    for (; k + 2 <= g.slices; k += 2) sum(k, std::integral_constant<int, 2>{});
    if (k < g.slices) sum(k, std::integral_constant<int, 1>{});
    if (g.bias)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += g.bias[batch * g.bbias + min(col + j, g.N - 1)];
    b8_store4<DT>(g.c, batch * g.bc + (long)row * g.ldc + col, s, valid, g.accumulate);
}

// Which tiles, and into how many slices K is cut: the least of the times that these measurements add up to (us):
//                                             bf16 results            exact products (fp32 results)
//   128 x 128 tiles, up to 256                7 + 0.6 a block of k    7 + 1.0
//     a pass of up to 512, two a CU          10.5 + 0.85              9 + 1.6
//     up to 256 that are left                 5 + 0.8                 5 + 0.95
//   256 x 256 tiles, a pass of up to 256      9 + 1.3                15 + 2.9
//   slices: the second launch 4, the partial sums 8 bytes an element and slice at 5 TB/s
// e.g. (M, K, N; small against large tiles, us) 2048 x 4096 x 4096: 39 / 46 (bf16), 62 / 98 (fp32); 2304 x 4096 x 4096: 67 / 47 and 92 / 98;
// 4096 x 4096 x 4096: 78 / 54 and 131 / 111; whole against sliced: 128 x 32768 x 768: 132 / 21; 1024 x 4096 x 768: 23 / 18;
// 1024 x 2048 x 2048: 16.3 / 20.1.
// A slice keeps 4 blocks (the ring), slices of the large form are equal, partial sums take at most 256 MB.  The large form is not
// for less than 128 rows on either side: such a tile is more than half empty.
// Large tiles that do not fill their last pass may be left to small ones (a second launch: 3): 4352 x 4096 x 4096 whole / shared 93 / 77
// and 188 / 139; 12 x (4096 x 8192 x 768): 346 / 326 and 584 / 511.
struct Plan { long large; int slices; };                 // large tiles (0: small ones only; else the rest are small), slices of K
double small_time(long tiles, double kb, bool wide) {
    if (tiles <= 256) return 7.0 + kb * (wide ? 1.0 : 0.6);
    const double pass = wide ? 9.0 + 1.6 * kb : 10.5 + 0.85 * kb, rest = 5.0 + kb * (wide ? 0.95 : 0.8);
    const long left = tiles % 512;
    return (double)(tiles / 512) * pass + (left > 256 ? pass : left ? rest : 0.0);
}
Plan plan_of(int M, int N, int KB, int batch, bool wide) {
    const double elements = (double)batch * M * N;
    Plan best = {0, 1};
    double least = 1e30;
    for (int large = 0; large < 2; ++large) {
        const long side = large ? 256 : 128, tiles = ((M - 1) / side + 1) * ((N - 1) / side + 1) * batch, full = tiles / 256 * 256;
        if (large && (M < 128 || N < 128 || KB < 1 || tiles > 0x3fffffffL)) break;
        auto pass = [&](double kb) { return wide ? 15.0 + 2.9 * kb : 9.0 + 1.3 * kb; };
        for (long s = 1; s == 1 || (s * tiles <= 256 && s * 4 <= KB && s * elements * 4.0 <= 268435456.0); ++s) {
            if (large && s > 1 && (KB % s || 1024L * N > 0x7fffffffL)) continue;       // (offsets of the partial sums: 32 bits)
            const long per = (KB + s - 1) / s, used = per ? (KB + per - 1) / per : 1;
            const double t = (large ? (double)((tiles * used + 255) / 256) * pass(per) : small_time(tiles * used, per, wide)) +
                             (used > 1 ? 4.0 + used * elements * 8.0 / 5e6 : 0.0);
            if (t < least) { least = t; best = {large ? tiles : 0, (int)used}; }
        }
        if (large && full && full < tiles) {
            const double t = (double)(full / 256) * pass(KB) + small_time(4 * (tiles - full), KB, wide) + 3.0;
            if (t < least) { least = t; best = {full, 1}; }
        }
    }
    return best;
}

// of a call: where the rows of C lie further apart than the large form's 32-bit offsets reach, small tiles
Plan plan_of_call(int M, int N, int KB, int batch, int c_dtype, long ldc) {
    Plan p = plan_of(M, N, KB, batch, c_dtype != CLT_DT_BF16);
    if (p.slices == 1 && 256 * ldc * 4 > 0x7fffffffL) p.large = 0;
    return p;
}

template <int DT, int FA, int FB, int DEPTH> int launch_depth(const Gemm8Args& g, long blocks, hipStream_t st) {
    const auto f = gemm8_kernel<DT, FA, FB, DEPTH>;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, DEPTH * STG) != hipSuccess) return CLT_ERR_LAUNCH;
    f<<<dim3((unsigned)blocks), dim3(256), DEPTH * STG, st>>>(g);
    CLT_LAUNCH_CHECK();
    return CLT_OK;
}
template <int DT, int FA, int FB> int launch_fmt(const Gemm8Args& g, long blocks, hipStream_t st) {
    return blocks > 256 ? launch_depth<DT, FA, FB, 2>(g, blocks, st) : launch_depth<DT, FA, FB, 4>(g, blocks, st);
}
template <int DT> int fold(const Gemm8Args& g, hipStream_t st) {
    const int quads = (g.N - 1) / 4 + 1;
    const long total = (long)g.batch * g.M * quads, fold = (total + 255) / 256;
    if (!b8_fits(fold, 256)) return CLT_ERR_RANGE;
    gemm8_fold_kernel<DT><<<dim3((unsigned)fold), dim3(256), 0, st>>>(g, quads, total);
    CLT_LAUNCH_CHECK();
    return CLT_OK;
}
template <int DT> int launch(const Gemm8Args& g, int fa, int fb, long blocks, hipStream_t st) {
    const int rc = fa == 0 ? (fb == 0 ? launch_fmt<DT, 0, 0>(g, blocks, st) : launch_fmt<DT, 0, 1>(g, blocks, st))
                           : (fb == 0 ? launch_fmt<DT, 1, 0>(g, blocks, st) : launch_fmt<DT, 1, 1>(g, blocks, st));
    return rc != CLT_OK || !g.part ? rc : fold<DT>(g, st);
}
}  // namespace

extern "C" size_t clt_gemm8_workspace_bytes(int M, int N, int K, int batch) {
    if (M <= 0 || N <= 0 || K <= 0 || batch <= 0) return 0;
    const int KB = (int)(up128(K) / 128);
    const int s = plan_of(M, N, KB, batch, false).slices, w = plan_of(M, N, KB, batch, true).slices, most = s > w ? s : w;
    return most > 1 ? (size_t)most * batch * M * N * 4 : 0;
}

extern "C" int clt_gemm8_plan(int M, int N, int K, int batch, int c_dtype, long ldc, int64_t* plan) {
    if (M <= 0 || N <= 0 || K < 0 || batch <= 0 || c_dtype < 0 || c_dtype > 2 || ldc < N || !plan) return CLT_ERR_SHAPE;
    const Plan p = plan_of_call(M, N, (int)(up128(K) / 128), batch, c_dtype, ldc);
    plan[0] = ((M - 1) / 256 + 1L) * ((N - 1) / 256 + 1) * batch; plan[1] = p.large; plan[2] = p.slices;
    return CLT_OK;
}

extern "C" int clt_gemm8(const void* a, const void* a_scale, int a_format, long lda, long ldas, long a_batch, long as_batch,
                         const void* b, const void* b_scale, int b_format, long ldb, long ldbs, long b_batch, long bs_batch,
                         void* c, int c_dtype, long ldc, long c_batch, const float* bias, long bias_batch, int M, int N, int K,
                         int batch, int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
    if (M <= 0 || N <= 0 || K < 0 || batch <= 0 || c_dtype < 0 || c_dtype > 2 || (a_format & ~1) || (b_format & ~1) || !c) return CLT_ERR_SHAPE;
    if (accumulate && c_dtype != CLT_DT_F32) return CLT_ERR_SHAPE;                 // (a 16-bit sum would round at every call)
    const int KB = (int)(up128(K) / 128);
    if (ldc < N || (KB && (!a || !a_scale || !b || !b_scale || lda < up128(K) || ldb < up128(K) || ldas < M || ldbs < N))) return CLT_ERR_SHAPE;
    if (KB && (!aligned16(a) || !aligned16(b) || lda % 16 || ldb % 16 || a_batch % 16 || b_batch % 16)) return CLT_ERR_ALIGN;
    if (KB && (((uintptr_t)a_scale & 3) || ((uintptr_t)b_scale & 3) || ldas % 4 || ldbs % 4 || as_batch % 4 || bs_batch % 4)) return CLT_ERR_ALIGN;
    if (((uintptr_t)c & (c_dtype == CLT_DT_F32 ? 3 : 1)) || ((uintptr_t)bias & 3)) return CLT_ERR_ALIGN;
    // 32-bit offsets inside a tile's rows and over an operand's scale bytes
    if (KB && (256 * lda > 0x7fffffffL || 256 * ldb > 0x7fffffffL || KB * ldas > 0x7ffffeffL || KB * ldbs > 0x7ffffeffL)) return CLT_ERR_RANGE;
    Gemm8Args g = {static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(a_scale), static_cast<const uint8_t*>(b),
                   static_cast<const uint8_t*>(b_scale), c, bias, lda, ldas, ldb, ldbs, ldc, a_batch, as_batch, b_batch, bs_batch,
                   c_batch, bias_batch, M, N, KB, (M - 1) / 128 + 1, (N - 1) / 128 + 1, accumulate, batch, 0u, 0u, 0u, 1, KB, nullptr, 0, 0};
    const hipStream_t st = as_stream(stream);
    const Plan plan = plan_of_call(M, N, KB, batch, c_dtype, ldc);
    g.slices = plan.slices;
    if (g.slices > 1) {
        if (!workspace || !aligned16(workspace) || workspace_bytes < (size_t)g.slices * batch * M * N * 4) return CLT_ERR_WORKSPACE;
        g.part = static_cast<float*>(workspace);
        g.slice_kb = (KB + g.slices - 1) / g.slices;
    }
    long blocks = (long)g.tilesA * g.tilesB * batch * g.slices;
    if (plan.large) {
        b8_tile_order(g);
        const long tiles = (long)g.tilesA * g.tilesB * batch;
        const int rc = clt_internal_gemm8_large(g, a_format, b_format, c_dtype, (int)plan.large, st);
        if (rc != CLT_OK) return rc;
        if (g.part) return c_dtype == CLT_DT_F32 ? fold<CLT_DT_F32>(g, st) : c_dtype == CLT_DT_BF16 ? fold<CLT_DT_BF16>(g, st) : fold<CLT_DT_F16>(g, st);
        if (plan.large == tiles) return CLT_OK;
        g.first = (int)plan.large;
        blocks = 4 * (tiles - plan.large);
    }
    if (!b8_fits(blocks, 256)) return CLT_ERR_RANGE;
    return c_dtype == CLT_DT_F32 ? launch<CLT_DT_F32>(g, a_format, b_format, blocks, st)
           : c_dtype == CLT_DT_BF16 ? launch<CLT_DT_BF16>(g, a_format, b_format, blocks, st)
                                    : launch<CLT_DT_F16>(g, a_format, b_format, blocks, st);
}
