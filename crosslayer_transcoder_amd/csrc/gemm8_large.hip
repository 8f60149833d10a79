// The large form of clt_gemm8 (see gemm8.hip for the operator and its two inner products): 256 x 256 tiles for shapes that fill
// the chip with them.
//
// One block of 4 waves per CU, 2 x 2 waves of 128 x 128 (256 accumulators and ~200 other registers a lane: one wave per SIMD has
// all 512).  The wave tile is what the LDS allows: a block of 128 k costs a wave 16 fragments of 32 bytes a lane = 32 KB of
// reads for 64 matrix instructions of 32 cycles; four waves read 128 KB in those 2048 cycles, half of the LDS's rate, where 8
// waves of 128 x 64 would need three quarters and wait for it.
// Operands go global -> LDS by DMA, two buffers of 64 KB, one 128-byte block of k at a time; the scale bytes of the block (256 + 256)
// and the tile's bias ride along.  The grid is persistent; the epilogue's LDS is its own, so both buffers already receive the
// next tile's first two blocks while this tile's results are stored.
//
// Row order.  LDS row p of a 128-row half holds matrix row (p % 16) * 8 + p / 16 (A) or c(p % 16) * 8 + p / 16 with
// c(4 q + i) = 4 i + q (B), so fragment j of a wave is rows 8 * lane + j: (a) the scale bytes of a lane's eight fragments are eight
// consecutive bytes — one 8-byte read per operand and block, the instruction picks its byte by op_sel; (b) a lane's
// accumulators of the eight B fragments are eight consecutive columns of C — 16 bytes of 16-bit results, 32 of fp32 — and four
// lanes make 64 / 128 consecutive bytes.  bf16 results pass through a 4 KB slab of LDS a wave, so that 256 bytes of a row leave
// together, and past the caches, which hold the operands' panels (4096 x 768 x 32768 x 12: 1728 -> 1462 us; without the slab the
// uncached stores are slower than cached ones, 1765 us).
// Bound: the matrix units, at what clock the power leaves them (8192^3: 373 .. 437 us from card to card = 2.5 .. 2.9 PFLOP/s; the large library
// product in 8 bits 2.9); with a short contraction the stores next to them (K = 768, 12 layers, 3.2 GB of results: 1410 .. 1440 us; 1530 us
// where the rows of a layer lie 786 KB apart; matrix units busy 35 % of the time).  Those are times of a row of launches; the first few of a
// process take 1.6 .. 1.9 ms.
#include <type_traits>
#include "block8_common.h"

namespace {
typedef b8_f32x4 f32x4;
typedef b8_i32x8 i32x8;
typedef b8_bf16x8 bf16x8;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
constexpr int OPB = 256 * 128;                        // one operand's block in LDS
constexpr int STG = 2 * OPB;
constexpr int SCALE_BASE = 2 * STG;                   // per buffer: 256 scale bytes of A, 256 of B
constexpr int BIAS_BASE = SCALE_BASE + 2 * 512;       // four slots of 256 floats (a tile's, while up to two more are on their way)
constexpr int SLAB_BASE = BIAS_BASE + 4 * 1024;       // a slab a wave: 16 rows of 128 16-bit results (padded against conflicts)
constexpr int SLAB_ROW = 256 + 16, SLAB = 16 * SLAB_ROW;
constexpr int LDS_BYTES = SLAB_BASE + 4 * SLAB;
static_assert(LDS_BYTES <= 160 * 1024, "LDS");
extern __shared__ __attribute__((aligned(1024))) unsigned char g8_smem[];
typedef __attribute__((address_space(3))) void lds_void;

template <int N, class F> __device__ __forceinline__ void unroll(F f) {
    if constexpr (N > 0) { unroll<N - 1>(f); f(std::integral_constant<int, N - 1>{}); }
}

typedef b8_u32x4_u u32x4_u;
typedef b8_f32x4_u f32x4_u;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, long records) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)records, 0x00020000);
}

template <int DT, int FA, int FB>
__global__ __launch_bounds__(256, 1) void gemm8_large_kernel(Gemm8Args g, int total) {
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wb = w >> 1, wa = w & 1, fr = lane & 15, fq = lane >> 4;
    const int nk = g.slice_kb;                            // blocks of k of a tile (K, or a slice of it)
    auto decode = [&](int vb) { return b8_tile(g, vb); };

    // ---- DMA: piece i of wave w fills LDS rows (4 i + w) * 8 .. + 7; a lane supplies 16 bytes (chunk XOR-swizzled with bits 1..3 of the
    // row).  Descriptors start at the tile's first row and end behind its last one: rows past the matrix arrive as zeros.
    const int q8 = (w & 1) * 8 + (lane >> 3);             // LDS row mod 16
    const int ch = (lane & 7) ^ ((q8 >> 1) & 7);
    const int vA = (q8 * 8 + (w >> 1)) * (int)g.lda + ch * 16;
    const int vB = ((((q8 & 3) << 2) | (q8 >> 2)) * 8 + (w >> 1)) * (int)g.ldb + ch * 16;
    __amdgpu_buffer_rsrc_t rA, rB, rS, rBias;
    auto aim = [&](const B8Tile& t) {
        // (a slice of K starts slice_kb blocks into the rows: the range ends where the last row does)
        const long k0 = (long)t.slice * g.slice_kb;
        rA = rsrc(g.a + t.batch * g.ba + (long)t.a0 * g.lda + k0 * 128, (long)min(g.M - t.a0, 256) * g.lda - k0 * 128);
        rB = rsrc(g.b + t.batch * g.bb + (long)t.b0 * g.ldb + k0 * 128, (long)min(g.N - t.b0, 256) * g.ldb - k0 * 128);
        // scale bytes (the dwords that hold a row's byte): even waves A's, odd waves B's — twice the same bytes instead of a branch
        const uint8_t* sp = w & 1 ? g.bs + t.batch * g.bbs + k0 * g.ldbs + t.b0 : g.as + t.batch * g.bas + k0 * g.ldas + t.a0;
        // (the range check counts the scalar offset, here the block's scale row, too: the range ends with this tile's rows in the last one)
        rS = rsrc(sp, (long)(nk - 1) * (w & 1 ? g.ldbs : g.ldas) + min(((w & 1 ? g.N - t.b0 : g.M - t.a0) + 3) & ~3, 256));
        if (g.bias) rBias = rsrc(g.bias + t.batch * g.bbias + t.b0, min(g.N - t.b0, 256) * 4L);
    };
    auto piece = [&](int buf, int kt, int i) {
        unsigned char* base = g8_smem + buf * STG + (i * 4 + w) * 1024;
        const int rows = (i & 3) * 2 + (i >> 2) * 128;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rA, (lds_void*)base, 16, vA + rows * (int)g.lda, kt * 128, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rB, (lds_void*)(base + OPB), 16, vB + rows * (int)g.ldb, kt * 128, 0, 0);
    };
    const int srow = (int)(w & 1 ? g.ldbs : g.ldas);
    auto scale_piece = [&](int buf, int kt) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rS, (lds_void*)(g8_smem + SCALE_BASE + buf * 512 + (w & 1) * 256), 4, lane * 4, kt * srow, 0, 0);
    };
    // ---- fragment addresses: LDS row j * 16 + fr of the wave's half
    const int x = fr >> 1;
    const int cB = ((fr & 3) << 2) | (fr >> 2);
    const int scA = SCALE_BASE + wa * 128 + fr * 8, scB = SCALE_BASE + 256 + wb * 128 + cB * 8;
    const int rowA = (wa * 128 + fr) * 128, rowB = OPB + (wb * 128 + fr) * 128;

    f32x4 acc[8][8];
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
        for (int n = 0; n < 8; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int NST = DT == CLT_DT_F32 ? 63 : 32;       // stores of an interior tile per lane (63: the counter's limit, 64 are issued)

    // ---- the stream of k-blocks: staging runs two blocks ahead of the products, across tiles
    int vb = blockIdx.x, svb = vb, skt = 0, sslot = 0, slot = 0, buf = 0;
    B8Tile t = decode(vb);
    auto enter = [&](const B8Tile& e) {                     // staging enters tile svb = e
        if (svb < total) {
            aim(e);
            if (g.bias && w == 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(rBias, (lds_void*)(g8_smem + BIAS_BASE + sslot * 1024), 16, lane * 16, 0, 0, 0);
        } else { rA = rsrc(g.a, 0); rB = rsrc(g.b, 0); rS = rsrc(g.as, 0); }      // nothing left: zeros arrive in a buffer nobody reads
    };
    // (moved on at the head of a block, where the staging state is needed: control flow behind the matrix instructions would let the
    // compiler sink them, which have no side effects, below everything they are meant to overlap)
    auto advance = [&](const B8Tile& next) {
        if (++skt == nk) { skt = 0; svb += (int)gridDim.x; sslot = (sslot + 1) & 3; enter(next); }
    };
    enter(t);
    for (int k = 0; k < 2; ++k) {
        if (k) advance(decode(svb + (int)gridDim.x));
        scale_piece(k, skt);
#pragma unroll
        for (int i = 0; i < 8; ++i) piece(k, skt, i);
    }
    B8Tile nt = decode(svb + (int)gridDim.x);               // the tile staging enters next (decoded off the critical path)
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    // Buffer handover: this wave's reads of the block are complete and its pieces of the next block have landed; then all waves'.
    // Vector memory retires in order: in a tile's first block the next block's pieces are older than the previous tile's stores,
    // which may stay outstanding.  One asm statement: the scheduling region around it stays whole.
    auto handover = [](int kt) {
        asm volatile("s_cmp_eq_u32 %0, 0\n\ts_cbranch_scc1 1f\n\ts_waitcnt vmcnt(0)\n1:\ts_waitcnt vmcnt(%1) lgkmcnt(0)\n\ts_barrier" ::"s"(kt), "i"(NST) : "scc", "memory");
    };
    const int lo = (fq ^ x) << 4;
    int aA = rowA, aB = rowB, aSA = scA, aSB = scB;       // the block's addresses; the other buffer's by XOR
    auto flip = [&]() { aA ^= STG; aB ^= STG; aSA ^= 512; aSB ^= 512; };

    // fragments of the current block (and, from its second half on, of the next)
    i32x8 fa[8], fb[8];
    i32x2 sa, sb;
    auto ld = [&](int at, int off) {                      // chunks fq and fq + 4: any split of the block's k that both operands share
        const i32x4 u = *reinterpret_cast<const i32x4*>(g8_smem + (at + lo) + off), v = *reinterpret_cast<const i32x4*>(g8_smem + (at + (lo ^ 64)) + off);
        return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    sa = *reinterpret_cast<const i32x2*>(g8_smem + aSA);
    sb = *reinterpret_cast<const i32x2*>(g8_smem + aSB);
#pragma unroll
    for (int n = 0; n < 8; ++n) fa[n] = ld(aA, n * 2048);
#pragma unroll
    for (int m = 0; m < 4; ++m) fb[m] = ld(aB, m * 2048);

    for (;;) {
        for (int kt = 0; kt < nk; ++kt) {
            advance(nt);
            // 64 instructions a block.  First half: B fragments 0..3, A fragments fastest; B fragments 4..7 are read meanwhile.
            // Handover.  Second half: A fragment by A fragment against B fragments 4..7; the block after next is staged, the
            // next block's B fragments 0..3 are read, and every A fragment is replaced by the next block's after its last use.
            auto mfma = [&](auto m_, auto n_) {
                constexpr int m = decltype(m_)::value, n = decltype(n_)::value;
                acc[m][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[m], fa[n], acc[m][n], FB, FA, m & 3, sb[m >> 2], n & 3, sa[n >> 2]);
                __builtin_amdgcn_sched_barrier(0);
            };
            unroll<4>([&](auto m) {
                fb[m + 4] = ld(aB, (m + 4) * 2048);
                __builtin_amdgcn_sched_barrier(0);
                unroll<8>([&](auto n) { mfma(m, n); });
            });
            handover(kt);
            flip();
            const i32x2 sa_n = *reinterpret_cast<const i32x2*>(g8_smem + aSA), sb_n = *reinterpret_cast<const i32x2*>(g8_smem + aSB);
            scale_piece(buf, skt);
            unroll<8>([&](auto n) {
                unroll<4>([&](auto j) {
                    if constexpr (j < 2 && n < 4) piece(buf, skt, 2 * n + j);
                    if constexpr (j == 2 && n >= 4) fb[n - 4] = ld(aB, (n - 4) * 2048);
                    mfma(std::integral_constant<int, 4 + decltype(j)::value>{}, n);
                });
                fa[n] = ld(aA, n * 2048);
            });
            sa = sa_n; sb = sb_n;
            buf ^= 1;
        }
        const B8Tile cur = t;
        const int cslot = slot;
        vb += (int)gridDim.x;
        slot = (slot + 1) & 3;
        const bool more = vb < total;
        if (more) t = decode(vb);
        nt = decode(svb + (int)gridDim.x);
        // ---- results: for (n, i) a lane has row 8 fr + n and eight columns 8 (4 i + fq) .. of its wave's 128 x 128: 16 bytes.  Row by row
        // (n) they pass through the wave's own slab of LDS, so that 16 lanes store 256 consecutive bytes.
        typedef typename Elem<DT>::type T;
        const bool interior = cur.a0 + 256 <= g.M && cur.b0 + 256 <= g.N, has_bias = g.bias != nullptr;
        const float* bl = reinterpret_cast<const float*>(g8_smem + BIAS_BASE + cslot * 1024) + wb * 128 + fq * 8;
        T* ctile = static_cast<T*>(g.c) + cur.batch * g.bc + cur.slice * g.slice_stride + (long)(cur.a0 + wa * 128) * g.ldc + cur.b0 + wb * 128;
        unsigned char* slab = g8_smem + SLAB_BASE + w * SLAB;
        const int wr = fr * SLAB_ROW + fq * 16, rd = fq * SLAB_ROW + fr * 16;
        const unsigned at = (unsigned)(fq * 8 * (int)g.ldc + fr * 8) * (unsigned)sizeof(T);      // a lane's offset: 32 bits (host check)
        const int rows = g.M - (cur.a0 + wa * 128 + fq * 8), cols = g.N - (cur.b0 + wb * 128 + fr * 8);
        auto put = [&](int n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 lo = f32x4{acc[0][n][i], acc[1][n][i], acc[2][n][i], acc[3][n][i]};
                f32x4 hi = f32x4{acc[4][n][i], acc[5][n][i], acc[6][n][i], acc[7][n][i]};
                if (has_bias) { lo += *reinterpret_cast<const f32x4*>(bl + i * 32); hi += *reinterpret_cast<const f32x4*>(bl + i * 32 + 4); }
                *reinterpret_cast<u32x4*>(slab + wr + i * 64) = u32x4{pack_out16<DT>(lo[0], lo[1]), pack_out16<DT>(lo[2], lo[3]), pack_out16<DT>(hi[0], hi[1]), pack_out16<DT>(hi[2], hi[3])};
            }
        };
        if constexpr (DT == CLT_DT_F32) {                 // partial sums of a slice
            const int prow = g.M - (cur.a0 + wa * 128 + fr * 8), pcol = g.N - (cur.b0 + wb * 128 + fq * 8);
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    T* p = ctile + (long)(fr * 8 + n) * g.ldc + fq * 8 + i * 32;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const f32x4 v = f32x4{acc[4 * j][n][i], acc[4 * j + 1][n][i], acc[4 * j + 2][n][i], acc[4 * j + 3][n][i]};
                        if (interior || (n < prow && i * 32 + 4 * j + 4 <= pcol)) *reinterpret_cast<f32x4_u*>(p + 4 * j) = v;
                        else if (n < prow)
#pragma unroll
                            for (int e = 0; e < 4; ++e) if (i * 32 + 4 * j + e < pcol) p[4 * j + e] = v[e];
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
        } else {
        put(0);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            u32x4 v[4];                                   // (a wave's LDS operations execute in order: the next row group may follow at once)
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const u32x4*>(slab + rd + k * 4 * SLAB_ROW);
            if (n < 7) put(n + 1);
#pragma unroll
            for (int k = 0; k < 4; ++k) {                 // rows (4 k + fq) * 8 + n
                const u32x4 u = v[k];
                T* p = reinterpret_cast<T*>(reinterpret_cast<char*>(ctile + (long)(k * 32 + n) * g.ldc) + at);
                if (interior || (k * 32 + n < rows && cols >= 8)) __builtin_nontemporal_store((u32x4_u)u, reinterpret_cast<u32x4_u*>(p));
                else if (k * 32 + n < rows)
#pragma unroll
                    for (int j = 0; j < 8; ++j) if (j < cols) p[j] = (T)(u[j >> 1] >> (16 * (j & 1)));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        }
        if (!more) break;
#pragma unroll
        for (int m = 0; m < 8; ++m)
#pragma unroll
            for (int n = 0; n < 8; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!interior) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // (not NST stores: handover could not count)
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // no DMA into this block's LDS outlives it
}

// ---- exact products (fp32 and fp16 results): the codes become bf16 in registers and the products run at the 16-bit rate, so a block of k costs twice the
// cycles for the same LDS bytes: 8 waves of 128 x 64 (B x A; 192 KB of reads in 4096 cycles), two per SIMD, whose conversions run
// under each other's matrix instructions.  Tiles, DMA, row order and the stream of blocks as above; A fragments are 4 rows of a
// 64-row group (row 4 * lane + n).  8192^3: 770 .. 825 us (fp16 results: 740) = 1.33 .. 1.49 PFLOP/s; the large library product in bf16 1.32.
// K = 768, 12 layers: 2640 .. 2720 us for the 6.4 GB of fp32 results, 2160 of fp16.
template <int DT, int FA, int FB>
__global__ __launch_bounds__(512, 2) void gemm8_large_exact_kernel(Gemm8Args g, int total) {
    typedef typename Elem<DT>::type T;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wb = w >> 2, wa = w & 3, fr = lane & 15, fq = lane >> 4;
    const int nk = g.slice_kb;                            // blocks of k of a tile (K, or a slice of it)
    // piece i of wave w fills LDS rows (8 i + w) * 8 .. + 7
    const int q8 = (w & 1) * 8 + (lane >> 3), ch = (lane & 7) ^ ((q8 >> 1) & 7);
    const int vA = (q8 * 4 + (w >> 1)) * (int)g.lda + ch * 16;
    const int vB = ((((q8 & 3) << 2) | (q8 >> 2)) * 8 + (w >> 1)) * (int)g.ldb + ch * 16;
    const int srow = (int)(w & 1 ? g.ldbs : g.ldas);
    __amdgpu_buffer_rsrc_t rA, rB, rS;
    int vb = blockIdx.x, svb = vb, skt = 0, sslot = 0, slot = 0, buf = 0;
    auto enter = [&](const B8Tile& t) {
        if (svb < total) {
            const long k0 = (long)t.slice * g.slice_kb;
            rA = rsrc(g.a + t.batch * g.ba + (long)t.a0 * g.lda + k0 * 128, (long)min(g.M - t.a0, 256) * g.lda - k0 * 128);
            rB = rsrc(g.b + t.batch * g.bb + (long)t.b0 * g.ldb + k0 * 128, (long)min(g.N - t.b0, 256) * g.ldb - k0 * 128);
            const uint8_t* sp = w & 1 ? g.bs + t.batch * g.bbs + k0 * g.ldbs + t.b0 : g.as + t.batch * g.bas + k0 * g.ldas + t.a0;
            rS = rsrc(sp, (long)(nk - 1) * srow + min(((w & 1 ? g.N - t.b0 : g.M - t.a0) + 3) & ~3, 256));
            if (g.bias && w == 2) {
                __amdgpu_buffer_rsrc_t r = rsrc(g.bias + t.batch * g.bbias + t.b0, min(g.N - t.b0, 256) * 4L);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(g8_smem + BIAS_BASE + sslot * 1024), 16, lane * 16, 0, 0, 0);
            }
        } else { rA = rsrc(g.a, 0); rB = rsrc(g.b, 0); rS = rsrc(g.as, 0); }
    };
    auto advance = [&](const B8Tile& next) {
        if (++skt == nk) { skt = 0; svb += (int)gridDim.x; sslot = (sslot + 1) & 3; enter(next); }
    };
    auto piece = [&](int b, int kt, int i) {
        unsigned char* base = g8_smem + b * STG + (i * 8 + w) * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rA, (lds_void*)base, 16, vA + i * 64 * (int)g.lda, kt * 128, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rB, (lds_void*)(base + OPB), 16, vB + ((i >> 1) * 128 + (i & 1) * 4) * (int)g.ldb, kt * 128, 0, 0);
    };
    auto scale_piece = [&](int b, int kt) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rS, (lds_void*)(g8_smem + SCALE_BASE + b * 512 + (w & 1) * 256), 4, lane * 4, kt * srow, 0, 0);
    };
    f32x4 acc[8][4];
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int NST = DT == CLT_DT_F32 ? 32 : 16;       // stores of an interior tile per lane
    B8Tile t = b8_tile(g, vb);
    enter(t);
    for (int k = 0; k < 2; ++k) {
        if (k) advance(b8_tile(g, svb + (int)gridDim.x));
        scale_piece(k, skt);
#pragma unroll
        for (int i = 0; i < 4; ++i) piece(k, skt, i);
    }
    B8Tile nt = b8_tile(g, svb + (int)gridDim.x);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    auto handover = [](int kt) {
        asm volatile("s_cmp_eq_u32 %0, 0\n\ts_cbranch_scc1 1f\n\ts_waitcnt vmcnt(0)\n1:\ts_waitcnt vmcnt(%1) lgkmcnt(0)\n\ts_barrier" ::"s"(kt), "i"(NST) : "scc", "memory");
    };
    const int x = fr >> 1, half = (fq & 1) << 3, cq = fq >> 1, cB = ((fr & 3) << 2) | (fr >> 2);
    int aA = (wa * 64 + fr) * 128 + half + ((cq ^ x) << 4), aB = aA - wa * 64 * 128 + OPB + wb * 128 * 128;
    int aSA = SCALE_BASE + wa * 64 + fr * 4, aSB = SCALE_BASE + 256 + wb * 128 + cB * 8;
    // a lane's 8 codes of a row and step of 32 k; scales as floats
    auto ldw = [&](int at, int off) { return *reinterpret_cast<const i32x2*>(g8_smem + at + off); };
    i32x2 ra[4], rb[8], sv;
    uint32_t su;
    float xa[4], xb[8];
    auto load_scales = [&]() { su = *reinterpret_cast<const uint32_t*>(g8_smem + aSA); sv = *reinterpret_cast<const i32x2*>(g8_smem + aSB); };
    load_scales();
#pragma unroll
    for (int n = 0; n < 4; ++n) ra[n] = ldw(aA, n * 2048);
#pragma unroll
    for (int m = 0; m < 8; ++m) rb[m] = ldw(aB, m * 2048);
    for (;;) {
        // A loop over steps of 32 k: one instruction per accumulator and iteration keeps every accumulator where it is (unrolled by block,
        // the register allocator moves them around).  The step's codes are in registers: A's are converted, then B's fragment by
        // fragment, and the next step's are read behind them.  A block's last step reads the next block: the handover is ahead of it.
        for (int it = 0; it < 4 * nk; ++it) {
            const int step = it & 3;
            if (step == 0) {
                advance(nt);
#pragma unroll
                for (int j = 0; j < 4; ++j) xa[j] = __uint_as_float(((su >> (8 * j)) & 0xffu) << 23);
#pragma unroll
                for (int j = 0; j < 8; ++j) xb[j] = __uint_as_float((((uint32_t)sv[j >> 2] >> (8 * (j & 3))) & 0xffu) << 23);
            }
            if (step == 3) {
                handover(it >> 2);
                aA ^= STG; aB ^= STG; aSA ^= 512; aSB ^= 512;
                load_scales();
                scale_piece(buf, skt);
#pragma unroll
                for (int i = 0; i < 4; ++i) piece(buf, skt, i);
                buf ^= 1;
            }
            const int next = ((it + 1) & 3) << 5, nA = aA ^ next, nB = aB ^ next;
            bf16x8 ha[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                ha[n] = widen8<FA>((uint32_t)ra[n][0], (uint32_t)ra[n][1], xa[n]);
                ra[n] = ldw(nA, n * 2048);
            }
            unroll<8>([&](auto m_) {
                constexpr int m = decltype(m_)::value;
                const bf16x8 hb = widen8<FB>((uint32_t)rb[m][0], (uint32_t)rb[m][1], xb[m]);
                rb[m] = ldw(nB, m * 2048);
#pragma unroll
                for (int n = 0; n < 4; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hb, ha[n], acc[m][n], 0, 0, 0);
            });
        }
        const B8Tile cur = t;
        const int cslot = slot;
        vb += (int)gridDim.x;
        slot = (slot + 1) & 3;
        const bool more = vb < total;
        if (more) t = b8_tile(g, vb);
        nt = b8_tile(g, svb + (int)gridDim.x);
        // ---- results: for (n, i) a lane has row 4 fr + n of its 64 and eight columns 8 (4 i + fq) .. of its 128
        const int r0 = wa * 64 + fr * 4, c0 = wb * 128 + fq * 8;
        const bool interior = cur.a0 + 256 <= g.M && cur.b0 + 256 <= g.N;
        T* ctile = static_cast<T*>(g.c) + cur.batch * g.bc + cur.slice * g.slice_stride + (long)cur.a0 * g.ldc + cur.b0;
        const float* bl = reinterpret_cast<const float*>(g8_smem + BIAS_BASE + cslot * 1024) + c0;
        const bool has_bias = g.bias != nullptr;
        const int rows = g.M - cur.a0 - r0, cols = g.N - cur.b0 - c0;
        const unsigned at = (unsigned)(r0 * (int)g.ldc + c0) * (unsigned)sizeof(T);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 lo = f32x4{acc[0][n][i], acc[1][n][i], acc[2][n][i], acc[3][n][i]};
                f32x4 hi = f32x4{acc[4][n][i], acc[5][n][i], acc[6][n][i], acc[7][n][i]};
                if (has_bias) { lo += *reinterpret_cast<const f32x4*>(bl + i * 32); hi += *reinterpret_cast<const f32x4*>(bl + i * 32 + 4); }
                T* p = reinterpret_cast<T*>(reinterpret_cast<char*>(ctile + (long)n * g.ldc + i * 32) + at);
                if constexpr (DT != CLT_DT_F32) {
                    const u32x4 u = {pack_out16<DT>(lo[0], lo[1]), pack_out16<DT>(lo[2], lo[3]), pack_out16<DT>(hi[0], hi[1]), pack_out16<DT>(hi[2], hi[3])};
                    if (interior || (n < rows && i * 32 + 8 <= cols)) *reinterpret_cast<u32x4_u*>(p) = u;
                    else if (n < rows)
#pragma unroll
                        for (int j = 0; j < 8; ++j) if (i * 32 + j < cols) p[j] = (T)(u[j >> 1] >> (16 * (j & 1)));
                } else if (interior || (n < rows && i * 32 + 8 <= cols)) {
                    if (g.accumulate) { lo += *reinterpret_cast<const f32x4_u*>(p); hi += *reinterpret_cast<const f32x4_u*>(p + 4); }
                    *reinterpret_cast<f32x4_u*>(p) = lo;
                    *reinterpret_cast<f32x4_u*>(p + 4) = hi;
                } else if (n < rows)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (i * 32 + j < cols) { const float v = j < 4 ? lo[j & 3] : hi[j & 3]; p[j] = g.accumulate ? p[j] + v : v; }
                __builtin_amdgcn_sched_barrier(0);
            }
        if (!more) break;
#pragma unroll
        for (int m = 0; m < 8; ++m)
#pragma unroll
            for (int n = 0; n < 4; ++n) acc[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!interior || g.accumulate) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <class F> int launch(F f, int threads, const Gemm8Args& g, int total, hipStream_t st) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES) != hipSuccess) return CLT_ERR_LAUNCH;
    f<<<dim3((unsigned)(total < 256 ? total : 256)), dim3(threads), LDS_BYTES, st>>>(g, total);
    CLT_LAUNCH_CHECK();
    return CLT_OK;
}
// fast: 8-bit instructions (bf16 results, or the partial sums of their slices)
template <int FA, int FB> int launch_dtype(const Gemm8Args& g, int dtype, bool fast, int total, hipStream_t st) {
    if (fast && dtype == CLT_DT_F32) return launch(gemm8_large_kernel<CLT_DT_F32, FA, FB>, 256, g, total, st);
    if (fast) return launch(gemm8_large_kernel<CLT_DT_BF16, FA, FB>, 256, g, total, st);
    if (dtype == CLT_DT_F32) return launch(gemm8_large_exact_kernel<CLT_DT_F32, FA, FB>, 512, g, total, st);
    return launch(gemm8_large_exact_kernel<CLT_DT_F16, FA, FB>, 512, g, total, st);
}
}  // namespace

// dtype: of the product asked for (it picks the instructions); g.part: partial sums go there, unfolded; tiles: the first ones in the order
// of b8_tile (slices: all)
int clt_internal_gemm8_large(const Gemm8Args& g0, int fa, int fb, int dtype, int tiles, hipStream_t st) {
    Gemm8Args g = g0;
    const bool fast = dtype == CLT_DT_BF16;
    if (g.part) {
        g.c = g.part; g.ldc = g.N; g.bc = (long)g.M * g.N; g.slice_stride = g.batch * g.bc;
        g.bias = nullptr; g.accumulate = 0;
        dtype = CLT_DT_F32;
    }
    const int total = tiles * g.slices;
    return fa == 0 ? (fb == 0 ? launch_dtype<0, 0>(g, dtype, fast, total, st) : launch_dtype<0, 1>(g, dtype, fast, total, st))
                   : (fb == 0 ? launch_dtype<1, 0>(g, dtype, fast, total, st) : launch_dtype<1, 1>(g, dtype, fast, total, st));
}
