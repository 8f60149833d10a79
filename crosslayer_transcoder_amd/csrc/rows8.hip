// y [T][L][N] = x [T][L][K] * w [L][N][K]^T + bias for few tokens (T <= 32) and kept 8-bit weights: the serving form of a linear
// map.  x is packed (e4m3, blocks along K) on the way; products are exact and sums fp32 whatever the result's type (bf16 matrix
// instructions on the values held, as clt_gemm8's fp32 form).
//
// Bound: HBM, the N * K weight bytes once.  A block of 8 waves owns a layer, a slice of K and some rows of w.  It packs its slice
// of x into LDS (the values held, as bf16), then every wave streams 1 or 2 groups of 16 rows x 128 k (2 KB each) a step, two to
// four steps ahead in registers; the first steps are requested before x is packed.  Tokens ride the matrix instruction's "N"
// index (16 of them, repeated where there are fewer), weight rows its "M" index.  Where rows alone give too few blocks, K is cut
// into slices whose partial sums a second launch adds in order.
// Measured: 768 -> 32768, 1 token 7.1 us (an empty launch: 3.3); 12 layers of it, 302 MB of weights: 57 us = 5.3 TB/s (1 token), 74 us
// (32 tokens); 393216 -> 768, 1 token: 54 us = 5.6 TB/s with the second launch; 4096 -> 4096: 9.3 us; 8192 -> 768: 7.9 us.
#include "block8_common.h"

namespace {
typedef b8_f32x4 f32x4;
typedef b8_bf16x8 bf16x8;
constexpr int WAVES = 8, MAX_T = 32;
constexpr int LDS_CAP = 136 * 1024;                  // packed slice of x at most
// (beyond 32 tokens packing and the tiled product are faster: 64 tokens, 12 layers of 768 -> 32768 102 against 138 us; 32 tokens: 102 against
// 78, 4096 -> 4096 20 against 13, 393216 -> 768 107 against 105.  No one border fits all: with packing, 32 / 33 tokens take 75 / 100 us for the 12
// layers, 13 / 19 for 4096 -> 4096, but 37 / 32 for 4096 -> 32768)

struct Rows8Args {
    const void* x; long x_token, x_layer;            // strides in elements
    const uint8_t *w, *ws; long ldw, ldws, bw, bws;
    const float* bias; long bbias;
    void* y; long y_token, y_layer; int y_dtype;     // results, or
    float* part;                                     // partial sums [slice][layer][token][N] when K is cut
    int T, N, K, KB, slice_kb, slices, chunks, row_blocks, layers;
    int x_dtype;
};

extern __shared__ __attribute__((aligned(16))) unsigned char r8_smem[];

// `valid` of four consecutive results
__device__ __forceinline__ void store_result(void* y, int dtype, long at, f32x4 v, int valid) {
    if (dtype == CLT_DT_F32) b8_store4<CLT_DT_F32>(y, at, v, valid, 0);
    else if (dtype == CLT_DT_BF16) b8_store4<CLT_DT_BF16>(y, at, v, valid, 0);
    else b8_store4<CLT_DT_F16>(y, at, v, valid, 0);
}

// MT: groups of 16 tokens; G: groups of 16 weight rows a wave has in hand; FMT: format of the weights.  A step is G x 16 rows x 128 k;
// D steps are in flight.
template <int MT, int G, int FMT> __global__ __launch_bounds__(WAVES * 64, 4) void rows8_kernel(Rows8Args a) {
    constexpr int D = G == 1 ? 4 : 2;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
    const int rbk = blockIdx.x % a.row_blocks, rest = blockIdx.x / a.row_blocks, slice = rest % a.slices, layer = rest / a.slices;
    const int kb0 = slice * a.slice_kb, nkb = min(a.slice_kb, a.KB - kb0);
    const int pitch = a.slice_kb * 256 + 16;             // bytes of a token's values in LDS
    const uint8_t *W = a.w + layer * a.bw + (long)kb0 * 128 + fq * 16, *S = a.ws + layer * a.bws + (long)kb0 * a.ldws;
    int n0 = (rbk * a.chunks * WAVES + w) * G * 16;      // first row of the wave's chunk; the next is WAVES * G * 16 further

    uint4 q[D][G][2];
    int sc[D][G];
    const uint8_t* wrow[G];
    int srow[G];
    auto request = [&](int d, int kb) {
        const int k = min(kb, nkb - 1);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint4* p = reinterpret_cast<const uint4*>(wrow[g] + k * 128);
            q[d][g][0] = p[0];                               // k = fq * 16 .. + 15 and 64 + fq * 16 ..: 64 contiguous bytes of a row per request
            q[d][g][1] = p[4];
            sc[d][g] = S[(long)k * a.ldws + srow[g]];
        }
    };
    // ---- pack the slice of x: 16 lanes a block of 128 of one token, 8 elements a lane
    constexpr int P = 3;                                 // items a lane group has in flight (their latency is the block's start-up)
    float xv0[P][8];
    auto load_item = [&](int id, float* v) {
        const int t = id / nkb, kb = id - t * nkb, k = (kb0 + kb) * 128 + fr * 8;
        const long at = t * a.x_token + layer * a.x_layer + k;
        if (a.x_dtype == CLT_DT_F32) b8_load8<CLT_DT_F32>(static_cast<const float*>(a.x) + at, a.K - k, v);
        else if (a.x_dtype == CLT_DT_BF16) b8_load8<CLT_DT_BF16>(static_cast<const uint16_t*>(a.x) + at, a.K - k, v);
        else b8_load8<CLT_DT_F16>(static_cast<const uint16_t*>(a.x) + at, a.K - k, v);
    };
    auto pack_item = [&](int id, const float* v) {
        const int t = id / nkb, kb = id - t * nkb;
        uint32_t m = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, finite_abs_bits(v[j]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
        const int e = block_exponent<0>(m);
        const float g = exp2_int(e);
        const uint32_t lo = pack_codes<0>(v[0], v[1], v[2], v[3], g), hi = pack_codes<0>(v[4], v[5], v[6], v[7], g);
        *reinterpret_cast<bf16x8*>(r8_smem + t * pitch + kb * 256 + fr * 16) = widen8<0>(lo, hi, g);
    };
    const int items = a.T * nkb, first = tid >> 4;
    auto load_items = [&](int id) {
#pragma unroll
        for (int p = 0; p < P; ++p) if (id + p * WAVES * 4 < items) load_item(id + p * WAVES * 4, xv0[p]);
    };
    load_items(first);                                   // (ahead of the weight requests: loads return in order)

    const unsigned char* xrow[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xrow[t] = r8_smem + min(t * 16 + fr, a.T - 1) * pitch + fq * 32;
    for (int chunk = 0; chunk < a.chunks; ++chunk) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            srow[g] = min(n0 + g * 16 + fr, a.N - 1);        // rows past the end: loaded, never stored
            wrow[g] = W + (long)srow[g] * a.ldw;
        }
        f32x4 bv[G];                                         // (ahead of the requests too)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) bv[g][i] = a.bias && !a.part ? a.bias[layer * a.bbias + min(n0 + g * 16 + fq * 4 + i, a.N - 1)] : 0.0f;
#pragma unroll
        for (int d = 0; d < D; ++d) request(d, d);
        if (chunk == 0) {
            for (int id = first; id < items; id += P * WAVES * 4) {
                if (id != first) load_items(id);
#pragma unroll
                for (int p = 0; p < P; ++p) if (id + p * WAVES * 4 < items) pack_item(id + p * WAVES * 4, xv0[p]);
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // (LDS only: the weight requests stay in flight)
        }
        f32x4 acc[G][MT];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[g][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        auto product = [&](int d, int kb) {
            float ws[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                int b = sc[d][g];
                asm volatile("" : "+v"(b));                  // (the byte is not looked at, i.e. waited for, before its step)
                ws[g] = __uint_as_float((uint32_t)b << 23);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bf16x8 xv[MT];
#pragma unroll
                for (int t = 0; t < MT; ++t) xv[t] = *reinterpret_cast<const bf16x8*>(xrow[t] + kb * 256 + (j >> 1) * 128 + (j & 1) * 16);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint4 u = q[d][g][j >> 1];
                    const bf16x8 h = widen8<FMT>(j & 1 ? u.z : u.x, j & 1 ? u.w : u.y, ws[g]);
#pragma unroll
                    for (int t = 0; t < MT; ++t) acc[g][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(h, xv[t], acc[g][t], 0, 0, 0);
                }
            }
        };
        int kb = 0;
        for (; kb + 2 * D <= nkb; kb += D) {                 // (no condition around a request: the compiler would wait for it at the join)
#pragma unroll
            for (int d = 0; d < D; ++d) { product(d, kb + d); request(d, kb + d + D); }
        }
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (kb + d < nkb) product(d, kb + d);
            if (kb + d + D < nkb) request(d, kb + d + D);
        }
#pragma unroll
        for (int d = 0; d < D; ++d) if (kb + d + D < nkb) product(d, kb + d + D);
        const int nc = n0;
        n0 += WAVES * G * 16;
#pragma unroll
        for (int g = 0; g < G; ++g) {                        // row nc + g * 16 + fq * 4 + i of token t * 16 + fr
            const int n = nc + g * 16 + fq * 4, valid = a.N - n;
            if (valid <= 0) continue;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int tok = t * 16 + fr;
                if (tok >= a.T) continue;
                if (a.part) store_result(a.part, CLT_DT_F32, (((long)slice * a.layers + layer) * a.T + tok) * a.N + n, acc[g][t], valid);
                else store_result(a.y, a.y_dtype, tok * a.y_token + layer * a.y_layer + n, acc[g][t] + bv[g], valid);
            }
        }
    }
}

// partial sums of the slices -> results, slices in order
__global__ __launch_bounds__(256) void rows8_fold_kernel(Rows8Args a, long n) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;                 // (layer, token, column)
    if (i >= n) return;
    const long lt = i / a.N;
    const int c = (int)(i - lt * a.N), layer = (int)(lt / a.T), t = (int)(lt - (long)layer * a.T);
    float s = 0.0f;
    const float* p = a.part + i;
    int k = 0;
    for (; k + 32 <= a.slices; k += 32) {                                // many requests at a time (few threads here), added in order
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = p[(k + j) * n];
#pragma unroll
        for (int j = 0; j < 32; ++j) s += v[j];
    }
    for (; k < a.slices; k += 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < a.slices ? p[(k + j) * n] : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
    }
    if (a.bias) s += a.bias[layer * a.bbias + c];
    store_result(a.y, a.y_dtype, t * a.y_token + layer * a.y_layer + c, f32x4{s, 0.0f, 0.0f, 0.0f}, 1);
}

// How the work is cut: blocks of K per slice, slices, row groups in a wave's hand (G), chunks of rows per block.
// Slices: at least as many as the packed x needs to fit LDS; from there to two blocks a CU (or twice those slices) the least of the times that these measurements add
// up to, in units of one step (a block of k, 0.5 us with every CU at work): a pass of blocks over the CUs takes the slice's steps and 1.5
// (1.3 times that where LDS holds one block of 32 tokens a CU: nothing runs while it packs x), the second launch 6 and 0.3 a slice.
// One token, 8192 -> 768 in 4 / 8 / 16 slices: 13.1 / 8.9 / 8.0 us; 4096 -> 4096 in 2 / 4 / 8: 13.6 / 10.7 / 9.3; 4096 -> 14336 in 2 / 4 (224 and
// 448 blocks): 15.7 / 17.8; 1024 -> 1024 in 1 / 2: 6.5 / 7.6; 393216 -> 768 in 42 / 64 / 86 (252, 384 and 516 blocks): 53 / 61 / 57.
// G grows while every CU keeps two blocks (x is read from LDS once for G row groups).  What is left over becomes chunks, so that x is
// packed once per resident block: up to 16 tokens above 2048 blocks, above that (a longer packing) above two rounds of the blocks that
// fit: 12 x (768 -> 32768), 32 tokens: 77 / 72 us in 1536 / 768 blocks, one token 47 / 49; 4096 -> 32768, 32 tokens: 64 / 45 in 512 / 256.
struct Cut { int slice_kb, slices, g, chunks, row_blocks; };
Cut cut_rows8(int T, int L, int N, int KB) {
    Cut c;
    const int fit = (LDS_CAP / T - 16) / 256;                            // blocks of k whose x fits LDS (>= 16 for 32 tokens)
    const long rb = (N + WAVES * 16 - 1) / (WAVES * 16), want = 512;
    auto alone = [&](int slice_kb) { return (long)T * (slice_kb * 256 + 16) > 80 * 1024; };      // one block a CU
    long least = -1;
    const long need = (KB + fit - 1) / fit, most = 2 * L * rb * need > want ? 2 * L * rb * need : want;
    for (long s = need; s == need || (s * 4 <= KB && L * rb * s <= most); ++s) {
        const int per = (int)((KB + s - 1) / s), used = (KB + per - 1) / per;
        const long pass = (L * rb * used + 255) / 256 * (10L * per + 15), t = (alone(per) ? pass * 13 / 10 : pass) + (used > 1 ? 60 + 3 * used : 0);
        if (least < 0 || t < least) { least = t; c.slice_kb = per; c.slices = used; }
    }
    const long blocks = L * rb * c.slices;                               // at G = 1
    const int most_g = T <= 16 ? 2 : 1;                                  // (two row groups and 32 tokens: one block per CU instead of two, 87 against 80 us)
    c.g = 1;
    while (c.g < most_g && blocks >= 2 * c.g * want) c.g *= 2;
    const long rows = (long)WAVES * 16 * c.g, per_layer = (N + rows - 1) / rows, round = alone(c.slice_kb) ? 256 : 512;
    c.chunks = (int)(L * per_layer * c.slices / (T > 16 ? 2 * round : 2048)) + 1;
    if (c.chunks > per_layer) c.chunks = (int)per_layer;
    c.row_blocks = (int)((per_layer + c.chunks - 1) / c.chunks);
    return c;
}

template <int MT, int G> int launch_rows(const Rows8Args& a, int fmt, long blocks, int lds, hipStream_t st) {
    const auto f = fmt ? rows8_kernel<MT, G, 1> : rows8_kernel<MT, G, 0>;
    if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return CLT_ERR_LAUNCH;
    f<<<dim3((unsigned)blocks), dim3(WAVES * 64), lds, st>>>(a);
    CLT_LAUNCH_CHECK();
    return CLT_OK;
}
}  // namespace

extern "C" size_t clt_linear8_rows_workspace_bytes(int tokens, int layers, int N, int K) {
    if (tokens <= 0 || tokens > MAX_T || layers <= 0 || N <= 0 || K <= 0) return 0;
    const Cut c = cut_rows8(tokens, layers, N, (int)(up128(K) / 128));
    return c.slices > 1 ? (size_t)c.slices * layers * tokens * N * 4 : 0;
}

extern "C" int clt_linear8_rows_plan(int tokens, int layers, int N, int K, int64_t* plan) {
    if (tokens <= 0 || tokens > MAX_T || layers <= 0 || N <= 0 || K <= 0 || !plan) return CLT_ERR_SHAPE;
    const Cut c = cut_rows8(tokens, layers, N, (int)(up128(K) / 128));
    plan[0] = c.slice_kb; plan[1] = c.slices; plan[2] = c.g; plan[3] = c.chunks; plan[4] = c.row_blocks;
    return CLT_OK;
}

extern "C" int clt_linear8_rows(const void* x, int x_dtype, long x_token_stride, long x_layer_stride, const void* w, const void* w_scale,
                                int w_format, long ldw, long ldws, long w_batch, long ws_batch, const float* bias, long bias_batch,
                                void* y, int y_dtype, long y_token_stride, long y_layer_stride, int tokens, int layers, int N, int K,
                                void* workspace, size_t workspace_bytes, void* stream) {
    if (tokens <= 0 || layers <= 0 || N <= 0 || K <= 0 || x_dtype < 0 || x_dtype > 2 || y_dtype < 0 || y_dtype > 2 || (w_format & ~1)) return CLT_ERR_SHAPE;
    if (tokens > MAX_T) return CLT_ERR_RANGE;                            // (more are clt_pack8's and clt_gemm8's)
    if (!x || !w || !w_scale || !y || ldw < up128(K) || ldws < N) return CLT_ERR_SHAPE;
    const size_t xs = x_dtype == CLT_DT_F32 ? 4 : 2, ys = y_dtype == CLT_DT_F32 ? 4 : 2;
    if (!aligned16(w) || ldw % 16 || w_batch % 16 || ((uintptr_t)x & (xs - 1)) || ((uintptr_t)y & (ys - 1)) || ((uintptr_t)bias & 3)) return CLT_ERR_ALIGN;
    const int KB = (int)(up128(K) / 128);
    const Cut c = cut_rows8(tokens, layers, N, KB);
    const size_t need = clt_linear8_rows_workspace_bytes(tokens, layers, N, K);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return CLT_ERR_WORKSPACE;
    Rows8Args a;
    a.x = x; a.x_token = x_token_stride; a.x_layer = x_layer_stride; a.x_dtype = x_dtype;
    a.w = static_cast<const uint8_t*>(w); a.ws = static_cast<const uint8_t*>(w_scale); a.ldw = ldw; a.ldws = ldws; a.bw = w_batch; a.bws = ws_batch;
    a.bias = bias; a.bbias = bias_batch;
    a.y = y; a.y_token = y_token_stride; a.y_layer = y_layer_stride; a.y_dtype = y_dtype;
    a.part = c.slices > 1 ? static_cast<float*>(workspace) : nullptr;
    a.T = tokens; a.N = N; a.K = K; a.KB = KB; a.slice_kb = c.slice_kb; a.slices = c.slices; a.chunks = c.chunks; a.row_blocks = c.row_blocks; a.layers = layers;
    const long blocks = (long)layers * c.slices * c.row_blocks;
    if (!b8_fits(blocks, WAVES * 64)) return CLT_ERR_RANGE;
    const int lds = tokens * (c.slice_kb * 256 + 16);
    const hipStream_t st = as_stream(stream);
    int rc;
    if (tokens <= 16) rc = c.g == 1 ? launch_rows<1, 1>(a, w_format, blocks, lds, st) : launch_rows<1, 2>(a, w_format, blocks, lds, st);
    else rc = launch_rows<2, 1>(a, w_format, blocks, lds, st);
    if (rc != CLT_OK || c.slices == 1) return rc;
    const long n = (long)layers * tokens * N, fold = (n + 255) / 256;
    if (!b8_fits(fold, 256)) return CLT_ERR_RANGE;
    rows8_fold_kernel<<<dim3((unsigned)fold), dim3(256), 0, st>>>(a, n);
    CLT_LAUNCH_CHECK();
    return CLT_OK;
}
