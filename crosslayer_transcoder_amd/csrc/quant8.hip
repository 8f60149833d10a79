// 8-bit block-scaled form of a matrix and back (held form: block8_common.h).
//
// Packing, one read of x [L][R][C] for up to two forms: codes along the rows (a scale per row and 128 columns: the operand of a
// contraction over the columns) and the transposed codes (a scale per column and 128 rows: the operand of a contraction over
// the rows, i.e. what a weight gradient reads — the 8-bit checkpoint of an activation).  Bound: HBM, es bytes read and
// 1 + 1/128 written per element and form.
// A block of 256 threads takes a 128 x 128 tile, a thread an 8 x 8 patch in registers: row maxima over 16 lanes, column maxima
// over 4 lanes and, through LDS, 4 waves.  8 x 8 patches because both forms then leave in 8-byte pieces without repacking: a
// patch row is 8 row-major codes, a patch column 8 transposed ones (these pass through a 16 KB LDS tile to go out as whole
// 128-byte lines).
// Measured: 4096 x 12 x 768 bf16, both forms 32 us = 4.7 TB/s (a large copy: 4.75); 4096 x 4 x 32768 bf16, both forms 492 us = 4.4;
// 12 x 32768 x 768 fp32 weights, one form 280 us = 5.4; 4096 x 12 x 32768 bf16, transposed form and column sums 1310 us = 3.7 (rows of a
// tile 786 KB apart; other tile orders and uncached stores: 1260 .. 1330); restoring 4096 x 4 x 32768 to bf16 305 us = 5.3.
#include "block8_common.h"

namespace {

struct Pack8Args {
    const void* x; long row_stride, batch_stride;
    uint8_t *q, *s;            // row form (or nullptr): codes [L][R][Cp], scale bytes [L][Cp / 128][Rp]
    uint8_t *qt, *st;          // transposed form (or nullptr): codes [L][C][Rp], scale bytes [L][Rp / 128][Cp]
    long q_pitch, q_batch, s_batch, qt_pitch, qt_batch, st_batch;            // bytes
    float* sums;               // column sums of each 128-row block [L][Rp / 128][C] (or nullptr)
    int R, C, tiles_r, tiles_c;
};

template <int DT, int FMT, bool TILES> __global__ __launch_bounds__(256) void pack8_kernel(Pack8Args a) {
    typedef typename Elem<DT>::type T;
    __shared__ uint32_t cmax[4][B8];
    __shared__ float csum[4][B8];
    __shared__ uint32_t rmax[4];
    __shared__ __attribute__((aligned(16))) uint8_t tile[B8 * B8];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int cg = tid & 15, rg = tid >> 4;              // patch: columns cg * 8 .., rows rg * 8 ..
    // a tile per block, column tiles fastest (neighbouring blocks read neighbouring lines of the same rows)
    const long per = (long)a.tiles_r * a.tiles_c, b = blockIdx.x / per;
    const int t = (int)(blockIdx.x - b * per), tr = t / a.tiles_c, tc = t - tr * a.tiles_c;
    const int r0 = tr * B8, c0 = tc * B8;
    const long Rp = (long)a.tiles_r * B8, Cp = (long)a.tiles_c * B8;

    float v[8][8];
    const int nc = a.C - (c0 + cg * 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = r0 + rg * 8 + i;
        const T* p = static_cast<const T*>(a.x) + b * a.batch_stride + (long)r * a.row_stride + c0 + cg * 8;
        b8_load8<DT>(p, r < a.R ? nc : 0, v[i]);
    }
    // maxima of the finite magnitudes, per row (over the 16 lanes of a row) and per column (over rows: 4 lanes, 4 waves).  As unsigned
    // integers the magnitudes of inf and NaN are larger than every finite one: only where one shows up are they sorted out.
    uint32_t rm[8], cm[8];
    auto maxima = [&](auto bits) {
#pragma unroll
        for (int k = 0; k < 8; ++k) rm[k] = cm[k] = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t m = bits(v[i][j]);
                rm[i] = max(rm[i], m);
                cm[j] = max(cm[j], m);
            }
    };
    maxima([](float x) { return __float_as_uint(x) & 0x7fffffffu; });
    uint32_t most = 0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = max(most, rm[k]);
    if (most >= 0x7f800000u) maxima([](float x) { return finite_abs_bits(x); });
    if (TILES) {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, rm[i]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
        if (lane == 0) rmax[w] = m;
    } else {
        if (a.q) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) rm[i] = max(rm[i], (uint32_t)__shfl_xor((int)rm[i], o, 64));
        }
        if (a.qt) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                cm[j] = max(cm[j], (uint32_t)__shfl_xor((int)cm[j], 16, 64));
                cm[j] = max(cm[j], (uint32_t)__shfl_xor((int)cm[j], 32, 64));
            }
            if (lane < 16) {
#pragma unroll
                for (int j = 0; j < 8; ++j) cmax[w][cg * 8 + j] = cm[j];
            }
        }
    }
    if (a.sums) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i][j];
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            if (lane < 16) csum[w][cg * 8 + j] = s;
        }
    }
    __syncthreads();
    if (TILES) {
        const uint32_t m = max(max(rmax[0], rmax[1]), max(rmax[2], rmax[3]));
#pragma unroll
        for (int k = 0; k < 8; ++k) rm[k] = cm[k] = m;
    } else if (a.qt) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = cg * 8 + j;
            cm[j] = max(max(cmax[0][c], cmax[1][c]), max(cmax[2][c], cmax[3][c]));
        }
    }
    if (a.sums && tid < B8 && c0 + tid < a.C)
        a.sums[(b * a.tiles_r + tr) * a.C + c0 + tid] = (csum[0][tid] + csum[1][tid]) + (csum[2][tid] + csum[3][tid]);

    if (a.q) {
        uint32_t sb[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = block_exponent<FMT>(rm[i]), r = r0 + rg * 8 + i;
            const float f = exp2_int(e);
            sb[i >> 2] |= (uint32_t)(e + 127) << (8 * (i & 3));
            uint2 o;
            o.x = pack_codes<FMT>(v[i][0], v[i][1], v[i][2], v[i][3], f);
            o.y = pack_codes<FMT>(v[i][4], v[i][5], v[i][6], v[i][7], f);
            if (r < a.R) *reinterpret_cast<uint2*>(a.q + b * a.q_batch + r * a.q_pitch + c0 + cg * 8) = o;
        }
        if (cg == 0) *reinterpret_cast<uint2*>(a.s + b * a.s_batch + tc * Rp + r0 + rg * 8) = make_uint2(sb[0], sb[1]);
    }
    if (a.qt) {
        uint32_t sb[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = block_exponent<FMT>(cm[j]), c = cg * 8 + j;
            const float f = exp2_int(e);
            sb[j >> 2] |= (uint32_t)(e + 127) << (8 * (j & 3));
            uint2 o;
            o.x = pack_codes<FMT>(v[0][j], v[1][j], v[2][j], v[3][j], f);
            o.y = pack_codes<FMT>(v[4][j], v[5][j], v[6][j], v[7][j], f);
            // 8-byte chunk rg of column c, chunks XOR-swizzled with the column group (the 16 groups of a store hit 16 chunks)
            *reinterpret_cast<uint2*>(tile + c * B8 + ((rg ^ cg) << 3)) = o;
        }
        if (rg == 0) *reinterpret_cast<uint2*>(a.st + b * a.st_batch + tr * Cp + c0 + cg * 8) = make_uint2(sb[0], sb[1]);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int id = k * 256 + tid, c = id >> 3, p = id & 7, x = c >> 3;
            const uint2 lo = *reinterpret_cast<const uint2*>(tile + c * B8 + (((2 * p) ^ x) << 3));
            const uint2 hi = *reinterpret_cast<const uint2*>(tile + c * B8 + (((2 * p + 1) ^ x) << 3));
            if (c0 + c < a.C) *reinterpret_cast<uint4*>(a.qt + b * a.qt_batch + (c0 + c) * a.qt_pitch + r0 + p * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
    }
}

// sums of the 128-row blocks -> column sums, blocks in order
__global__ __launch_bounds__(256) void fold_sums_kernel(const float* part, float* out, int blocks, int C, long n) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long b = i / C;
    const float* p = part + b * blocks * (long)C + (i - b * C);
    double s = 0.0;
    for (int k = 0; k < blocks; ++k) s += (double)p[(long)k * C];
    out[i] = (float)s;
}

// codes -> values 2^e x code, rounded once to the output type; 16 codes a thread (bound: HBM, 1 + es bytes an element)
template <int DT> __global__ __launch_bounds__(256) void unpack8_kernel(const uint8_t* q, const uint8_t* s, int fmt, int R, int C,
                                                                        long pitch, long Rp, long q_batch, long s_batch, void* out,
                                                                        int chunks, long total) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    const long row = id / chunks;                        // row of the whole batch
    const int c = (int)(id - row * chunks) * 16;
    const long b = row / R;
    const int r = (int)(row - b * R);
    const uint4 u = *reinterpret_cast<const uint4*>(q + b * q_batch + (long)r * pitch + c);
    const float f = exp2_int((int)s[b * s_batch + (long)(c >> 7) * Rp + r] - 127);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    typename Elem<DT>::type* o = static_cast<typename Elem<DT>::type*>(out) + row * C + c;
    if (c + 16 <= C) {
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const b8_f32x4 x = unpack_codes(fmt, w[k]) * f, y = unpack_codes(fmt, w[k + 1]) * f;
            if constexpr (DT == CLT_DT_F32) {
                reinterpret_cast<b8_f32x4_u*>(o)[k] = x;
                reinterpret_cast<b8_f32x4_u*>(o)[k + 1] = y;
            } else
                reinterpret_cast<b8_u32x4_u*>(o)[k >> 1] = b8_u32x4_u{pack_out16<DT>(x[0], x[1]), pack_out16<DT>(x[2], x[3]),
                                                                      pack_out16<DT>(y[0], y[1]), pack_out16<DT>(y[2], y[3])};
        }
    } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const b8_f32x4 x = unpack_codes(fmt, w[k >> 2]) * f;
            if (c + k < C) o[k] = f32_to_elem<DT>(x[k & 3]);
        }
    }
}

template <int DT> int launch_pack(const Pack8Args& a, int fmt, bool tiles, long blocks, hipStream_t st) {
    const dim3 g((unsigned)blocks), t(256);
    if (fmt == CLT_F8_E4M3) {
        if (tiles) pack8_kernel<DT, 0, true><<<g, t, 0, st>>>(a); else pack8_kernel<DT, 0, false><<<g, t, 0, st>>>(a);
    } else {
        if (tiles) pack8_kernel<DT, 1, true><<<g, t, 0, st>>>(a); else pack8_kernel<DT, 1, false><<<g, t, 0, st>>>(a);
    }
    CLT_LAUNCH_CHECK();
    return CLT_OK;
}
}  // namespace

// (up to 128 rows: the one block of rows writes the sums themselves)
extern "C" size_t clt_pack8_sums_workspace_bytes(int batch, int rows, int cols) {
    return batch > 0 && rows > B8 && cols > 0 ? (size_t)batch * ((rows - 1) / B8 + 1) * cols * 4 : 0;
}

extern "C" int clt_pack8(const void* x, int dtype, long row_stride, long batch_stride, int batch, int rows, int cols, int format,
                         int tiles, void* q, void* s, void* qt, void* st, float* column_sums, void* workspace,
                         size_t workspace_bytes, void* stream) {
    const long Rp = up128(rows), Cp = up128(cols);
    return clt_pack8_into(x, dtype, row_stride, batch_stride, batch, rows, cols, format, tiles, q, s, Cp, rows * Cp, Cp / B8 * Rp, qt, st,
                          Rp, cols * Rp, Rp / B8 * Cp, column_sums, workspace, workspace_bytes, stream);
}

extern "C" int clt_pack8_into(const void* x, int dtype, long row_stride, long batch_stride, int batch, int rows, int cols, int format,
                              int tiles, void* q, void* s, long q_pitch, long q_batch, long s_batch, void* qt, void* st, long qt_pitch,
                              long qt_batch, long st_batch, float* column_sums, void* workspace, size_t workspace_bytes, void* stream) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || dtype < 0 || dtype > 2 || format < 0 || format > 1) return CLT_ERR_SHAPE;
    if (!x || !q != !s || !qt != !st || (!q && !qt)) return CLT_ERR_SHAPE;
    const size_t es = dtype == CLT_DT_F32 ? 4 : 2;
    if (((uintptr_t)x & (es - 1)) || !(aligned16(q) && aligned16(s) && aligned16(qt) && aligned16(st))) return CLT_ERR_ALIGN;
    if ((q && q_pitch < up128(cols)) || (qt && qt_pitch < up128(rows))) return CLT_ERR_SHAPE;
    if (((q_pitch | q_batch | s_batch | qt_pitch | qt_batch | st_batch) & 15)) return CLT_ERR_ALIGN;
    Pack8Args a;
    a.q_pitch = q_pitch; a.q_batch = q_batch; a.s_batch = s_batch; a.qt_pitch = qt_pitch; a.qt_batch = qt_batch; a.st_batch = st_batch;
    a.x = x; a.row_stride = row_stride; a.batch_stride = batch_stride;
    a.q = static_cast<uint8_t*>(q); a.s = static_cast<uint8_t*>(s); a.qt = static_cast<uint8_t*>(qt); a.st = static_cast<uint8_t*>(st);
    a.R = rows; a.C = cols; a.tiles_r = (rows - 1) / B8 + 1; a.tiles_c = (cols - 1) / B8 + 1;
    const size_t need = clt_pack8_sums_workspace_bytes(batch, rows, cols);
    if (column_sums && need && (!workspace || workspace_bytes < need)) return CLT_ERR_WORKSPACE;
    a.sums = !column_sums ? nullptr : need ? static_cast<float*>(workspace) : column_sums;
    const long blocks = (long)batch * a.tiles_r * a.tiles_c, sums = ((long)batch * cols + 255) / 256;
    if (!b8_fits(blocks, 256) || (column_sums && need && !b8_fits(sums, 256))) return CLT_ERR_RANGE;
    const hipStream_t hs = as_stream(stream);
    const int rc = dtype == CLT_DT_F32 ? launch_pack<CLT_DT_F32>(a, format, tiles != 0, blocks, hs)
                   : dtype == CLT_DT_BF16 ? launch_pack<CLT_DT_BF16>(a, format, tiles != 0, blocks, hs)
                                          : launch_pack<CLT_DT_F16>(a, format, tiles != 0, blocks, hs);
    if (rc != CLT_OK || !column_sums || !need) return rc;
    const long n = (long)batch * cols;
    fold_sums_kernel<<<dim3((unsigned)sums), dim3(256), 0, hs>>>(a.sums, column_sums, a.tiles_r, cols, n);
    CLT_LAUNCH_CHECK();
    return CLT_OK;
}

extern "C" int clt_unpack8(const void* q, const void* s, int format, int batch, int rows, int cols, long pitch, long scale_pitch,
                           long q_batch_stride, long s_batch_stride, void* out, int dtype, void* stream) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || dtype < 0 || dtype > 2 || format < 0 || format > 1 || !q || !s || !out) return CLT_ERR_SHAPE;
    if (pitch < up128(cols) || scale_pitch < rows) return CLT_ERR_SHAPE;
    const size_t es = dtype == CLT_DT_F32 ? 4 : 2;
    if (!aligned16(q) || pitch % 16 || q_batch_stride % 16 || ((uintptr_t)out & (es - 1))) return CLT_ERR_ALIGN;
    const int chunks = (cols - 1) / 16 + 1;
    const long total = (long)batch * rows * chunks, blocks = (total + 255) / 256;
    if (!b8_fits(blocks, 256)) return CLT_ERR_RANGE;
    const dim3 g((unsigned)blocks), t(256);
    const hipStream_t hs = as_stream(stream);
    const uint8_t *qp = static_cast<const uint8_t*>(q), *sp = static_cast<const uint8_t*>(s);
#define UNPACK(DT) unpack8_kernel<DT><<<g, t, 0, hs>>>(qp, sp, format, rows, cols, pitch, scale_pitch, q_batch_stride, s_batch_stride, out, chunks, total)
    if (dtype == CLT_DT_F32) UNPACK(CLT_DT_F32); else if (dtype == CLT_DT_BF16) UNPACK(CLT_DT_BF16); else UNPACK(CLT_DT_F16);
#undef UNPACK
    CLT_LAUNCH_CHECK();
    return CLT_OK;
}
