// row_quant.hip -- rows to 8-bit blocks with power-of-two scales.
//
// A block's scale is the smallest power of two s with max |x| <= 448 s, so x / s is exact and the one rounding is the one to 8 bits: half
// a step of e4m3, 2^-4 of the value. (A scale of max / 448 would use up to one more bit of range and round twice; and the matrix
// instruction takes powers of two for nothing.) Bound by memory: 2 or 4 bytes in, 1 out.
#include "rows.h"

namespace lssvc {

struct QuantP {
    const void *x;
    uint8_t *q, *s;
    int64_t ldx, ldq, lds;
    int64_t rows;
    int cols, kb;
};

// 8 values from column c on, zeros behind the last column
template <typename T> __device__ __forceinline__ void load8(const T *row, int c, int cols, float (&v)[8]) {
    if (c + 8 <= cols) {
        const Pack<T, 8> d = load_pack<T, 8>(row + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_f32(d.v[j]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? to_f32(row[c + j]) : 0.f;
}
__device__ __forceinline__ void store8(uint8_t *q, const float (&v)[8], float inv) {
    uint2 o;
    o.x = to_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    o.y = to_e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    *reinterpret_cast<uint2 *>(q) = o;
}

// 1 x 128 blocks: 16 lanes hold a block (8 values each), the maximum goes around in the DPP row. A workgroup takes 16 consecutive blocks
// of the matrix, row by row. 34560x768 bf16: 14.6 us, 5.45 TB/s, the rate of a large copy.
template <typename T> __global__ __launch_bounds__(256) void quant_rows_kernel(QuantP p, int64_t blocks) {
    const int64_t b = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (b >= blocks) return;                                    // (all 16 lanes of a block leave together)
    const int64_t r = b / p.kb;
    const int k = (int)(b - r * p.kb), c = k * kFp8Block + (threadIdx.x & 15) * 8;
    float v[8];
    load8((const T *)p.x + r * p.ldx, c, p.cols, v);
    const uint32_t byte = fp8_scale_byte(row16_finite_max(v));
    if (c < ((p.cols + 15) & ~15)) store8(p.q + r * p.ldq + c, v, scale_inverse(byte));
    if ((threadIdx.x & 15) == 0) p.s[r * p.lds + k] = (uint8_t)byte;
}

// 128 x 128 blocks: a workgroup holds one, 4 rows of 8 columns per thread. 1000x5000 fp32: 7.0 us for 25 MB, 320 blocks: one load of 64 KB,
// its maximum and one store after the other.
template <typename T> __global__ __launch_bounds__(512) void quant_tiles_kernel(QuantP p) {
    __shared__ uint32_t wmax[32];
    const int64_t rb = blockIdx.x / (unsigned)p.kb;
    const int k = (int)(blockIdx.x - rb * p.kb), t = threadIdx.x;
    const int c = k * kFp8Block + (t & 15) * 8;
    const int64_t r0 = rb * kFp8Block + (t >> 4);
    float v[4][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + 32 * i;
        if (r < p.rows) load8((const T *)p.x + r * p.ldx, c, p.cols, v[i]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        m = max(m, row16_finite_max(v[i]));
    }
    if ((t & 15) == 0) wmax[t >> 4] = m;
    __syncthreads();
    m = row16_max(max(wmax[t & 15], wmax[16 + (t & 15)]));
    const uint32_t byte = fp8_scale_byte(m);
    const float inv = scale_inverse(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + 32 * i;
        if (r < p.rows && c < ((p.cols + 15) & ~15)) store8(p.q + r * p.ldq + c, v[i], inv);
    }
    if (t == 0) p.s[rb * p.lds + k] = (uint8_t)byte;
}

template <typename T> static int launch_quant(const QuantP &p, int block_rows, hipStream_t s) {
    if (block_rows == 1) {
        const int64_t blocks = p.rows * p.kb;
        LSSVC_CHECK(fits_launch((blocks + 15) / 16, 256), "quantize_fp8: %lld blocks do not fit one launch", (long long)blocks);
        quant_rows_kernel<T><<<(unsigned)((blocks + 15) / 16), 256, 0, s>>>(p, blocks);
    } else {
        const int64_t tiles = (p.rows + kFp8Block - 1) / kFp8Block * p.kb;
        LSSVC_CHECK(fits_launch(tiles, 512), "quantize_fp8: %lld blocks do not fit one launch", (long long)tiles);
        quant_tiles_kernel<T><<<(unsigned)tiles, 512, 0, s>>>(p);
    }
    return launch_status("quantize_fp8");
}

}  // namespace lssvc

using namespace lssvc;

extern "C" int lssvc_quantize_fp8(const lssvc_rows *x, const lssvc_fp8 *y, void *stream) {
    if (int rc = rows_check("quantize_fp8", x)) return rc;
    if (int rc = fp8_out_check("quantize_fp8", y, x->rows, x->cols)) return rc;
    LSSVC_CHECK(y->block_rows == 1 || y->block_rows == kFp8Block, "quantize_fp8: block_rows is 1 or 128, got %d", y->block_rows);
    if (x->rows == 0) return 0;
    LSSVC_CHECK(apart({values_of(y), scales_of(y)}, {span_of(x)}), "quantize_fp8: input, values and scales overlap");
    QuantP p{x->ptr, (uint8_t *)y->values, (uint8_t *)y->scale, x->ld, y->ld, y->scale_ld, x->rows, x->cols, (x->cols + kFp8Block - 1) / kFp8Block};
    hipStream_t s = (hipStream_t)stream;
    if (x->dtype == LSSVC_F32) return launch_quant<float>(p, y->block_rows, s);
    if (x->dtype == LSSVC_F16) return launch_quant<f16_t>(p, y->block_rows, s);
    return launch_quant<bf16_t>(p, y->block_rows, s);
}
