// fp8_matmul.hip -- y = act(A W^T + bias) + residual for 8-bit rows with a scale for each block of 128 along K.
//
// 16-bit results: one v_mfma_f32_16x16x128_f8f6f4 covers exactly one block of K, so a block's scales belong to one instruction:
//   e8m0 scales  the scaled form of the instruction multiplies by 2^(sa + sw) itself; the accumulator runs over all of K.
//   fp32 scales  each block's product starts from zero and is added to the accumulator with one FMA per value, factor sa * sw.
// The 8-bit instructions add the products of a group of 8 aligned to the largest of them and drop what lies 13 binary places below its
// exponent (measured, every 8-bit form does); blocks and groups are added in fp32. For operands that are 8-bit roundings of normal numbers
// that is 1.3e-5 of the result in the 2-norm: nothing beside half a step of bf16 (2^-8) or fp16 (2^-11), but 200 half steps of fp32.
// fp32 results: the 8-bit values are widened to fp16, which holds every e4m3 number, and multiplied by v_mfma_f32_16x16x32_f16, which adds in
// fp32; scales are applied to each block's partial sum. Half the rate, 1e-7.
// The weights are the instruction's FIRST operand: a lane then holds one row of A (lane & 15) and four consecutive columns of y per
// fragment, and with the weight rows of a 64-column group dealt to the fragments as n = 16 * (r / 4) + 4 * f + r % 4 it holds 16
// consecutive columns over four fragments: rows of y leave in 32- or 64-byte pieces. The order of k inside a block is free as long
// as both operands share it: a lane's 32 bytes are the 16-byte chunks q and q + 4 (q = lane / 16).
#include "rows.h"

namespace lssvc {

struct MatmulP {
    const uint8_t *a, *w;
    const void *sa, *sw;
    int64_t lda, ldw, ldsa, ldsw;
    const float *bias;
    const void *res;
    void *y;
    int64_t ldres, ldy;
    int M, N, K16, nkb;      // K16: bytes of a row that are read (K rounded up to 16; zeros behind K)
    int dtype;
    Act act;
    int tiles_m, tiles_n;
};

__device__ const i32x4 g_zero_chunk = {0, 0, 0, 0};

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ i32x8 join(const i32x4 &lo, const i32x4 &hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A fragment: a lane's 32 values of one block. Wide: as fp16, in four operands of the fp16 instruction.
template <bool WIDE> struct Frag {
    i32x8 v;
    __device__ __forceinline__ void set(const i32x4 &lo, const i32x4 &hi) { v = join(lo, hi); }
};
template <> struct Frag<true> {
    f16x8 v[4];
    __device__ __forceinline__ void half(const i32x4 &x, f16x8 &a, f16x8 &b) {
        union { f16x8 f[2]; f16x2 p[8]; } u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u.p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)x[i], 1.f, false);
            u.p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)x[i], 1.f, true);
        }
        a = u.f[0], b = u.f[1];
    }
    __device__ __forceinline__ void set(const i32x4 &lo, const i32x4 &hi) { half(lo, v[0], v[1]), half(hi, v[2], v[3]); }
};

// A block's scale: as the instruction takes it (an exponent byte in bits 7:0) or as a factor
template <bool E8M0, bool WIDE> __device__ __forceinline__ auto scale_of(uint32_t bits) {
    if constexpr (!E8M0) return __uint_as_float(bits);
    else if constexpr (WIDE) {
        const uint32_t b = bits & 0xff;                          // 2^(b - 127): the exponent field, but for the ends of the range
        return __uint_as_float(b == 255 ? 0x7fc00000u : b == 0 ? 0x400000u : b << 23);
    }
    else return (int)bits;
}

// acc += sw * sa * (block of W) (block of A)^T
template <bool E8M0, bool WIDE, typename S>
__device__ __forceinline__ void mma(const Frag<WIDE> &w, const Frag<WIDE> &a, f32x4 &acc, S sw, S sa) {
    if constexpr (E8M0 && !WIDE) {
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, acc, 0, 0, 0, sw, 0, sa);
    } else {
        f32x4 part = {0.f, 0.f, 0.f, 0.f};
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) part = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], a.v[i], part, 0, 0, 0);
        } else part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, part, 0, 0, 0, 0, 0, 0);      // (unscaled)
        const float s = sw * sa;
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = fmaf(part[r], s, acc[r]);
    }
}

// act(v) + residual for CNT consecutive columns of one row, rounded once
template <typename T, int CNT>
__device__ __forceinline__ void store_cols(const MatmulP &p, int64_t m, int n, float (&v)[CNT]) {
    T *dst = (T *)p.y + m * p.ldy + n;
    const T *res = p.res ? (const T *)p.res + m * p.ldres + n : nullptr;
    const bool full = n + CNT <= p.N;
    apply_act(v, p.act);
    if (res) {
        Pack<T, CNT> r;
        if (full) r = load_pack<T, CNT>(res);
        else
#pragma unroll
            for (int i = 0; i < CNT; ++i) r.v[i] = n + i < p.N ? res[i] : from_f32<T>(0.f);
#pragma unroll
        for (int i = 0; i < CNT; ++i) v[i] += to_f32(r.v[i]);
    }
    Pack<T, CNT> o;
#pragma unroll
    for (int i = 0; i < CNT; ++i) o.v[i] = from_f32<T>(v[i]);
    if (full) store_pack(dst, o);
    else
#pragma unroll
        for (int i = 0; i < CNT; ++i)
            if (n + i < p.N) dst[i] = o.v[i];
}
template <int CNT> __device__ __forceinline__ void load_bias(const MatmulP &p, int n, float (&b)[CNT]) {
#pragma unroll
    for (int i = 0; i < CNT; ++i) b[i] = p.bias && n + i < p.N ? p.bias[n + i] : 0.f;
}

template <bool E8M0> __device__ __forceinline__ uint32_t load_scale(const void *s, int64_t at) {
    if constexpr (E8M0) return ((const uint8_t *)s)[at];
    else return ((const uint32_t *)s)[at];
}

// ---- few rows: bound by the weight's bytes ------------------------------------------------------------------------------------------
// A workgroup owns 16 columns of y (16 weight rows); its waves deal K's blocks among themselves, read both operands straight into
// registers and add up through the LDS in a fixed order.
template <int MF, bool E8M0, typename T, int NW>
__global__ __launch_bounds__(NW * 64) void matmul_few_rows_kernel(MatmulP p) {
    constexpr int U = 4;                          // blocks of K in flight per wave
    constexpr bool WIDE = sizeof(T) == 4;
    __shared__ f32x4 red[NW][MF][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int wr = min(n0 + i16, p.N - 1);
    const uint8_t *wp = p.w + (int64_t)wr * p.ldw + q * 16;
    const uint8_t *ap[MF];
    int64_t sar[MF];
#pragma unroll
    for (int j = 0; j < MF; ++j) {
        const int m = min(j * 16 + i16, p.M - 1);
        ap[j] = p.a + (int64_t)m * p.lda + q * 16;
        sar[j] = (int64_t)m * p.ldsa;
    }
    const int64_t swr = (int64_t)(n0 / kFp8Block) * p.ldsw;
    f32x4 acc[MF] = {};
    for (int b0 = wave; b0 < p.nkb; b0 += NW * U) {
        i32x4 wv[U][2], av[U][MF][2];
        uint32_t ws[U], as[U][MF];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = b0 + u * NW;
            const bool on = kb < p.nkb;
            const int k = kb * kFp8Block;
            const bool lo = on && k + q * 16 < p.K16, hi = on && k + 64 + q * 16 < p.K16;
            const i32x4 z = {0, 0, 0, 0};
            wv[u][0] = lo ? *(const i32x4 *)(wp + k) : z, wv[u][1] = hi ? *(const i32x4 *)(wp + k + 64) : z;
            ws[u] = on ? load_scale<E8M0>(p.sw, swr + kb) : 0;
#pragma unroll
            for (int j = 0; j < MF; ++j) {
                av[u][j][0] = lo ? *(const i32x4 *)(ap[j] + k) : z, av[u][j][1] = hi ? *(const i32x4 *)(ap[j] + k + 64) : z;
                as[u][j] = on ? load_scale<E8M0>(p.sa, sar[j] + kb) : 0;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Frag<WIDE> wf, af;
            wf.set(wv[u][0], wv[u][1]);
#pragma unroll
            for (int j = 0; j < MF; ++j) {
                af.set(av[u][j][0], av[u][j][1]);
                mma<E8M0, WIDE>(wf, af, acc[j], scale_of<E8M0, WIDE>(ws[u]), scale_of<E8M0, WIDE>(as[u][j]));
            }
        }
    }
#pragma unroll
    for (int j = 0; j < MF; ++j) red[wave][j][lane] = acc[j];
    __syncthreads();
    for (int e = threadIdx.x; e < MF * 64; e += NW * 64) {
        const int j = e >> 6, l = e & 63;
        f32x4 s = red[0][j][l];
#pragma unroll
        for (int w = 1; w < NW; ++w) s += red[w][j][l];
        const int m = j * 16 + (l & 15), n = n0 + (l >> 4) * 4;
        if (m >= p.M || n >= p.N) continue;
        float b[4], v[4];
        load_bias(p, n, b);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = s[r] + b[r];
        store_cols<T, 4>(p, m, n, v);
    }
}

// ---- tiles --------------------------------------------------------------------------------------------------------------------------
// BM x BN of y per workgroup, WM x WN per wave. K's blocks pass through two LDS stages of (BM + BN) x 128 bytes, filled by LDS-DMA
// (16 bytes a lane, no registers) one block ahead. A row's eight 16-byte chunks are stored permuted, chunk c at c ^ key(row), so that the 16
// rows of a fragment read cover all 64 banks; the permutation is applied to the DMA's SOURCE address, its destination is linear.
__device__ __forceinline__ int key_a(int row) { return (row >> 1) & 7; }                                     // fragment rows: consecutive
__device__ __forceinline__ int key_w(int row) { return ((row >> 1) & 1) | (((row >> 4) & 3) << 1); }         // fragment rows: 16 (r / 4) + 4 f + r % 4

template <int BM, int BN, int WM, int WN, bool E8M0, typename T>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void matmul_tile_kernel(MatmulP p) {
    constexpr int NWAVE = (BM / WM) * (BN / WN), FM = WM / 16, FN = WN / 16, STAGE = (BM + BN) * kFp8Block;
    constexpr int PER = (BM + BN) / 8 / NWAVE;
    constexpr bool WIDE = sizeof(T) == 4;
    static_assert(WN % 64 == 0 && (BM + BN) % (8 * NWAVE) == 0 && BM % 8 == 0 && 128 % WN == 0, "tile");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q = lane >> 4;
    // workgroups go to the eight XCDs in turn: give each XCD a run of tiles, walked in bands of 8 tile rows, so that its L2 sees the
    // same operands again
    const int total = p.tiles_m * p.tiles_n;
    int id = blockIdx.x;
    {
        const int xcd = id & 7, at = id >> 3, per = total >> 3, more = total & 7;
        id = xcd * per + min(xcd, more) + at;
    }
    const int band = id / (8 * p.tiles_n), in_band = id - band * 8 * p.tiles_n, rows = min(8, p.tiles_m - band * 8);
    const int tm = band * 8 + in_band % rows, tn = in_band / rows;
    const int m0 = tm * BM, n0 = tn * BN;

    const uint8_t *src[PER];
    int chunk[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int row = (wave + i * NWAVE) * 8 + (lane >> 3);          // rows 0 ... BM - 1: A; then W
        if (row < BM) {
            chunk[i] = (lane & 7) ^ key_a(row);
            src[i] = p.a + (int64_t)min(m0 + row, p.M - 1) * p.lda + chunk[i] * 16;
        } else {
            chunk[i] = (lane & 7) ^ key_w(row - BM);
            src[i] = p.w + (int64_t)min(n0 + row - BM, p.N - 1) * p.ldw + chunk[i] * 16;
        }
    }
    auto fill = [&](int kb, int stage) {
        const int k = kb * kFp8Block;
        const bool ragged = k + kFp8Block > p.K16;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint8_t *s = src[i] + k;
            if (ragged && k + chunk[i] * 16 >= p.K16) s = (const uint8_t *)&g_zero_chunk;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)s,
                                             (__attribute__((address_space(3))) void *)(lds + stage * STAGE + (wave + i * NWAVE) * 1024), 16, 0, 0);
        }
    };

    const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
    int64_t sar[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) sar[j] = (int64_t)min(m0 + wm + j * 16 + i16, p.M - 1) * p.ldsa;
    const int64_t swr = (int64_t)(min(n0 + wn, p.N - 1) / kFp8Block) * p.ldsw;
    // e8m0: four blocks' scale bytes per dword; fp32: one block's. The next ones are on their way while these are used.
    uint32_t sa[FM], san[FM], sw = 0, swn;
    auto fetch = [&](int kb) {
        if constexpr (E8M0) {
            const int at = min(kb, (p.nkb - 1) & ~3);
#pragma unroll
            for (int j = 0; j < FM; ++j) san[j] = *(const uint32_t *)((const uint8_t *)p.sa + sar[j] + at);
            swn = *(const uint32_t *)((const uint8_t *)p.sw + swr + at);
        } else {
            const int at = min(kb, p.nkb - 1);
#pragma unroll
            for (int j = 0; j < FM; ++j) san[j] = load_scale<false>(p.sa, sar[j] + at);
            swn = load_scale<false>(p.sw, swr + at);
        }
    };
    fill(0, 0);
    fetch(0);

    f32x4 acc[FN][FM] = {};
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int kb = 0; kb < p.nkb; ++kb) {
        const uint8_t *st = lds + (kb & 1) * STAGE;
        if (kb + 1 < p.nkb) fill(kb + 1, (kb + 1) & 1);
        if (!E8M0 || (kb & 3) == 0) {
#pragma unroll
            for (int j = 0; j < FM; ++j) sa[j] = san[j];
            sw = swn;
            fetch(kb + (E8M0 ? 4 : 1));
        }
        Frag<WIDE> af[FM];
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int row = wm + j * 16 + i16;
            const uint8_t *r = st + row * kFp8Block;
            af[j].set(*(const i32x4 *)(r + ((q ^ key_a(row)) * 16)), *(const i32x4 *)(r + (((q + 4) ^ key_a(row)) * 16)));
        }
#pragma unroll
        for (int f = 0; f < FN; ++f) {
            const int row = wn + (f >> 2) * 64 + (i16 >> 2) * 16 + (f & 3) * 4 + (i16 & 3);
            const uint8_t *r = st + (BM + row) * kFp8Block;
            Frag<WIDE> wf;
            wf.set(*(const i32x4 *)(r + ((q ^ key_w(row)) * 16)), *(const i32x4 *)(r + (((q + 4) ^ key_w(row)) * 16)));
#pragma unroll
            for (int j = 0; j < FM; ++j) mma<E8M0, WIDE>(wf, af[j], acc[f][j], scale_of<E8M0, WIDE>(sw), scale_of<E8M0, WIDE>(sa[j]));
        }
        if constexpr (E8M0) {
#pragma unroll
            for (int j = 0; j < FM; ++j) sa[j] >>= 8;
            sw >>= 8;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // this wave's part of the next block has landed
        __syncthreads();
    }

#pragma unroll
    for (int g = 0; g < FN / 4; ++g) {
        const int n = n0 + wn + g * 64 + q * 16;
        if (n >= p.N) continue;
        float b[16];
        load_bias(p, n, b);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int m = m0 + wm + j * 16 + i16;
            if (m >= p.M) continue;
            float v[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) v[c] = acc[g * 4 + (c >> 2)][j][c & 3] + b[c];
            store_cols<T, 16>(p, m, n, v);
        }
    }
}

template <int MF, bool E8M0, typename T> static int launch_few(const MatmulP &p, hipStream_t s) {
    const unsigned grid = (unsigned)((p.N + 15) / 16);
    if (p.nkb <= 8) matmul_few_rows_kernel<MF, E8M0, T, 4><<<grid, 256, 0, s>>>(p);
    else matmul_few_rows_kernel<MF, E8M0, T, 8><<<grid, 512, 0, s>>>(p);
    return launch_status("matmul_fp8");
}

template <int BM, int BN, int WM, int WN, bool E8M0, typename T> static int launch_tile(MatmulP p, hipStream_t s) {
    static LdsGrant grant;
    constexpr size_t bytes = 2 * (BM + BN) * kFp8Block;
    if (int rc = grant.ensure((const void *)matmul_tile_kernel<BM, BN, WM, WN, E8M0, T>, bytes, 64 * 1024)) return rc;
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
    LSSVC_CHECK(total < (1LL << 28), "matmul_fp8: %lld tiles do not fit one launch", (long long)total);
    matmul_tile_kernel<BM, BN, WM, WN, E8M0, T><<<(unsigned)total, (BM / WM) * (BN / WN) * 64, bytes, s>>>(p);
    return launch_status("matmul_fp8");
}

template <bool E8M0, typename T> static int launch_matmul(const MatmulP &p, hipStream_t s) {
    if (p.M <= 16) return launch_few<1, E8M0, T>(p, s);
    if (p.M <= 32) return launch_few<2, E8M0, T>(p, s);
    auto tiles = [&](int bm, int bn) { return (int64_t)((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
    if constexpr (sizeof(T) == 2)
        if (tiles(256, 256) >= 200) return launch_tile<256, 256, 128, 64, E8M0, T>(p, s);
    if (tiles(128, 128) >= 200) return launch_tile<128, 128, 64, 64, E8M0, T>(p, s);
    return launch_tile<64, 64, 16, 64, E8M0, T>(p, s);
}
template <bool E8M0> static int launch_typed(const MatmulP &p, hipStream_t s) {
    if (p.dtype == LSSVC_F32) return launch_matmul<E8M0, float>(p, s);
    if (p.dtype == LSSVC_F16) return launch_matmul<E8M0, f16_t>(p, s);
    return launch_matmul<E8M0, bf16_t>(p, s);
}

static int operand_check(const lssvc_fp8 *x, const char *who, int block_rows) {
    LSSVC_CHECK(x && x->rows >= 0 && x->cols > 0 && x->reserved == 0, "matmul_fp8: bad operand %s", who);
    LSSVC_CHECK(x->rows == 0 || (x->values && x->scale), "matmul_fp8: operand %s has no data", who);
    LSSVC_CHECK(x->block_rows == block_rows, "matmul_fp8: operand %s has scales for %d rows, expected %d", who, x->block_rows, block_rows);
    LSSVC_CHECK(aligned(x->values, 16) && x->ld % 16 == 0 && x->ld >= ((int64_t)x->cols + 15) / 16 * 16, "matmul_fp8: operand %s needs a 16-byte aligned base and a pitch that is a multiple of 16", who);
    const int64_t kb = ((int64_t)x->cols + kFp8Block - 1) / kFp8Block;
    LSSVC_CHECK(x->scale_ld >= kb && aligned(x->scale, 4) && (!x->scale_e8m0 || x->scale_ld % 4 == 0), "matmul_fp8: operand %s: bad scale layout", who);
    LSSVC_CHECK(x->rows < (1LL << 31) - 512 && x->cols <= (1 << 30) && x->ld < (1LL << 32), "matmul_fp8: operand %s is too large", who);
    return 0;
}

}  // namespace lssvc

using namespace lssvc;

extern "C" int64_t lssvc_matmul_fp8_workspace_bytes(int64_t m, int64_t n, int32_t k) {
    (void)m, (void)n, (void)k;
    return 0;
}

extern "C" int lssvc_matmul_fp8(const lssvc_fp8 *a, const lssvc_fp8 *w, const float *bias, int32_t act, float slope, const lssvc_rows *residual,
                                const lssvc_rows *y, void *workspace, int64_t workspace_bytes, void *stream) {
    (void)workspace, (void)workspace_bytes;
    if (int rc = operand_check(a, "a", 1)) return rc;
    if (int rc = operand_check(w, "w", kFp8Block)) return rc;
    LSSVC_CHECK(a->cols == w->cols, "matmul_fp8: a has %d columns, w has %d", a->cols, w->cols);
    LSSVC_CHECK((a->scale_e8m0 != 0) == (w->scale_e8m0 != 0), "matmul_fp8: one operand has e8m0 scales, the other fp32 scales");
    LSSVC_CHECK(act_ok(act), "matmul_fp8: unknown activation %d", act);
    LSSVC_CHECK(y && rows_type_ok(y->dtype) && y->rows == a->rows && y->cols == w->rows && y->ld >= y->cols && y->ld < (1LL << 32), "matmul_fp8: the output is not %lld x %lld", (long long)a->rows, (long long)w->rows);
    if (a->rows == 0 || w->rows == 0) return 0;
    LSSVC_CHECK(y->ptr && aligned(y->ptr, rows_type_size(y->dtype)), "matmul_fp8: bad output pointer");
    if (residual) {
        LSSVC_CHECK(residual->ptr && residual->rows == y->rows && residual->cols == y->cols && residual->dtype == y->dtype && residual->ld >= residual->cols && residual->ld < (1LL << 32) &&
                        aligned(residual->ptr, rows_type_size(y->dtype)), "matmul_fp8: the residual's shape or type is not the output's");
        LSSVC_CHECK(rows_disjoint_or_same(residual, y), "matmul_fp8: residual and output overlap in part");
    }
    MatmulP p{};
    p.a = (const uint8_t *)a->values, p.w = (const uint8_t *)w->values;
    p.sa = a->scale, p.sw = w->scale;
    p.lda = a->ld, p.ldw = w->ld, p.ldsa = a->scale_ld, p.ldsw = w->scale_ld;
    p.bias = bias;
    p.res = residual ? residual->ptr : nullptr, p.ldres = residual ? residual->ld : 0;
    p.y = y->ptr, p.ldy = y->ld;
    p.M = (int)a->rows, p.N = (int)w->rows, p.K16 = (a->cols + 15) / 16 * 16, p.nkb = (a->cols + kFp8Block - 1) / kFp8Block;
    p.dtype = y->dtype, p.act = make_act(act, slope);
    return a->scale_e8m0 ? launch_typed<true>(p, (hipStream_t)stream) : launch_typed<false>(p, (hipStream_t)stream);
}
