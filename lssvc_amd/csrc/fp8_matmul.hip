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
#include <algorithm>
#include <cmath>
#include <type_traits>
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

// a fragment as it is read: chunks q and q + 4 of a row's block
struct Raw {
    i32x4 lo, hi;
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

// (block of W) (block of A)^T without the scales
template <bool WIDE> __device__ __forceinline__ f32x4 product(const Frag<WIDE> &w, const Frag<WIDE> &a) {
    f32x4 part = {0.f, 0.f, 0.f, 0.f};
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) part = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], a.v[i], part, 0, 0, 0);
    } else part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, part, 0, 0, 0, 0, 0, 0);      // (unscaled)
    return part;
}
__device__ __forceinline__ void add_scaled(f32x4 &acc, const f32x4 &part, float s) {
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] = fmaf(part[r], s, acc[r]);
}
// acc += sw * sa * (block of W) (block of A)^T; WB: the byte of sw that the scaled instruction takes
template <bool E8M0, bool WIDE, int WB = 0, typename S>
__device__ __forceinline__ void mma(const Frag<WIDE> &w, const Frag<WIDE> &a, f32x4 &acc, S sw, S sa) {
    if constexpr (E8M0 && !WIDE) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, acc, 0, 0, WB, sw, 0, sa);
    else add_scaled(acc, product<WIDE>(w, a), sw * sa);
}

// act(v) + residual for CNT consecutive columns of one row, rounded once. FULL: all of them are inside; otherwise the first `left`.
template <bool FULL, typename T, int CNT>
__device__ __forceinline__ void store_cols(const Act &act, T *dst, const T *res, int left, float (&v)[CNT]) {
    apply_act(v, act);
    if (res) {
        Pack<T, CNT> r;
        if (FULL) r = load_pack<T, CNT>(res);
        else
#pragma unroll
            for (int i = 0; i < CNT; ++i) r.v[i] = i < left ? res[i] : from_f32<T>(0.f);
#pragma unroll
        for (int i = 0; i < CNT; ++i) v[i] += to_f32(r.v[i]);
    }
    Pack<T, CNT> o;
#pragma unroll
    for (int i = 0; i < CNT; ++i) o.v[i] = from_f32<T>(v[i]);
    if (FULL) store_pack(dst, o);
    else
#pragma unroll
        for (int i = 0; i < CNT; ++i)
            if (i < left) dst[i] = o.v[i];
}
template <int CNT> __device__ __forceinline__ void load_bias(const MatmulP &p, int n, float (&b)[CNT]) {
#pragma unroll
    for (int i = 0; i < CNT; ++i) b[i] = p.bias && n + i < p.N ? p.bias[n + i] : 0.f;
}

template <bool E8M0> __device__ __forceinline__ uint32_t load_scale(const void *s, int64_t at) {
    if constexpr (E8M0) return ((const uint8_t *)s)[at];
    else return ((const uint32_t *)s)[at];
}

// ---- small products: bound by the weight's bytes, or by latency ------------------------------------------------------------------------
// A workgroup owns MF * 16 rows and NF * 16 columns of y; its waves deal K's blocks among themselves, read both operands straight into
// registers (nothing is read twice within the workgroup, no barrier until the end, little code) and add up through the LDS in a fixed order.
template <int MF, int NF, bool E8M0, typename T, int NW>
__global__ __launch_bounds__(NW * 64) void matmul_direct_kernel(MatmulP p) {
    constexpr int U = MF + NF <= 3 ? 4 : MF + NF <= 5 ? 2 : 1;     // blocks of K in flight per wave
    constexpr int C = 4 * NF;                                      // consecutive columns of y per lane
    constexpr bool WIDE = sizeof(T) == 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    f32x4 *red = (f32x4 *)lds;                                     // [wave][column fragment][row fragment][lane]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, q = lane >> 4;
    const int tm = blockIdx.x / (unsigned)p.tiles_n, tn = blockIdx.x - tm * p.tiles_n;
    const int m0 = tm * (16 * MF), n0 = tn * (16 * NF);
    const uint8_t *wp[NF], *ap[MF];
    int64_t sar[MF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const int n = n0 + (NF == 1 ? i16 : (i16 >> 2) * C + f * 4 + (i16 & 3));
        wp[f] = p.w + (int64_t)min(n, p.N - 1) * p.ldw + q * 16;
    }
#pragma unroll
    for (int j = 0; j < MF; ++j) {
        const int64_t m = min(m0 + j * 16 + i16, p.M - 1);
        ap[j] = p.a + m * p.lda + q * 16;
        sar[j] = m * p.ldsa;
    }
    const int64_t swr = (int64_t)(n0 / kFp8Block) * p.ldsw;
    f32x4 acc[NF][MF] = {};
    for (int b0 = wave; b0 < p.nkb; b0 += NW * U) {
        Raw wv[U][NF], av[U][MF];
        uint32_t ws[U], as[U][MF];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = b0 + u * NW, k = kb * kFp8Block;
            const bool on = kb < p.nkb, lo = on && k + q * 16 < p.K16, hi = on && k + 64 + q * 16 < p.K16;
            const i32x4 z = {0, 0, 0, 0};
#pragma unroll
            for (int f = 0; f < NF; ++f) wv[u][f] = Raw{lo ? *(const i32x4 *)(wp[f] + k) : z, hi ? *(const i32x4 *)(wp[f] + k + 64) : z};
            ws[u] = on ? load_scale<E8M0>(p.sw, swr + kb) : 0;
#pragma unroll
            for (int j = 0; j < MF; ++j) {
                av[u][j] = Raw{lo ? *(const i32x4 *)(ap[j] + k) : z, hi ? *(const i32x4 *)(ap[j] + k + 64) : z};
                as[u][j] = on ? load_scale<E8M0>(p.sa, sar[j] + kb) : 0;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Frag<WIDE> wf[NF], af;
#pragma unroll
            for (int f = 0; f < NF; ++f) wf[f].set(wv[u][f].lo, wv[u][f].hi);
#pragma unroll
            for (int j = 0; j < MF; ++j) {
                af.set(av[u][j].lo, av[u][j].hi);
#pragma unroll
                for (int f = 0; f < NF; ++f) mma<E8M0, WIDE>(wf[f], af, acc[f][j], scale_of<E8M0, WIDE>(ws[u]), scale_of<E8M0, WIDE>(as[u][j]));
            }
        }
    }
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int j = 0; j < MF; ++j) red[((wave * NF + f) * MF + j) * 64 + lane] = acc[f][j];
    __syncthreads();
    const int waves = min(NW, p.nkb);                              // (the others had no block)
    for (int e = threadIdx.x; e < MF * 64; e += NW * 64) {
        const int64_t m = m0 + (e >> 6) * 16 + (e & 15), n = n0 + ((e >> 4) & 3) * C;
        if (m >= p.M || n >= p.N) continue;
        float v[C];
        load_bias(p, n, v);
        f32x4 s[NF] = {};
        for (int w = 0; w < waves; ++w)
#pragma unroll
            for (int f = 0; f < NF; ++f) s[f] += red[(w * NF + f) * MF * 64 + e];
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] += s[c >> 2][c & 3];
        T *dst = (T *)p.y + m * p.ldy + n;
        const T *res = p.res ? (const T *)p.res + m * p.ldres + n : nullptr;
        if (n0 + 16 * NF <= p.N) store_cols<true, T, C>(p.act, dst, res, C, v);        // (the workgroup agrees)
        else store_cols<false, T, C>(p.act, dst, res, p.N - n, v);
    }
}

// ---- tiles --------------------------------------------------------------------------------------------------------------------------
// BM x BN of y per workgroup, WM x WN per wave. K's blocks pass through two LDS stages of (BM + BN) x 128 bytes, filled by LDS-DMA
// (16 bytes a lane, no registers). A row's eight 16-byte chunks are stored permuted, chunk c at c ^ key(row), so that the 16 rows of a
// fragment read cover all 64 banks; the permutation is applied to the DMA's SOURCE address, its destination is linear.
//
// The matrix units are the bound, so they must not see the LDS: a wave multiplies the fragments of A one after the other against its FN
// fragments of W and reads PD fragments ahead, over the end of the block too. The one barrier of a block stands PD fragments before its
// end: there every wave has all of this block in registers and its part of the next one has landed; behind it the stage just read
// is filled with the block after the next, a quarter of the instructions with each of the next four fragments. (All at once they fill the
// address unit's queue, and the waves stand in front of it with the matrix units idle: 0.5 us of a block's 1.8 at 256 x 256.)
__device__ __forceinline__ int key_a(int row) { return (row >> 1) & 7; }                                     // fragment rows: consecutive
__device__ __forceinline__ int key_w(int row) { return ((row >> 1) & 1) | (((row >> 4) & 3) << 1); }         // fragment rows: 16 (r / 4) + 4 f + r % 4

struct RawA {
    i32x4 lo, hi;
    uint32_t scale;
};
// a raw buffer of the bytes [p, p + range)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(const uint8_t *p, int range) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, range, 0x00027000);
}
// a value that all lanes share, in scalar registers
__device__ __forceinline__ const uint8_t *uniform(const uint8_t *p) {
    const uint64_t v = (uint64_t)p;
    return (const uint8_t *)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

template <int BM, int BN, int WM, int WN, bool E8M0, typename T>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void matmul_tile_kernel(MatmulP p) {
    constexpr int NWAVE = (BM / WM) * (BN / WN), FM = WM / 16, FN = WN / 16, STAGE = (BM + BN) * kFp8Block;
    constexpr int PA = BM / 8 / NWAVE, PW = BN / 8 / NWAVE;    // DMA instructions of a wave per block
    constexpr int SLOTS = 2, PD = 1, LAST = FM - PD;
    constexpr int DPG = (PA + PW + 3) / 4;                     // DMA instructions per fragment of A
    constexpr bool WIDE = sizeof(T) == 4;
    static_assert(WN % 64 == 0 && BM % (8 * NWAVE) == 0 && BN % (8 * NWAVE) == 0 && 128 % WN == 0 && FM % SLOTS == 0 && FM >= 4, "tile");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15, q = lane >> 4;
    // workgroups go to the eight XCDs in turn: give each XCD a run of tiles, walked in bands of 8 tile rows, so that its L2 sees the
    // same operands again
    const int total = p.tiles_m * p.tiles_n;
    int id = blockIdx.x;
    {
        const int xcd = id & 7, at = id >> 3, per = total >> 3, more = total & 7;
        id = xcd * per + min(xcd, more) + at;
    }
    const int band = id / (8 * p.tiles_n), in_band = id - band * 8 * p.tiles_n, rows = min(8, p.tiles_m - band * 8);
    const int tm = __builtin_amdgcn_readfirstlane(band * 8 + in_band % rows), tn = __builtin_amdgcn_readfirstlane(in_band / rows);
    const int m0 = tm * BM, n0 = tn * BN;

    // Both operands are read through buffer descriptors that start at the tile's rows: a lane's offset within the tile in a register (the host
    // keeps 256 pitches below 2^31), k in the instruction's scalar offset. Rows behind the last one are the last one (their results are not
    // stored); chunks behind K16 get an offset beyond the range and arrive as zeros; a block behind the last one is the last one.
    constexpr int STEP = 8 * NWAVE;                            // rows between two DMA instructions of a wave
    const uint8_t *abase = uniform(p.a + (int64_t)m0 * p.lda), *wbase = uniform(p.w + (int64_t)n0 * p.ldw);
    const int drow = wave * 8 + (lane >> 3);
    const int achunk = ((lane & 7) ^ key_a(drow)) * 16;        // (the key of a row of A repeats after 16 rows, that of W after 64)
    uint32_t aoff[PA], woff[PW];
    int wchunk[PW];
#pragma unroll
    for (int i = 0; i < PA; ++i) aoff[i] = (uint32_t)min(drow + i * STEP, p.M - 1 - m0) * (uint32_t)p.lda + achunk;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
        wchunk[i] = ((lane & 7) ^ key_w(drow + i * STEP)) * 16;
        woff[i] = (uint32_t)min(drow + i * STEP, p.N - 1 - n0) * (uint32_t)p.ldw + wchunk[i];
    }
    auto dma = [&](const uint8_t *base, uint32_t off, int k, int at) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(descriptor(base, 0x7fffffff), (__attribute__((address_space(3))) void *)(lds + at), 16, off, k, 0, 0);
    };
    auto fill = [&](int kb, int from, int to) {                // DMA instructions from ... to - 1 of a block's
        const int k = min(kb, p.nkb - 1) * kFp8Block, at = (kb & 1) * STAGE + wave * 1024;
#pragma unroll
        for (int i = 0; i < PA + PW; ++i) {
            if (i < from || i >= to) continue;
            if (i < PA) dma(abase, k + achunk < p.K16 ? aoff[i] : 0x80000000u, k, at + i * STEP * kFp8Block);
            else dma(wbase, k + wchunk[i - PA] < p.K16 ? woff[i - PA] : 0x80000000u, k, at + (BM + (i - PA) * STEP) * kFp8Block);
        }
    };

    // A's scales go through the LDS as well, for four blocks of K at a time (a dword of e8m0 bytes or four fp32 values per row, two such groups):
    // read straight from memory every wave would gather them for itself, 16 cache lines an instruction, and the address unit would be the
    // bound. A wave's DMA covers 64 rows; where there are more waves than that some write the same values twice.
    const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
    constexpr int SB = E8M0 ? 1 : 4, SROW = 4 * SB;
    const int srow = (wave * 64) % BM;
    // (a group behind the last one is the last one; behind the row's last scale the buffer may end, so the range does: zeros)
    const uint8_t *sabase = uniform((const uint8_t *)p.sa + (int64_t)m0 * p.ldsa * SB);
    const int64_t sleft = ((int64_t)(p.M - 1 - m0) * p.ldsa + (E8M0 ? (p.nkb + 3) & ~3 : p.nkb)) * SB;
    const int srange = __builtin_amdgcn_readfirstlane((int)min(sleft, (int64_t)0x7fffffff));
    const uint32_t saoff = (uint32_t)min(srow + lane, p.M - 1 - m0) * (uint32_t)p.ldsa * SB;
    auto fill_scales = [&](int g) {
        const int gk = min(g, (p.nkb - 1) >> 2) * SROW;
        const auto to = (__attribute__((address_space(3))) void *)(lds + 2 * STAGE + ((g & 1) * BM + srow) * SROW);
        if constexpr (E8M0) __builtin_amdgcn_raw_ptr_buffer_load_lds(descriptor(sabase, srange), to, 4, saoff + gk, 0, 0, 0);
        else __builtin_amdgcn_raw_ptr_buffer_load_lds(descriptor(sabase, srange), to, 16, saoff + gk, 0, 0, 0);
    };
    // W's scales: one per block and wave, in registers, four blocks at a time
    const uint8_t *swp = (const uint8_t *)p.sw + (int64_t)(min(n0 + wn, p.N - 1) / kFp8Block) * p.ldsw * SB;
    constexpr int NSW = E8M0 ? 1 : 4;
    uint32_t sw[NSW], swn[NSW];
    auto fetch_w = [&](int g, uint32_t (&to)[NSW]) {
        if constexpr (E8M0) to[0] = *(const uint32_t *)(swp + min(g * 4, (p.nkb - 1) & ~3));
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = *(const uint32_t *)(swp + 4 * min(g * 4 + i, p.nkb - 1));
    };

    // fragment addresses within a stage: consecutive fragments of A are 16 rows apart and share their key; those of W differ in row bits 3:2,
    // which the key does not see
    const int arow = wm + i16, wrow = wn + (i16 >> 2) * 16 + (i16 & 3);
    const int a_lo = arow * kFp8Block + ((q ^ key_a(arow)) * 16), a_hi = arow * kFp8Block + (((q + 4) ^ key_a(arow)) * 16);
    const int w_lo = (BM + wrow) * kFp8Block + ((q ^ key_w(wrow)) * 16), w_hi = (BM + wrow) * kFp8Block + (((q + 4) ^ key_w(wrow)) * 16);
    const int sc0 = 2 * STAGE + arow * SROW;
    auto read_a = [&](int kb, int j) {
        const uint8_t *st = lds + (kb & 1) * STAGE + j * (16 * kFp8Block), *sc = lds + sc0 + ((kb >> 2) & 1) * (BM * SROW) + (kb & 3) * SB + j * (16 * SROW);
        RawA r{*(const i32x4 *)(st + a_lo), *(const i32x4 *)(st + a_hi), 0};
        if constexpr (E8M0) r.scale = *sc;
        else r.scale = *(const uint32_t *)sc;
        return r;
    };
    auto read_w = [&](int kb, int f) {
        const uint8_t *st = lds + (kb & 1) * STAGE + ((f >> 2) * 64 + (f & 3) * 4) * kFp8Block;
        return Raw{*(const i32x4 *)(st + w_lo), *(const i32x4 *)(st + w_hi)};
    };

    fill(0, 0, PA + PW);
    fill_scales(0);
    fetch_w(0, sw);
    f32x4 acc[FN][FM] = {};
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    fill(1, 0, DPG);
    Raw wraw[FN];
    RawA araw[SLOTS];
#pragma unroll
    for (int f = 0; f < FN; ++f) wraw[f] = read_w(0, f);
#pragma unroll
    for (int j = 0; j < PD; ++j) araw[j] = read_a(0, j);
    // parts that are scaled by the vector unit are added one product later: the matrix unit has the next one by then
    constexpr bool BY_PART = !E8M0 || WIDE;
    f32x4 late = {0.f, 0.f, 0.f, 0.f};
    float late_scale = 0.f;
    // one block of K; S = kb % 4. No branches inside: the compiler would gather the products behind them. (A block behind the last one is filled
    // with zeros, its descriptor's range being empty, and read for nothing.)
    auto step = [&](int kb, auto s_) {
        constexpr int S = decltype(s_)::value;
        Frag<WIDE> wf[FN];
#pragma unroll
        for (int f = 0; f < FN; ++f) wf[f].set(wraw[f].lo, wraw[f].hi);
        if constexpr (S == 0) fetch_w((kb >> 2) + 1, swn);
        const auto swv = scale_of<E8M0, WIDE>(E8M0 ? (WIDE ? sw[0] >> (8 * S) : sw[0]) : sw[E8M0 ? 0 : S]);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            if (j == LAST) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");        // this block is in registers, this wave's part of the next has landed
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if constexpr (S == 1) fill_scales((kb >> 2) + 1);
                fill(kb + 2, 0, DPG);
            } else if (j < 3) fill(kb + 1, (j + 1) * DPG, (j + 2) * DPG);
            if (j + PD < FM) araw[(j + PD) % SLOTS] = read_a(kb, j + PD);
            else araw[(j + PD) % SLOTS] = read_a(kb + 1, j + PD - FM);
            __builtin_amdgcn_sched_barrier(0);
            Frag<WIDE> af;
            af.set(araw[j % SLOTS].lo, araw[j % SLOTS].hi);
            const auto sav = scale_of<E8M0, WIDE>(araw[j % SLOTS].scale);
#pragma unroll
            for (int f = 0; f < FN; ++f) {
                if constexpr (BY_PART) {
                    const f32x4 part = product<WIDE>(wf[f], af);
                    __builtin_amdgcn_sched_barrier(0);
                    f32x4 &to = f ? acc[f - 1][j] : j ? acc[FN - 1][j - 1] : acc[FN - 1][FM - 1];
                    add_scaled(to, late, late_scale);
                    asm volatile("" : "+v"(to));               // (the sum is made here: kept back, the parts would fill the registers)
                    late = part, late_scale = swv * sav;
                } else mma<E8M0, WIDE, S>(wf[f], af, acc[f][j], swv, sav);
                if (j == FM - 1) {                             // this was the fragment's last use: the next block's takes its registers
                    __builtin_amdgcn_sched_barrier(0);
                    wraw[f] = read_w(kb + 1, f);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (S == 3)
#pragma unroll
            for (int i = 0; i < NSW; ++i) sw[i] = swn[i];
    };
    for (int kb = 0;;) {
        step(kb, std::integral_constant<int, 0>{});
        if (++kb == p.nkb) break;
        step(kb, std::integral_constant<int, 1>{});
        if (++kb == p.nkb) break;
        step(kb, std::integral_constant<int, 2>{});
        if (++kb == p.nkb) break;
        step(kb, std::integral_constant<int, 3>{});
        if (++kb == p.nkb) break;
    }

    if constexpr (BY_PART) add_scaled(acc[FN - 1][FM - 1], late, late_scale);

    // Out through the LDS, 64 (or 48) rows of a wave's tile at a time in a part of its own: whole 128- or 256-byte pieces of rows, and a short loop
    // instead of a long unrolled one (a tile's registers cannot be indexed; 16 KB of code cost more to fetch than the tile takes to store).
    // A row's 16-byte chunk c lies at c ^ (row % 16): both directions cover the banks.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");                    // (fills behind the last block)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    constexpr int HJ = FM % 4 ? 3 : 4;                         // fragments of A at a time
    static_assert(FM % HJ == 0 && FN == 4 && NWAVE * HJ * 4096 <= 2 * STAGE, "epilogue");
    f32x4 *part = (f32x4 *)(lds + wave * (HJ * 4096));
    const int c8 = lane & 7, n = n0 + wn + c8 * 8;
    float bias[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        bias[i] = p.bias ? p.bias[min(n + i, p.N - 1)] : 0.f;
        asm volatile("" : "+v"(bias[i]));                      // (waited for here, not in the loop: there the wait would be for its stores)
    }
    const int r0 = lane >> 3, x0 = (c8 * 2) ^ r0, y0 = (c8 * 2 + 1) ^ r0;          // (rows r0 + 8 k: the key alternates between r0 and r0 ^ 8)
    auto out = [&](auto full_, int mh) {
        constexpr bool FULL = decltype(full_)::value;
        const int rows_left = min(HJ * 16, p.M - mh);
        T *dst = (T *)p.y + (int64_t)(mh + r0) * p.ldy + n;
        const T *res = (const T *)p.res + (p.res ? (int64_t)(mh + r0) * p.ldres + n : 0);
        const f32x4 *from = part + r0 * 16;
#pragma unroll 2
        for (int k = 0; k < HJ * 2; ++k) {
            const f32x4 x = from[x0 ^ ((k & 1) * 8)], y = from[y0 ^ ((k & 1) * 8)];
            float v[8] = {x[0] + bias[0], x[1] + bias[1], x[2] + bias[2], x[3] + bias[3], y[0] + bias[4], y[1] + bias[5], y[2] + bias[6], y[3] + bias[7]};
            if (r0 + 8 * k < rows_left && (FULL || n < p.N)) store_cols<FULL, T, 8>(p.act, dst, p.res ? res : nullptr, p.N - n, v);
            dst += 8 * p.ldy;
            res += 8 * p.ldres;
            from += 8 * 16;
        }
    };
#pragma unroll
    for (int h = 0; h < FM / HJ; ++h) {
#pragma unroll
        for (int j = 0; j < HJ; ++j)
#pragma unroll
            for (int f = 0; f < 4; ++f) part[(j * 16 + i16) * 16 + ((q * 4 + f) ^ i16)] = acc[f][h * HJ + j];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (n0 + BN <= p.N) out(std::true_type{}, m0 + wm + h * (HJ * 16));
        else out(std::false_type{}, m0 + wm + h * (HJ * 16));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <int MF, int NF, bool E8M0, typename T, int NW> static int launch_direct(const MatmulP &p, int64_t total, hipStream_t s) {
    static LdsGrant grant;
    constexpr size_t bytes = (size_t)NW * MF * NF * 1024;
    if (int rc = grant.ensure((const void *)matmul_direct_kernel<MF, NF, E8M0, T, NW>, bytes, 64 * 1024)) return rc;
    matmul_direct_kernel<MF, NF, E8M0, T, NW><<<(unsigned)total, NW * 64, bytes, s>>>(p);
    return launch_status("matmul_fp8");
}
template <int MF, int NF, bool E8M0, typename T> static int launch_direct(MatmulP p, hipStream_t s) {
    p.tiles_m = (p.M + 16 * MF - 1) / (16 * MF);
    p.tiles_n = (p.N + 16 * NF - 1) / (16 * NF);
    const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
    LSSVC_CHECK(total < (1LL << 31), "matmul_fp8: %lld tiles do not fit one launch", (long long)total);
    // (8 waves need 8 blocks each has one of; 16 waves are no faster at any size)
    return p.nkb <= 8 ? launch_direct<MF, NF, E8M0, T, 4>(p, total, s) : launch_direct<MF, NF, E8M0, T, 8>(p, total, s);
}

template <int BM, int BN, int WM, int WN, bool E8M0, typename T> static int launch_tile(MatmulP p, hipStream_t s) {
    static LdsGrant grant;
    constexpr size_t bytes = 2 * (BM + BN) * kFp8Block + 2 * BM * (E8M0 ? 4 : 16);
    if (int rc = grant.ensure((const void *)matmul_tile_kernel<BM, BN, WM, WN, E8M0, T>, bytes, 64 * 1024)) return rc;
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
    LSSVC_CHECK(total < (1LL << 28), "matmul_fp8: %lld tiles do not fit one launch", (long long)total);
    matmul_tile_kernel<BM, BN, WM, WN, E8M0, T><<<(unsigned)total, (BM / WM) * (BN / WN) * 64, bytes, s>>>(p);
    return launch_status("matmul_fp8");
}

// Which form: the one with the least estimated time, in us, from times measured at 26 sizes between 1 x 4096 x 4096 and 8192^3 (bf16, e8m0;
// estimates are within 30 % of them). Direct: 3 us, what its workgroups read (6.5 MB a us if all CUs have one) and 0.25 us for every 256
// workgroups. Tiles: a start, and for every tile that a CU gets its blocks of K and an end. Two rounds' worth of tiles cost two rounds: the
// estimate is where the 256 x 256 form's half-empty last round is weighed against the smaller tiles' lower rate.
template <bool E8M0, typename T> static int launch_matmul(const MatmulP &p, hipStream_t s) {
    constexpr bool WIDE = sizeof(T) == 4;
    auto tiles = [&](int bm, int bn) { return (double)((p.M + bm - 1) / bm) * (double)((p.N + bn - 1) / bn); };
    auto direct = [&](int mf, int nf) {
        const double t = tiles(16 * mf, 16 * nf);
        return 3.0 + t * p.nkb * (mf + nf) * 2048 / (6.5e6 * std::min(1.0, t / 256)) + t / 1024;
    };
    auto tiled = [&](int bm, int bn, double start, double block, double end) { return start + std::ceil(tiles(bm, bn) / 256) * (p.nkb * block + end); };
    // (a pitch that is no multiple of 128: a block of K straddles two lines)
    const double rate = (WIDE ? 1.9 : E8M0 ? 1.0 : 1.17) * ((p.lda | p.ldw) % 128 && p.nkb > 1 ? 1.6 : 1.0);
    const double cost[7] = {direct(1, 1), direct(1, 4), direct(2, 4), direct(4, 4), tiled(128, 128, 4.5, 0.56 * rate, 1.0),
                            WIDE ? 1e30 : tiled(256, 256, 7.0, 1.42 * rate, 5.0), WIDE ? 1e30 : tiled(192, 256, 6.5, 1.12 * rate, 4.0)};
#ifdef FP8_SWEEP
    const int best = getenv("FP8_FORCE") && atoi(getenv("FP8_FORCE")) >= 0 ? atoi(getenv("FP8_FORCE")) : (int)(std::min_element(cost, cost + 7) - cost);
#else
    const int best = (int)(std::min_element(cost, cost + 7) - cost);
#endif
    switch (best) {
        case 0: return launch_direct<1, 1, E8M0, T>(p, s);
        case 1: return launch_direct<1, 4, E8M0, T>(p, s);
        case 2: return launch_direct<2, 4, E8M0, T>(p, s);
        case 3: return launch_direct<4, 4, E8M0, T>(p, s);
        case 5:
            if constexpr (!WIDE) return launch_tile<256, 256, 128, 64, E8M0, T>(p, s);
            break;
        case 6:
            if constexpr (!WIDE) return launch_tile<192, 256, 96, 64, E8M0, T>(p, s);
            break;
    }
    return launch_tile<128, 128, 64, 64, E8M0, T>(p, s);
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
    LSSVC_CHECK(x->rows < (1LL << 31) - 512 && x->ld < (1LL << 22) && x->scale_ld < (1LL << 21), "matmul_fp8: operand %s is too large", who);
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
    p.dtype = y->dtype, p.act = Act{act, slope};
    return a->scale_e8m0 ? launch_typed<true>(p, (hipStream_t)stream) : launch_typed<false>(p, (hipStream_t)stream);
}
