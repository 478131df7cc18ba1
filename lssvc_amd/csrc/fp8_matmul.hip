// fp8_matmul.hip -- y = act(A W^T + bias) + residual for 8-bit rows with a scale for each block of 128 along K.
//
// 16-bit results: one v_mfma_f32_16x16x128_f8f6f4 covers exactly one block of K, so a block's scales belong to one instruction:
//   e8m0 scales  the scaled form of the instruction multiplies by 2^(sa + sw) itself; the accumulator runs over all of K.
//   fp32 scales  each block's product starts from zero and is added to the accumulator with one FMA per value, factor sa * sw.
// The 8-bit instructions (every form) cut the products of 8 neighbouring columns toward zero at 2^(e - 13), e the largest sum of two operands'
// exponents among the 8, and add in fp32 from there on: measured, and bit for bit so in the tests. Of the result in the 2-norm that is 1.5e-5 for
// operands that are 8-bit roundings of normal numbers (K = 1000 ... 50000), 2.1e-5 ... 2.4e-5 where channels differ in spread, 6.7e-5 where one of
// 8 is 64 times the others, 2.6e-6 (all of it toward zero) where all products are positive. Beside the rounding of bf16 results that is
// nothing, fp16 results are 0.3 - 5 % further from the exact ones than one rounding would leave them, and fp32 results would be off by hundreds of half
// steps. Where the large products of a group cancel, what is left may be wrong altogether: a caller whose sums do takes fp32 results.
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
    int depth;               // LDS stages of a wave (split form)
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

// ---- operands on their way to the LDS ---------------------------------------------------------------------------------------------------
// Both kernels fill the LDS by DMA, 8 rows x 128 bytes an instruction: whole lines. (Fragments loaded straight into registers are 16 rows x 64
// bytes an instruction, and the address unit takes 3.5 cycles a line however much of it is used: half the rate, measured.) A row's eight
// 16-byte chunks are stored permuted, chunk c at c ^ key(row), so that the 16 rows of a fragment read cover all 64 banks; the permutation is
// applied to the DMA's SOURCE address, its destination is linear.
__device__ __forceinline__ int key_a(int row) { return (row >> 1) & 7; }                                     // fragment rows: consecutive
__device__ __forceinline__ int key_w(int row) { return ((row >> 1) & 1) | (((row >> 4) & 3) << 1); }         // fragment rows: 16 (r / 4) + 4 f + r % 4

// a raw buffer of the bytes [p, p + range)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(const uint8_t *p, int range) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, range, 0x00027000);
}
// a value that all lanes share, in scalar registers
__device__ __forceinline__ const uint8_t *uniform(const uint8_t *p) {
    const uint64_t v = (uint64_t)p;
    return (const uint8_t *)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}
// 16 bytes a lane from base + off (bytes; beyond 2^31: zeros) + k to the LDS at `to`, lane after lane
__device__ __forceinline__ void dma(const uint8_t *base, uint32_t off, int k, uint8_t *to) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(descriptor(base, 0x7fffffff), (__attribute__((address_space(3))) void *)to, 16, off, k, 0, 0);
}
constexpr uint32_t kOutside = 0x80000000u;
// Workgroups go to the eight XCDs in turn: the work of workgroup `id` of `total` if each XCD is to have a run of neighbours
__device__ __forceinline__ int xcd_run(int id, int total) {
    const int xcd = id & 7, per = total >> 3, more = total & 7;
    return xcd * per + min(xcd, more) + (id >> 3);
}

// ---- small products: bound by the weight's bytes, or by latency ------------------------------------------------------------------------
// A workgroup owns MF * 16 rows and NF * 16 columns of y. Its waves deal K's blocks among themselves: nothing is read twice within the
// workgroup, each wave fills and reads a part of the LDS of its own, one block ahead, and there is no barrier until the sums are
// added up through the LDS in a fixed order. The fewer rows and columns a workgroup has, the more workgroups read W at once: 16 x 16
// tiles are right for one row (1x4096x4096 4.2 us = 4.0 TB/s from the caches, 5.8 cold; 16 x 64 tiles 6.5), 16 x 64 for 64x4096x4096 (6.9 us; 16 x 16
// 9.7), 32 x 64 for 128x4096x4096 (8.0; 12.2 by 16 x 64), 64 x 64 for 512x4096x4096 (20; 26 by 32 x 64, 25 by 128 x 128 tiles).
template <int MF, int NF> struct Split {
    static constexpr int SCALES = MF == 4 ? 2 : 1;                                  // DMA instructions for a block's scales
    static constexpr int STAGE = (MF + NF) * 2048 + SCALES * 256, PER = (MF + NF) * 2 + SCALES;     // a block: bytes, DMA instructions
    static constexpr int WAVES = MF + NF == 2 ? 8 : 4;                              // at most
    static constexpr int BYTES = WAVES * 2 * STAGE;                                 // LDS, at most
    static_assert(BYTES <= 160 * 1024 && PER < 64, "split");
    // blocks for every wave: the same number, but for the last; 16 x 16 tiles are so little work that a wave takes two at least
    // (24x5000x1000 3.9 us, with one block each 4.4). No more LDS than there are blocks, so that more workgroups share a CU.
    static int rounds(int nkb) { return std::max((nkb + WAVES - 1) / WAVES, MF + NF == 2 ? std::min(2, nkb) : 1); }
    static int waves(int nkb) { return (nkb + rounds(nkb) - 1) / rounds(nkb); }
    static int depth(int nkb) { return rounds(nkb) > 1 ? 2 : 1; }
    static size_t bytes(int nkb) { return (size_t)waves(nkb) * std::max(depth(nkb) * STAGE, MF * NF * 1024); }
};
template <int MF, int NF, bool E8M0, typename T>
__global__ __launch_bounds__((Split<MF, NF>::WAVES * 64)) void matmul_split_kernel(MatmulP p) {
    constexpr bool WIDE = sizeof(T) == 4;
    constexpr int SB = E8M0 ? 1 : 4, SD = Split<MF, NF>::SCALES, STAGE = Split<MF, NF>::STAGE, PER = Split<MF, NF>::PER;
    const int NW = blockDim.x >> 6, D = p.depth;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15, q = lane >> 4;
    // an XCD takes neighbouring columns with all rows, or neighbouring rows with all columns, whichever there are more of: its L2 sees its
    // part of the longer operand once (with tiles dealt to the XCDs in turn 767x1945x3004 takes 46 us by 16 x 64, so 29)
    const bool tall = p.M > p.N;
    const int id = xcd_run(blockIdx.x, p.tiles_m * p.tiles_n), inner = tall ? p.tiles_n : p.tiles_m;
    const int outer_at = __builtin_amdgcn_readfirstlane(id / inner), inner_at = id - outer_at * inner;
    const int tm = tall ? outer_at : inner_at, tn = tall ? inner_at : outer_at;
    const int m0 = tm * (16 * MF), n0 = tn * (16 * NF);

    // DMA: instruction i of an operand covers its rows 8 i ... 8 i + 7
    const uint8_t *abase = uniform(p.a + (int64_t)m0 * p.lda), *wbase = uniform(p.w + (int64_t)n0 * p.ldw);
    uint32_t aoff[MF * 2], woff[NF * 2];
    int wchunk[NF * 2];
    const int achunk = ((lane & 7) ^ key_a(lane >> 3)) * 16, achunk8 = ((lane & 7) ^ key_a(8 + (lane >> 3))) * 16;
#pragma unroll
    for (int i = 0; i < MF * 2; ++i) aoff[i] = (uint32_t)min(i * 8 + (lane >> 3), p.M - 1 - m0) * (uint32_t)p.lda + (i & 1 ? achunk8 : achunk);
#pragma unroll
    for (int i = 0; i < NF * 2; ++i) {
        const int row = i * 8 + (lane >> 3);
        wchunk[i] = ((lane & 7) ^ (NF == 1 ? key_a(row) : key_w(row))) * 16;
        woff[i] = (uint32_t)min(row, p.N - 1 - n0) * (uint32_t)p.ldw + wchunk[i];
    }
    // scales: lane r takes A's of row r, the lane behind them (of an instruction of its own where there is none) W's
    const uint8_t *sap = (const uint8_t *)p.sa + (int64_t)min(m0 + min(lane, MF * 16 - 1), p.M - 1) * p.ldsa * SB;
    const uint8_t *swp = (const uint8_t *)p.sw + (int64_t)(n0 / kFp8Block) * p.ldsw * SB;
    const uint8_t *first = SD == 1 && lane == MF * 16 ? swp : sap;
    uint8_t *mine = lds + wave * (D * STAGE);
    auto fill = [&](int kb, int stage) {
        uint8_t *to = mine + stage * STAGE;
        const int k = kb * kFp8Block, at = E8M0 ? kb & ~3 : kb * 4;
#pragma unroll
        for (int i = 0; i < MF * 2; ++i) dma(abase, k + (i & 1 ? achunk8 : achunk) < p.K16 ? aoff[i] : kOutside, k, to + i * 1024);
#pragma unroll
        for (int i = 0; i < NF * 2; ++i) dma(wbase, k + wchunk[i] < p.K16 ? woff[i] : kOutside, k, to + (MF * 2 + i) * 1024);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(first + at), (__attribute__((address_space(3))) void *)(to + (MF + NF) * 2048), 4, 0, 0);
        if constexpr (SD == 2)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(swp + at), (__attribute__((address_space(3))) void *)(to + (MF + NF) * 2048 + 256), 4, 0, 0);
    };

    // a thread's columns on the way out: a piece of PF fragments; its bias is under way from here
    constexpr int PF = NF == 4 && !WIDE ? 2 : 1, PIECES = 4 * NF / PF;
    const int piece = threadIdx.x % PIECES, pq = piece / (NF / PF), pf = piece % (NF / PF) * PF, n = n0 + (pq * NF + pf) * 4;
    float bias[4 * PF];
    load_bias(p, n, bias);

    f32x4 acc[NF][MF] = {};
    const int blocks = wave < p.nkb ? (p.nkb - wave + NW - 1) / NW : 0;
    for (int d = 0; d < min(D, blocks); ++d) fill(wave + d * NW, d);        // (one block if D = 1)
    const int wrow = NF == 1 ? i16 : (i16 >> 2) * 16 + (i16 & 3), wkey = NF == 1 ? key_a(wrow) : key_w(wrow);
    for (int t = 0, stage = 0; t < blocks; ++t) {
        if (D > 1 && t + 1 < blocks) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");        // (the next block may be under way)
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const int kb = wave + t * NW;
        const uint8_t *st = mine + stage * STAGE, *sc = st + (MF + NF) * 2048 + (E8M0 ? kb & 3 : 0);
        auto scale = [&](int row) {
            if constexpr (E8M0) return (uint32_t)sc[row * 4];
            else return *(const uint32_t *)(sc + row * 4);
        };
        Raw wv[NF], av[MF];
        uint32_t as[MF];
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const uint8_t *r = st + MF * 2048 + (wrow + f * 4) * kFp8Block;
            wv[f] = Raw{*(const i32x4 *)(r + ((q ^ wkey) * 16)), *(const i32x4 *)(r + (((q + 4) ^ wkey) * 16))};
        }
#pragma unroll
        for (int j = 0; j < MF; ++j) {
            const uint8_t *r = st + (j * 16 + i16) * kFp8Block;
            av[j] = Raw{*(const i32x4 *)(r + ((q ^ key_a(i16)) * 16)), *(const i32x4 *)(r + (((q + 4) ^ key_a(i16)) * 16))};
            as[j] = scale(j * 16 + i16);
        }
        const uint32_t ws = scale(MF * 16);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // in registers: the stage may be filled again
        if (t + D < blocks) fill(kb + D * NW, stage);
        stage = D - 1 - stage;
        Frag<WIDE> wf[NF], af;
#pragma unroll
        for (int f = 0; f < NF; ++f) wf[f].set(wv[f].lo, wv[f].hi);
#pragma unroll
        for (int j = 0; j < MF; ++j) {
            af.set(av[j].lo, av[j].hi);
#pragma unroll
            for (int f = 0; f < NF; ++f) mma<E8M0, WIDE>(wf[f], af, acc[f][j], scale_of<E8M0, WIDE>(ws), scale_of<E8M0, WIDE>(as[j]));
        }
    }
    __syncthreads();                                               // (every wave's fills have landed and been read)
    // [wave][column fragment][row fragment][lane]; the order of the lanes that share q spreads a row's pieces over the banks
    f32x4 *red = (f32x4 *)lds;
    auto at = [&](int f, int j, int fq, int row) { return (f * MF + j) * 64 + ((fq * 16 + row) ^ (((fq + f) & 3) * 4)); };
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int j = 0; j < MF; ++j) red[wave * (NF * MF * 64) + at(f, j, q, i16)] = acc[f][j];
    __syncthreads();
    if (n >= p.N) return;
    // out in 16-byte pieces, neighbouring threads along a row
#pragma unroll 1
    for (int row = threadIdx.x / PIECES; row < min(MF * 16, p.M - m0); row += NW * (64 / PIECES)) {
        float v[4 * PF];
        f32x4 s[PF] = {};
#pragma unroll 4
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int f = 0; f < PF; ++f) s[f] += red[w * (NF * MF * 64) + at(pf + f, row >> 4, pq, row & 15)];
#pragma unroll
        for (int c = 0; c < 4 * PF; ++c) v[c] = s[c >> 2][c & 3] + bias[c];
        T *dst = (T *)p.y + (int64_t)(m0 + row) * p.ldy + n;
        const T *res = p.res ? (const T *)p.res + (int64_t)(m0 + row) * p.ldres + n : nullptr;
        if (n0 + 16 * NF <= p.N) store_cols<true, T, 4 * PF>(p.act, dst, res, 4 * PF, v);        // (the workgroup agrees)
        else store_cols<false, T, 4 * PF>(p.act, dst, res, p.N - n, v);
    }
}

// ---- tiles --------------------------------------------------------------------------------------------------------------------------
// BM x BN of y per workgroup, WM x WN per wave. K's blocks pass through two LDS stages of (BM + BN) x 128 bytes, filled by LDS-DMA
// (16 bytes a lane, no registers).
//
// The matrix units are the bound, so they must not see the LDS: a wave multiplies the fragments of A one after the other against its FN
// fragments of W and reads PD fragments ahead, over the end of the block too. The one barrier of a block stands PD fragments before its
// end: there every wave has all of this block in registers and its part of the next one has landed; behind it the stage just read
// is filled with the block after the next, a quarter of the instructions with each of the next four fragments. (All at once they fill the
// address unit's queue, and the waves stand in front of it with the matrix units idle: 0.5 us of a block's 1.8 at 256 x 256.)
// 8192^3 bf16 by 256 x 256: 400 - 446 us, 2.5 - 2.75 PFLOP/s (library 426 us); a block of K takes 1.03 us on one CU alone and 1.4 with all at work.
// 4000x2500x4096: 192 x 256 (210 tiles) 46 us, 256 x 256 (160 tiles) 54, 128 x 128 60; with fp32 scales 52, 61, 70.
struct RawA {
    i32x4 lo, hi;
    uint32_t scale;
};
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
    // an XCD walks its run of tiles in bands of 8 tile rows, so that its L2 sees the same operands again
    const int id = xcd_run(blockIdx.x, p.tiles_m * p.tiles_n);
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
    auto fill = [&](int kb, int from, int to) {                // DMA instructions from ... to - 1 of a block's
        const int k = min(kb, p.nkb - 1) * kFp8Block, at = (kb & 1) * STAGE + wave * 1024;
#pragma unroll
        for (int i = 0; i < PA + PW; ++i) {
            if (i < from || i >= to) continue;
            if (i < PA) dma(abase, k + achunk < p.K16 ? aoff[i] : kOutside, k, lds + at + i * STEP * kFp8Block);
            else dma(wbase, k + wchunk[i - PA] < p.K16 ? woff[i - PA] : kOutside, k, lds + at + (BM + (i - PA) * STEP) * kFp8Block);
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
    // one block of K; S = kb % 4. No branches inside: the compiler would gather the products behind them. (Behind the last block the look-ahead
    // loads that block again; its fragments are read and never multiplied. Such loads are still on their way into the LDS when the loop ends: the
    // wait and the barrier before the epilogue are what lets it use that memory.)
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

template <int MF, int NF, bool E8M0, typename T> static int launch_split(MatmulP p, hipStream_t s) {
    using Form = Split<MF, NF>;
    p.tiles_m = (p.M + 16 * MF - 1) / (16 * MF);
    p.tiles_n = (p.N + 16 * NF - 1) / (16 * NF);
    const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
    LSSVC_CHECK(fits_launch(total, Form::waves(p.nkb) * 64), "matmul_fp8: %lld tiles do not fit one launch", (long long)total);
    p.depth = Form::depth(p.nkb);
    static LdsGrant grant;
    if (int rc = grant.ensure((const void *)matmul_split_kernel<MF, NF, E8M0, T>, Form::BYTES, 64 * 1024)) return rc;
    matmul_split_kernel<MF, NF, E8M0, T><<<(unsigned)total, Form::waves(p.nkb) * 64, Form::bytes(p.nkb), s>>>(p);
    return launch_status("matmul_fp8");
}

template <int BM, int BN, int WM, int WN, bool E8M0, typename T> static int launch_tile(MatmulP p, hipStream_t s) {
    static LdsGrant grant;
    constexpr size_t bytes = 2 * (BM + BN) * kFp8Block + 2 * BM * (E8M0 ? 4 : 16);
    if (int rc = grant.ensure((const void *)matmul_tile_kernel<BM, BN, WM, WN, E8M0, T>, bytes, 64 * 1024)) return rc;
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
    LSSVC_CHECK(fits_launch(total, (BM / WM) * (BN / WN) * 64), "matmul_fp8: %lld tiles do not fit one launch", (long long)total);
    matmul_tile_kernel<BM, BN, WM, WN, E8M0, T><<<(unsigned)total, (BM / WM) * (BN / WN) * 64, bytes, s>>>(p);
    return launch_status("matmul_fp8");
}

// Which form: the one with the least estimated time, in us, fitted to times measured at 72 sizes (1 x 4096 x 4096 ... 8192^3 and random ones,
// 16-bit and fp32 results, both kinds of scales); the form so chosen takes 0.5 % more than the fastest one in the geometric mean. Split: a start,
// and for every tile that a CU gets what it reads and an end; where only one workgroup fits a CU, whole rounds of them. Tiles: the
// same with whole rounds, since a 256 x 256 form's half-empty last round is what the smaller tiles' lower rate is weighed against.
constexpr int kTile[7][2] = {{16, 16}, {16, 64}, {32, 64}, {64, 64}, {128, 128}, {256, 256}, {192, 256}};      // rows and columns of y per workgroup; 0 - 3: split
static int choose(const MatmulP &p, bool e8m0) {
    const bool wide = p.dtype == LSSVC_F32;
    auto tiles = [&](int i) { return (double)((p.M + kTile[i][0] - 1) / kTile[i][0]) * (double)((p.N + kTile[i][1] - 1) / kTile[i][1]); };
    auto split = [&](auto form, int i, double start, double read, double widen, double end) {
        using Form = decltype(form);
        const double t = tiles(i) / 256, x = 2 * Form::bytes(p.nkb) > 160 * 1024 ? std::ceil(t) : std::max(1.0, t);
        return start + x * (p.nkb * ((kTile[i][0] + kTile[i][1]) / 16) * read * (wide ? widen : 1.0) + end);
    };
    auto tiled = [&](int i, double start, double block, double end) { return start + std::ceil(tiles(i) / 256) * (p.nkb * block + end); };
    // (a pitch that is no multiple of 128: a block of K straddles two lines)
    const double pitch = (p.lda | p.ldw) % 128 && p.nkb > 1 ? 1.6 : 1.0, rate = (e8m0 ? 1.0 : 1.17) * pitch, small_rate = (wide ? 2.2 : e8m0 ? 1.0 : 1.2) * pitch;
    const double cost[7] = {split(Split<1, 1>{}, 0, 2.8, 0.028, 1.25, 0.07), split(Split<1, 4>{}, 1, 3.1, 0.028, 1.38, 0.18),
                            split(Split<2, 4>{}, 2, 2.9, 0.029, 1.55, 0.9), split(Split<4, 4>{}, 3, 2.6, 0.03, 1.65, 2.4),
                            tiled(4, 4.3, 0.5 * small_rate, 2.5), wide ? 1e30 : tiled(5, 7.0, 1.38 * rate, 5.0),
                            wide ? 1e30 : tiled(6, 6.5, 1.1 * rate, 4.0)};
    return (int)(std::min_element(cost, cost + 7) - cost);
}
template <bool E8M0, typename T> static int launch_matmul(const MatmulP &p, hipStream_t s) {
    constexpr bool WIDE = sizeof(T) == 4;
    switch (choose(p, E8M0)) {
        case 0: return launch_split<1, 1, E8M0, T>(p, s);
        case 1: return launch_split<1, 4, E8M0, T>(p, s);
        case 2: return launch_split<2, 4, E8M0, T>(p, s);
        case 3: return launch_split<4, 4, E8M0, T>(p, s);
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
static int operands_check(const lssvc_fp8 *a, const lssvc_fp8 *w) {
    if (int rc = operand_check(a, "a", 1)) return rc;
    if (int rc = operand_check(w, "w", kFp8Block)) return rc;
    LSSVC_CHECK(w->rows > 0, "matmul_fp8: w has no rows");
    LSSVC_CHECK(a->cols == w->cols, "matmul_fp8: a has %d columns, w has %d", a->cols, w->cols);
    LSSVC_CHECK((a->scale_e8m0 != 0) == (w->scale_e8m0 != 0), "matmul_fp8: one operand has e8m0 scales, the other fp32 scales");
    return 0;
}
static MatmulP operands_of(const lssvc_fp8 *a, const lssvc_fp8 *w, int dtype) {
    MatmulP p{};
    p.a = (const uint8_t *)a->values, p.w = (const uint8_t *)w->values;
    p.sa = a->scale, p.sw = w->scale;
    p.lda = a->ld, p.ldw = w->ld, p.ldsa = a->scale_ld, p.ldsw = w->scale_ld;
    p.M = (int)a->rows, p.N = (int)w->rows, p.K16 = (a->cols + 15) / 16 * 16, p.nkb = (a->cols + kFp8Block - 1) / kFp8Block;
    p.dtype = dtype;
    return p;
}

}  // namespace lssvc

using namespace lssvc;

extern "C" int lssvc_matmul_fp8_tile(const lssvc_fp8 *a, const lssvc_fp8 *w, int32_t dtype, int32_t *rows, int32_t *cols) {
    if (int rc = operands_check(a, w)) return rc;
    LSSVC_CHECK(rows_type_ok(dtype) && rows && cols, "matmul_fp8_tile: unknown result type %d, or nowhere to put the tile", dtype);
    const int form = choose(operands_of(a, w, dtype), a->scale_e8m0 != 0);
    *rows = kTile[form][0], *cols = kTile[form][1];
    return 0;
}

extern "C" int lssvc_matmul_fp8(const lssvc_fp8 *a, const lssvc_fp8 *w, const float *bias, int32_t act, float slope, const lssvc_rows *residual,
                                const lssvc_rows *y, void *stream) {
    if (int rc = operands_check(a, w)) return rc;
    LSSVC_CHECK(act_ok(act), "matmul_fp8: unknown activation %d", act);
    if (int rc = rows_check("matmul_fp8", y)) return rc;
    LSSVC_CHECK(y->rows == a->rows && y->cols == w->rows, "matmul_fp8: the output is not %lld x %lld", (long long)a->rows, (long long)w->rows);
    if (residual) {
        if (int rc = rows_check("matmul_fp8", residual)) return rc;
        LSSVC_CHECK(residual->rows == y->rows && residual->cols == y->cols && residual->dtype == y->dtype, "matmul_fp8: the residual's shape or type is not the output's");
    }
    if (a->rows == 0) return 0;
    LSSVC_CHECK(!residual || rows_disjoint_or_same(residual, y), "matmul_fp8: residual and output overlap in part");
    LSSVC_CHECK(apart({span_of(y)}, {values_of(a), scales_of(a), values_of(w), scales_of(w), span_of(bias, w->rows)}), "matmul_fp8: the output overlaps an operand or the bias");
    MatmulP p = operands_of(a, w, y->dtype);
    p.bias = bias;
    p.res = residual ? residual->ptr : nullptr, p.ldres = residual ? residual->ld : 0;
    p.y = y->ptr, p.ldy = y->ld;
    p.act = Act{act, slope};
    return a->scale_e8m0 ? launch_typed<true>(p, (hipStream_t)stream) : launch_typed<false>(p, (hipStream_t)stream);
}
