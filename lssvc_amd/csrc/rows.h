// Shared device helpers of the row operators (group norm, block quantiser, 8-bit product): typed rows, activations, 8-bit encoding.
#pragma once
#include <initializer_list>
#include "common.h"

namespace lssvc {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kFp8Block = 128;   // columns that share a scale

inline bool rows_type_ok(int t) { return t == LSSVC_F32 || t == LSSVC_F16 || t == LSSVC_BF16; }
inline int rows_type_size(int t) { return t == LSSVC_F32 ? 4 : 2; }
inline bool act_ok(int a) { return a >= LSSVC_ACT_NONE && a <= LSSVC_ACT_SILU; }
inline bool aligned(const void *p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Two row matrices either share no byte, or are the very same one: a channel slice beside another slice of the same wide buffer
// overlaps as an address range and is fine; anything in between would be read after it was written.
inline bool rows_disjoint_or_same(const lssvc_rows *a, const lssvc_rows *b) {
    const int sa = rows_type_size(a->dtype), sb = rows_type_size(b->dtype);
    const uintptr_t pa = (uintptr_t)a->ptr, pb = (uintptr_t)b->ptr;
    const uint64_t wa = (uint64_t)a->cols * sa, wb = (uint64_t)b->cols * sb, la = (uint64_t)a->ld * sa, lb = (uint64_t)b->ld * sb;
    const uintptr_t ea = pa + (uint64_t)(a->rows - 1) * la + wa, eb = pb + (uint64_t)(b->rows - 1) * lb + wb;
    if (ea <= pb || eb <= pa) return true;
    if (la != lb) return false;
    if (pa == pb) return a->dtype == b->dtype;
    const uint64_t d = pb > pa ? (pb - pa) % la : (la - (pa - pb) % la) % la;       // where b's columns start within a's pitch
    return d >= wa && d + wb <= la;
}

// A range of bytes that a call reads or writes. What it writes shares no byte with what it reads.
struct Span {
    uintptr_t at;
    uint64_t bytes;
    bool apart(const Span &o) const { return !bytes || !o.bytes || at + bytes <= o.at || o.at + o.bytes <= at; }
};
inline Span span_of(const lssvc_rows *x) {
    const int es = rows_type_size(x->dtype);
    return {(uintptr_t)x->ptr, x->rows ? ((uint64_t)(x->rows - 1) * (uint64_t)x->ld + x->cols) * es : 0};
}
inline Span span_of(const float *v, int64_t n) { return {(uintptr_t)v, v ? (uint64_t)n * 4 : 0}; }
inline Span values_of(const lssvc_fp8 *x) {
    return {(uintptr_t)x->values, x->rows ? (uint64_t)(x->rows - 1) * (uint64_t)x->ld + (x->cols + 15) / 16 * 16 : 0};
}
inline Span scales_of(const lssvc_fp8 *x) {
    const int64_t kb = (x->cols + kFp8Block - 1) / kFp8Block, blocks = x->rows ? (x->rows - 1) / x->block_rows : 0;
    return {(uintptr_t)x->scale, x->rows ? ((uint64_t)blocks * (uint64_t)x->scale_ld + kb) * (x->scale_e8m0 ? 1 : 4) : 0};
}
inline bool apart(std::initializer_list<Span> written, std::initializer_list<Span> read) {
    for (const Span *w = written.begin(); w != written.end(); ++w) {
        for (const Span &r : read)
            if (!w->apart(r)) return false;
        for (const Span *o = w + 1; o != written.end(); ++o)
            if (!w->apart(*o)) return false;
    }
    return true;
}
// The runtime counts a launch's threads in 32 bits
inline bool fits_launch(int64_t workgroups, int threads) { return workgroups < (1LL << 31) && workgroups * threads < (1LL << 32); }

int rows_check(const char *what, const lssvc_rows *x);                                       // row_norm.hip
int fp8_out_check(const char *what, const lssvc_fp8 *y, int64_t rows, int cols);

// ---- typed values: every kernel computes in fp32; storing to 16 bits is the one rounding (to nearest even) ----------------------
struct bf16_t { uint16_t v; };
struct f16_t { _Float16 v; };
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(f16_t x) { return (float)x.v; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __uint_as_float((uint32_t)x.v << 16); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float x) { return f16_t{(_Float16)x}; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) {
    const __bf16 b = (__bf16)x;
    return bf16_t{__builtin_bit_cast(uint16_t, b)};
}

// N consecutive values as they lie in memory, at the type's own alignment: global loads and stores of any width need no more on
// gfx950, so slices and odd pitches take the wide path too.
template <typename T, int N> struct Pack { T v[N]; };
template <int BYTES> struct Words;                              // the widest pieces of BYTES, as a vector of 2-byte alignment
template <> struct Words<2> { typedef uint16_t type; };
template <> struct Words<4> { typedef uint32_t type __attribute__((aligned(2))); };
template <> struct Words<8> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Words<16> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <int BYTES> constexpr int kPiece = BYTES > 16 ? 16 : BYTES;
template <typename T, int N> __device__ __forceinline__ Pack<T, N> load_pack(const T *p) {
    using W = typename Words<kPiece<sizeof(Pack<T, N>)>>::type;
    constexpr int Q = sizeof(Pack<T, N>) / sizeof(W);
    W w[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) w[i] = ((const W *)p)[i];
    Pack<T, N> r;
    __builtin_memcpy(&r, w, sizeof(r));
    return r;
}
template <typename T, int N> __device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &r) {
    using W = typename Words<kPiece<sizeof(Pack<T, N>)>>::type;
    constexpr int Q = sizeof(Pack<T, N>) / sizeof(W);
    W w[Q];
    __builtin_memcpy(w, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < Q; ++i) ((W *)p)[i] = w[i];
}

// Activations, for N values at a time so that the choice is made once. silu: exp and reciprocal at the hardware's 1 ulp, and exp's argument is
// rounded, up to 1.23 |v| half steps: relative to the result 2^-23.5 around 0, 2^-21 at -10, 2^-19 at -40, 2^-18 at -80 (measured). Below -87.3, where the
// reciprocal leaves the normal numbers, it is 0 for less than 1.1e-36. An exact argument would cost 4 instructions a value, and the pass into
// 8 bits is bound by them. NaN passes through all of them.
struct Act {
    int kind;
    float slope;
};
template <int N> __device__ __forceinline__ void apply_act(float (&v)[N], const Act &a) {
    if (a.kind == LSSVC_ACT_NONE) return;
    if (a.kind == LSSVC_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] * __builtin_amdgcn_rcpf(1.f + __expf(-v[i]));
    } else if (a.kind == LSSVC_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? v[i] * a.slope : v[i];
    }
}

// ---- 8-bit blocks ---------------------------------------------------------------------------------------------------------------
// max over the 16 lanes of a DPP row; every lane gets it
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));   // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));
}
// The largest |x| among 8 values per lane of the finite ones, over the 16 lanes of a DPP row, as ordered bits. The plain maximum first: only
// where it is not finite are such values left out one by one.
__device__ __forceinline__ uint32_t row16_finite_max(const float (&z)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(z[j]) & 0x7fffffffu);
    m = row16_max(m);
    if (m >= 0x7f800000u) {                  // (the 16 lanes agree)
        m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t b = __float_as_uint(z[j]) & 0x7fffffffu;
            m = max(m, b < 0x7f800000u ? b : 0u);
        }
        m = row16_max(m);
    }
    return m;
}
// sum over the wave in a fixed order, valid in lane 63
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_move(double v) {      // lanes that get nothing get 0
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_hi(double v) {
    v += dpp_move<0x111, 0xf>(v);            // row_shr:1, 2, 4, 8: lane 15 of each row has the row's sum
    v += dpp_move<0x112, 0xf>(v);
    v += dpp_move<0x114, 0xf>(v);
    v += dpp_move<0x118, 0xf>(v);
    v += dpp_move<0x142, 0xa>(v);            // row_bcast:15 into rows 1 and 3
    v += dpp_move<0x143, 0xc>(v);            // row_bcast:31 into rows 2 and 3
    return v;
}
// t / n for t < 2^16 and n < 2^16: one multiplication; magic = division_magic(n)
__host__ __device__ __forceinline__ uint32_t division_magic(uint32_t n) { return n > 1 ? 0xffffffffu / n + 1 : 0; }
__device__ __forceinline__ int divided(int t, uint32_t magic) { return magic ? (int)__umulhi((uint32_t)t, magic) : t; }

// The exponent byte of the smallest power of two s >= 2^-126 with amax <= 448 s (1 where amax = 0). amax = m 2^k with m in [0.5, 1)
// and 448 = 0.875 * 2^9, so s = 2^(k - 9) where m <= 0.875 and 2^(k - 8) otherwise; k = field - 126.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax_bits) {
    if (amax_bits == 0u) return 127u;
    const int field = (int)(amax_bits >> 23), e = field - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)(e < 1 ? 1 : e);
}
__device__ __forceinline__ float scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }   // 2^-(byte - 127), byte <= 247: exact
// four values that lie within +-448 (or are not finite: NaN) to e4m3, to nearest even
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

}  // namespace lssvc
