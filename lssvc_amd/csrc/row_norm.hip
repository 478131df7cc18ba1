// row_norm.hip -- group norm with an activation over channels-last rows, optionally straight into 8-bit blocks.
//
// y = act((x - mu) * rsqrt(var + eps) * w_c + b_c), mu / var over the rows of an image and the cg = C / G channels of a group. The
// operator is bound by memory: one read and one write of the map if it stays on the chip between the statistics and their use, two reads
// otherwise. Two forms:
//   resident  a workgroup owns all rows of a slice of whole groups and holds the slice in the LDS (up to 159 KB; every thread reads back
//             what it wrote itself): one read, one write, one launch.
//   split     rows are split over workgroups that write sums per chunk and group; the chunks are joined by a launch of their own, or, where
//             they are few, by every workgroup of the normalising pass for itself; that pass reads the map again, in the opposite order,
//             so that what the first pass read last comes from the caches.
// Measured: 18x30x64 fp32 4.2 us (resident); 1152x1920x48 fp32 266 us = 113 (3.8 TB/s, what a read-only
// pass reaches) + 5 + 148 (5.7 TB/s); 34560x256 bf16 to 8 bits 7.5 + 3.5 + 10.7 us, of which the activation and the encoding are half.
// Sums S1 = sum x and S2 = sum x^2 are in 64 bits from the first value on: squares of fp32 and bf16 values leave fp32's range (from 1.8e19 and
// below 1e-19 on), and S2 - S1^2 / N keeps what fp32 data can hold: an offset a thousand times the spread costs 2^-33 of the variance. That
// is a conversion, an addition and an FMA a value: nothing beside HBM (1152x1920x48 fp32), 2 - 4 % of 16-bit maps in the caches (34560x256 bf16 18.1 -> 18.4 us,
// 8640x512 14.4 -> 15.0, against per-thread sums of differences in fp32). The mean is held as two fp32 numbers, the second folded
// into the shift, so an offset costs no digits of the result.
//
// One thread handles V consecutive channels: 16 bytes at any alignment (8 channels where 8-bit blocks are written). Where V does not divide
// the slice, a row's last thread loads the LAST V channels -- wide loads only -- and owns those that its neighbour does not (a slice of fewer
// than V channels takes V = 1). An integer division costs about 40 instructions: a thread's place and its first group come from one
// multiplication each.
#include <algorithm>
#include <type_traits>
#include "rows.h"

namespace lssvc {

struct NormP {
    const void *x;
    void *y;                     // T rows (to_fp8: unused)
    uint8_t *q, *qs;             // 8-bit values and scale bytes (to_fp8)
    int64_t ldx, ldy, ldq, ldqs;
    int64_t R;                   // rows of an image
    const float *w, *b;
    double2 *part;               // split form: [image][unit][chunk] (S1, S2): whole lines for those who add a unit up
    float *mean, *scale, *shift; // split form without join: [image][channel] mean, weight / sqrt(var + eps), bias less the mean's second part
    int64_t chunk;               // rows of a chunk
    int C, G, cg;
    int S;                       // chunks of an image
    int P, piece;                // pieces of a group: 1, or `piece` columns each where a group is wider than a workgroup takes
    int slice, nslices;          // columns of a slice (P = 1), slices of a row
    Act act;
    float eps;
    int in_place;                // y is x: a row's last thread stores its own channels only
    int parts;                   // resident form: workgroups that share a slice's rows on the way out
    int nv;                      // threads of a row of a full slice; multiplications that divide by it, by a unit's width and by its share of a row
    uint32_t m_nv, m_uw, m_w;
};

constexpr int kSliceMax = 1024;  // columns of a slice in the split form: 256 threads x 4; 256 where V = 1
template <typename T> constexpr int kVecOf = 16 / (int)sizeof(T);

// a thread's V channels of a slice that is `sc` columns wide
template <int V> struct Lane {
    int cv, rt;        // which V channels, which of the rows in flight
    int lo;            // first channel that is loaded
    int own;           // loaded channels from `own` on are this thread's (below `end`)
    int end;
    bool live;
    __device__ __forceinline__ Lane(int t, int nv, uint32_t m_nv, int rp, int sc) {
        rt = divided(t, m_nv);
        cv = t - rt * nv;
        live = rt < rp;
        const int c0 = cv * V;
        lo = sc >= V ? min(c0, sc - V) : 0;
        own = c0 - lo;
        end = sc >= V ? V : sc;
        if (c0 >= sc) own = end = 0, lo = 0;         // padding lane of the 8-bit form: owns nothing
    }
    __device__ __forceinline__ bool owns(int j) const { return j >= own && j < end; }
    // the unit (group, or piece) of each channel: units are `uw` wide and start at the slice's first column
    template <bool ALIKE> __device__ __forceinline__ void units(int uw, uint32_t m_uw, int nu, int (&un)[V]) const {
        int u = divided(lo, m_uw), c = lo - u * uw;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            un[j] = min(u, nu - 1);
            if (!ALIKE && ++c == uw) c = 0, ++u;
        }
    }
};

// quotients of uniform values, once per workgroup
__device__ __forceinline__ int divided_any(int a, int b) { return (int)((unsigned)a / (unsigned)b); }

// threads of a row that is `sc` columns wide (the 8-bit form: 16 for every block of 128)
template <int V, bool TO8> __host__ __device__ __forceinline__ int threads_of(int sc) {
    return TO8 ? (sc + kFp8Block - 1) / kFp8Block * (kFp8Block / 8) : (sc + V - 1) / V;
}

template <typename T, int V, bool NARROW = false> __device__ __forceinline__ Pack<T, V> load_lane(const T *row, const Lane<V> &l) {
    if (!NARROW || l.end == V) return load_pack<T, V>(row + l.lo);
    Pack<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = j < l.end ? row[l.lo + j] : from_f32<T>(0.f);
    return r;
}

// (S1, S2) of every unit of a slice from the threads' sums: entries go to the LDS, a unit's are added up by 2^sh lanes (of several waves where
// there are fewer units than waves) in a fixed order, and one lane hands the totals on. What a thread enters:
//   ONE   V divides the unit width: its V channels lie in one unit, one pair
//   TWO   they lie in two units at most: a pair for each
//   EACH  narrow units: a pair for every channel
//   TURNS the same in half the LDS, for a map that needs the rest: S1 first and S2 after it, unit u's totals by the same lane (2160x12 fp16 in
//         12 groups 8.6 us, by EACH 7.1; 3x1961x100 fp16 9.5, by TWO 8.0)
enum Sums { ONE, TWO, EACH, TURNS };
__host__ __device__ constexpr Sums sums_of(int uw, int V) { return uw % V == 0 ? ONE : uw >= V - 1 || 2 * uw == V ? TWO : EACH; }
__host__ __device__ constexpr int entries_of(Sums how, int uw, int V) { return how == ONE ? uw / V : how == TWO ? (uw + V - 2) / V + 1 : uw; }   // of a unit in a row, at most
// 64-bit sums that a thread keeps: one for each channel; where all of them lie in one unit, enough that an addition need not wait for the one before
template <int V, Sums HOW> constexpr int kChains = HOW == ONE && V > 2 ? 2 : V;
constexpr int entry_bytes(int threads, Sums how, int V) { return threads * (how == ONE ? 16 : how == TWO ? 32 : how == EACH ? 16 * V : 8 * V); }
__device__ __forceinline__ double2 operator+(const double2 &a, const double2 &b) { return make_double2(a.x + b.x, a.y + b.y); }
__device__ __forceinline__ double wave_total(double a) { return wave_sum_hi(a); }
__device__ __forceinline__ double2 wave_total(const double2 &a) { return make_double2(wave_sum_hi(a.x), wave_sum_hi(a.y)); }
__device__ __forceinline__ double from_lane(double a, int o) { return __shfl_xor(a, o); }
__device__ __forceinline__ double2 from_lane(const double2 &a, int o) { return make_double2(__shfl_xor(a.x, o), __shfl_xor(a.y, o)); }
// `entry(u, r, c)`: the c-th of W of unit u in row r
template <int TPB, typename E, typename G, typename F> __device__ __forceinline__ void add_up(int W, uint32_t m_w, int rows, int nu, G entry, F done) {
    __shared__ E wsum[TPB / 64];
    const int t = threadIdx.x;
    int sh = TPB == 512 ? 9 : 8;
    while (sh > 0 && (nu << sh) > TPB) --sh;
    const int lpu = 1 << sh, li = t & (lpu - 1);
    const int dr = divided(lpu, m_w), dc = lpu - dr * W;
    const int r0 = divided(li, m_w), c0 = li - r0 * W;
    for (int u = t >> sh; u < nu; u += TPB >> sh) {
        E a{};
        int r = r0, c = c0;
#pragma unroll 2
        while (r < rows) {
            a = a + entry(u, r, c);
            r += dr;
            c += dc;
            if (c >= W) c -= W, ++r;
        }
        if (sh >= 6) {
            a = wave_total(a);
            if ((t & 63) == 63) {
                if (sh == 6) done(u, a);
                else wsum[t >> 6] = a;
            }
        } else {
            for (int o = lpu >> 1; o > 0; o >>= 1) a = a + from_lane(a, o);
            if (li == 0) done(u, a);
        }
    }
    if (sh > 6) {                                              // (then there are at most TPB / 128 units)
        __syncthreads();
        if (t < nu) {
            E a{};
            for (int w = 0; w < 1 << (sh - 6); ++w) a = a + wsum[(t << (sh - 6)) + w];
            done(t, a);
        }
    }
}
// `hold(u)` (TURNS only): where S1 of a unit waits for S2, 8 bytes, the lane's own until then. `rows`: rows in flight that hold anything
template <int TPB, int V, Sums HOW, typename H, typename F>
__device__ __forceinline__ void unit_sums(const double (&s1)[kChains<V, HOW>], const double (&s2)[kChains<V, HOW>], int rows, const Lane<V> &l, int nv, int sc, int uw, uint32_t m_uw, uint32_t m_w,
                                          int nu, void *entries, H hold, F done) {
    const int W = entries_of(HOW, uw, V);
    if constexpr (HOW == TURNS) {
        double *e = (double *)entries;
        auto put = [&](const double (&v)[V]) {
            if (l.live)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (l.owns(j)) e[l.rt * sc + l.lo + j] = v[j];
            __syncthreads();
        };
        auto entry = [&](int u, int r, int c) { return e[r * sc + u * W + c]; };
        put(s1);
        add_up<TPB, double>(W, m_w, rows, nu, entry, [&](int u, double a) { *hold(u) = a; });
        __syncthreads();
        put(s2);
        add_up<TPB, double>(W, m_w, rows, nu, entry, [&](int u, double b) { done(u, *hold(u), b); });
    } else {
        double2 *e = (double2 *)entries;
        if constexpr (HOW == EACH) {
            if (l.live)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (l.owns(j)) e[l.rt * sc + l.lo + j] = make_double2(s1[j], s2[j]);
        } else if (l.live) {
            const int c0 = l.cv * V, next = HOW == ONE ? V : (divided(c0, m_uw) + 1) * uw - l.lo;       // the first channel of the second unit
            double2 a{}, b{};
#pragma unroll
            for (int j = 0; j < kChains<V, HOW>; ++j)
                if (HOW == ONE || l.owns(j)) {
                    const double2 v = make_double2(s1[j], s2[j]);
                    if (HOW == ONE || j < next) a = a + v;
                    else b = b + v;
                }
            e[l.rt * nv + l.cv] = a;
            if constexpr (HOW == TWO) e[TPB + l.rt * nv + l.cv] = b;
        }
        __syncthreads();
        add_up<TPB, double2>(W, m_w, rows, nu, [&](int u, int r, int c) {
            if constexpr (HOW == ONE) return e[r * nv + u * W + c];
            else if constexpr (HOW == EACH) return e[r * sc + u * W + c];
            else {                                             // the unit's threads; it is the first one's second unit if that one starts before it
                const int from = u * uw / V, cv = from + c;
                return cv * V < (u + 1) * uw && cv < nv ? e[(c == 0 && from * V < u * uw ? TPB : 0) + r * nv + cv] : double2{};
            }
        }, [&](int u, const double2 &a) { done(u, a.x, a.y); });
    }
}
struct __attribute__((aligned(16))) Moments {
    float mean, rstd, low;                                    // mean + low: the mean
};
__device__ __forceinline__ Moments moments(double s1, double s2, double n, float eps) {       // (one rounding each; NaN stays NaN)
    const double mean = s1 / n, var = s2 / n - mean * mean;
    const float hi = (float)mean;
    return Moments{hi, (float)(1.0 / sqrt((var < 0 ? 0.0 : var) + eps)), (float)(mean - hi)};
}

// ---- split form, first pass: (S1, S2) of each chunk and unit -----------------------------------------------------------------------
template <typename T, int V, Sums HOW>
__global__ __launch_bounds__(256) void norm_stats_kernel(NormP p) {
    constexpr int TPB = 256, NB = 4;
    __shared__ __attribute__((aligned(16))) uint8_t entries[entry_bytes(TPB, HOW, V)];
    unsigned id = blockIdx.x;
    const int sl = id % (unsigned)p.nslices;
    id /= (unsigned)p.nslices;
    const int chunk = id % (unsigned)p.S, img = id / (unsigned)p.S;
    int s0, sc, nu, uw;
    if (p.P == 1) {
        s0 = sl * p.slice;
        sc = min(p.slice, p.C - s0);
        uw = p.cg;
        nu = divided(sc, p.m_uw);
    } else {
        const int g = sl / p.P, k = sl - g * p.P;
        s0 = g * p.cg + k * p.piece;
        sc = uw = min(p.piece, p.cg - k * p.piece);
        nu = 1;
    }
    int nv = p.nv;
    uint32_t m_nv = p.m_nv, m_w = p.m_w;
    if (sc != p.slice) {                                       // the last slice; the last piece of a group
        nv = (sc + V - 1) / V, m_nv = division_magic(nv);
        if (p.P > 1) m_w = division_magic(entries_of(HOW, uw, V));
    }
    const int rp = divided(TPB, m_nv), t = threadIdx.x;
    const Lane<V> l(t, nv, m_nv, rp, sc);
    const int64_t r0 = chunk * p.chunk, r1 = min(r0 + p.chunk, p.R);
    const T *base = (const T *)p.x + ((int64_t)img * p.R + r0) * p.ldx + s0;
    const int rows = (int)(r1 - r0);

    constexpr int CH = kChains<V, HOW>;
    double s1[CH] = {}, s2[CH] = {};
    auto add = [&](const Pack<T, V> &e) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const double x = to_f32(e.v[j]);
            s1[j % CH] += x;
            s2[j % CH] = fma(x, x, s2[j % CH]);
        }
    };
    if (l.live) {
        int r = l.rt;
        const T *q = base + (int64_t)r * p.ldx;
        const int64_t step = (int64_t)rp * p.ldx;
        Pack<T, V> d[NB], nx[NB];
        if (r + (NB - 1) * rp < rows)
#pragma unroll
            for (int k = 0; k < NB; ++k) d[k] = load_lane<T, V>(q + k * step, l);
        for (; r + (NB - 1) * rp < rows; r += NB * rp) {
            q += NB * step;
            if (r + (2 * NB - 1) * rp < rows)
#pragma unroll
                for (int k = 0; k < NB; ++k) nx[k] = load_lane<T, V>(q + k * step, l);
#pragma unroll
            for (int k = 0; k < NB; ++k) add(d[k]);
#pragma unroll
            for (int k = 0; k < NB; ++k) d[k] = nx[k];
        }
        for (; r < rows; r += rp, q += step) add(load_lane<T, V>(q, l));
    }
    const int per = divided_any(rows, rp), rem = rows - per * rp;
    double2 *out = p.part + ((int64_t)img * p.G * p.P + (p.P == 1 ? divided_any(s0, p.cg) : sl)) * p.S + chunk;
    unit_sums<TPB, V, HOW>(s1, s2, per > 0 ? rp : rem, l, nv, sc, uw, p.m_uw, m_w, nu, entries, nullptr,
                           [&](int u, double a, double b) { out[(int64_t)u * p.S] = make_double2(a, b); });
}

// ---- split form, merge: a workgroup per image and group adds up the chunks and writes mean, scale and shift of its channels ------------
__global__ __launch_bounds__(256) void norm_merge_kernel(NormP p) {
    __shared__ double2 red[4];
    const int img = blockIdx.x / (unsigned)p.G, g = blockIdx.x - img * p.G, t = threadIdx.x;
    const int n = p.S * p.P;
    const double2 *src = p.part + ((int64_t)img * p.G + g) * n;
    double a = 0, b = 0;
#pragma unroll 4
    for (int e = t; e < n; e += 256) a += src[e].x, b += src[e].y;
    a = wave_sum_hi(a), b = wave_sum_hi(b);
    if ((t & 63) == 63) red[t >> 6] = make_double2(a, b);
    __syncthreads();
    const Moments m = moments((red[0].x + red[1].x) + (red[2].x + red[3].x), (red[0].y + red[1].y) + (red[2].y + red[3].y), (double)p.R * p.cg, p.eps);
    const int64_t at = (int64_t)img * p.C + g * p.cg;
    const float *wt = p.w ? p.w + g * p.cg : nullptr, *bt = p.b ? p.b + g * p.cg : nullptr;
    for (int c = t; c < p.cg; c += 256) {
        const float a = wt ? m.rstd * wt[c] : m.rstd;
        p.mean[at + c] = m.mean, p.scale[at + c] = a, p.shift[at + c] = fmaf(-m.low, a, bt ? bt[c] : 0.f);
    }
}

// A thread's V channels of a per-channel array that starts at the slice, as wide loads: one by one each of them touches every line of the row
// again (with 8 channels to a thread those loads were half of the normalising pass: 34560x256 bf16 to 8 bits 25 -> 21 us). NARROW: a slice may
// be narrower than V.
template <int V, bool NARROW> __device__ __forceinline__ void load_channels(const float *p, const Lane<V> &l, int sc, float none, float (&o)[V]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = none;
    } else if (!NARROW || sc >= V) {
        const Pack<float, V> d = load_pack<float, V>(p + l.lo);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = d.v[j];
    } else
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = p[min(l.lo + j, sc - 1)];
}

// ---- normalise, activate, store: shared by both forms -------------------------------------------------------------------------------
template <int V> struct Affine {
    float mean[V], a[V], b[V];                                // (a, b: weight and bias before `set`)
    __device__ __forceinline__ void set(int j, const Moments &m) { mean[j] = m.mean, a[j] *= m.rstd, b[j] = fmaf(-m.low, a[j], b[j]); }
};
template <typename T, int V> __device__ __forceinline__ void finish(const Pack<T, V> &d, const Affine<V> &f, const NormP &p, float (&y)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = fmaf(to_f32(d.v[j]) - f.mean[j], f.a[j], f.b[j]);
    apply_act(y, p.act);
}
// `whole`: the V channels that were loaded are stored, those of the neighbour with the same values (not where x is written over: this thread
// may have read them after the neighbour stored)
template <typename T, int V> __device__ __forceinline__ void store_lane(T *row, const Lane<V> &l, const float (&y)[V], bool whole) {
    if (l.end == V && (l.own == 0 || whole)) {
        Pack<T, V> r;
#pragma unroll
        for (int j = 0; j < V; ++j) r.v[j] = from_f32<T>(y[j]);
        store_pack(row + l.lo, r);
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (l.owns(j)) row[l.lo + j] = from_f32<T>(y[j]);
}
// 8-bit store of a row's slice (its first column a multiple of 128): 16 consecutive lanes hold one block of 128 columns. `y` of channels that
// the thread does not own is not looked at; a tail thread's own channels start at `own`, its bytes at column cv * 8.
__device__ __forceinline__ void store_lane_fp8(uint8_t *qrow, uint8_t *srow, const Lane<8> &l, int sc, const float (&y)[8]) {
    float z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = y[j];
    if (l.own != 0 || l.end != 8) {                             // own channels to the front, in three steps; zeros behind them
#pragma unroll
        for (int b = 1; b < 8; b *= 2)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (l.own & b) z[j] = j + b < 8 ? z[j + b] : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j >= l.end - l.own) z[j] = 0.f;
    }
    const uint32_t byte = fp8_scale_byte(row16_finite_max(z));
    const float inv = scale_inverse(byte);
    const int c0 = l.cv * 8;
    if (c0 < ((sc + 15) & ~15)) {
        uint2 o;
        o.x = to_e4m3x4(z[0] * inv, z[1] * inv, z[2] * inv, z[3] * inv);
        o.y = to_e4m3x4(z[4] * inv, z[5] * inv, z[6] * inv, z[7] * inv);
        *reinterpret_cast<uint2 *>(qrow + c0) = o;
    }
    if ((l.cv & 15) == 0) srow[l.cv >> 4] = (uint8_t)byte;
}

// JOIN: the moments of the slice's groups from the chunks' sums, here
template <typename T, int V, bool TO8, bool JOIN>
__global__ __launch_bounds__(256) void norm_apply_kernel(NormP p, int width, int nsl, int S2, int64_t chunk2) {
    constexpr int TPB = 256, NB = TO8 ? 2 : 4;
    unsigned id = gridDim.x - 1 - blockIdx.x;                  // the opposite order of the first pass
    const int sl = id % (unsigned)nsl;
    id /= (unsigned)nsl;
    const int chunk = id % (unsigned)S2, img = id / (unsigned)S2;
    const int s0 = sl * width, sc = min(width, p.C - s0), t = threadIdx.x;
    int nv = p.nv;
    uint32_t m_nv = p.m_nv;
    if (sc != width) nv = threads_of<V, TO8>(sc), m_nv = division_magic(nv);
    const int rp = divided(TPB, m_nv);
    const Lane<V> l(t, nv, m_nv, rp, sc);
    __shared__ Moments joined[JOIN ? kSliceMax : 1];
    const int first = JOIN ? divided_any(s0, p.cg) : 0;        // the slice's first group
    if constexpr (JOIN) {
        const int ng = divided_any(s0 + sc - 1, p.cg) - first + 1, n = p.S * p.P;
        int sh = 6;
        while (sh > 0 && (ng << sh) > TPB) --sh;
        const int lanes = 1 << sh, li = t & (lanes - 1);
        for (int g = t >> sh; g < ng; g += TPB >> sh) {
            const double2 *src = p.part + ((int64_t)img * p.G + first + g) * n;
            double a = 0, b = 0;
#pragma unroll 4
            for (int e = li; e < n; e += lanes) a += src[e].x, b += src[e].y;
            for (int o = lanes >> 1; o > 0; o >>= 1) a += __shfl_xor(a, o), b += __shfl_xor(b, o);
            if (li == 0) joined[g] = moments(a, b, (double)p.R * p.cg, p.eps);
        }
        __syncthreads();
    }
    if (!l.live) return;
    const int64_t r0 = chunk * chunk2;
    const int rows = (int)(min(r0 + chunk2, p.R) - r0);
    const int64_t at = (int64_t)img * p.R + r0 + l.rt;
    const T *q = (const T *)p.x + at * p.ldx + s0;
    T *o = TO8 ? nullptr : (T *)p.y + at * p.ldy + s0;
    uint8_t *oq = TO8 ? p.q + at * p.ldq + s0 : nullptr, *os = TO8 ? p.qs + at * p.ldqs + s0 / kFp8Block : nullptr;
    const int64_t sx = (int64_t)rp * p.ldx;
    Affine<V> f;
    if constexpr (JOIN) {
        load_channels<V, TO8>(p.b ? p.b + s0 : nullptr, l, sc, 0.f, f.b);
        load_channels<V, TO8>(p.w ? p.w + s0 : nullptr, l, sc, 1.f, f.a);
        int g = divided_any(s0 + l.lo, p.cg), in_g = s0 + l.lo - g * p.cg;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            f.set(j, joined[min(g - first, kSliceMax - 1)]);
            if (++in_g == p.cg) in_g = 0, ++g;
        }
    } else {
        load_channels<V, TO8>(p.mean + (int64_t)img * p.C + s0, l, sc, 0.f, f.mean);
        load_channels<V, TO8>(p.scale + (int64_t)img * p.C + s0, l, sc, 0.f, f.a);
        load_channels<V, TO8>(p.shift + (int64_t)img * p.C + s0, l, sc, 0.f, f.b);
    }
    auto emit = [&](const Pack<T, V> &d, int64_t k) {
        float y[V];
        finish<T, V>(d, f, p, y);
        if constexpr (TO8) store_lane_fp8(oq + k * rp * p.ldq, os + k * rp * p.ldqs, l, sc, y);
        else store_lane<T, V>(o + k * rp * p.ldy, l, y, !p.in_place);
    };
    int r = l.rt;
    int64_t k = 0;
    // (lanes of a row of 16 share rt: they enter and leave these loops together, so the block maximum sees all of them)
    for (; r + (NB - 1) * rp < rows; r += NB * rp, k += NB) {
        Pack<T, V> d[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) d[i] = load_lane<T, V, TO8>(q + (k + i) * sx, l);
#pragma unroll
        for (int i = 0; i < NB; ++i) emit(d[i], k + i);
    }
    for (; r < rows; r += rp, ++k) emit(load_lane<T, V, TO8>(q + k * sx, l), k);
}

// ---- resident form --------------------------------------------------------------------------------------------------------------------
// Where there are few groups, several workgroups hold the same slice, make the same statistics of it and share its rows on the way out, which
// is the longest part (and not possible where x is written over).
// Rolled loops on purpose: the form serves small maps, whose time is latency, and 50 KB of straight-line code cost more to fetch than the map
// (27 us for 3 x 1961 x 100 fp16 with the slice in registers and everything unrolled; 8.3 as it is, 8.5 with 4 rows at a time and 10.6 with 8).
constexpr int kResidentRows = 2; // rows that a thread has under way
template <typename T, int V, int TPB, Sums HOW, bool TO8>
__global__ __launch_bounds__(TPB) void norm_resident_kernel(NormP p) {
    constexpr int NB = kResidentRows;
    using D = Pack<T, V>;
    using W = std::conditional_t<(sizeof(D) >= 16), i32x4, T>;  // how a thread's data lies in the LDS
    extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];
    unsigned id = blockIdx.x;
    const int part = id % (unsigned)p.parts;
    id /= (unsigned)p.parts;
    const int sl = id % (unsigned)p.nslices, img = id / (unsigned)p.nslices, t = threadIdx.x;
    const int s0 = sl * p.slice, sc = min(p.slice, p.C - s0), uw = p.cg, mu = divided(p.slice, p.m_uw), nu = divided(sc, p.m_uw);
    Moments *stat = (Moments *)(dyn + entry_bytes(TPB, HOW, V));
    constexpr int Q = sizeof(D) / sizeof(W);
    W *data = (W *)(dyn + entry_bytes(TPB, HOW, V) + 16 * mu) + t;
    auto put = [&](W *to, const D &x) {
        W v[Q];
        __builtin_memcpy(v, &x, sizeof(x));
#pragma unroll
        for (int i = 0; i < Q; ++i) to[i * TPB] = v[i];
    };
    auto get = [&](const W *from) {
        W v[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) v[i] = from[i * TPB];
        D x;
        __builtin_memcpy(&x, v, sizeof(x));
        return x;
    };
    int nv = p.nv;
    uint32_t m_nv = p.m_nv;
    if (sc != p.slice) nv = threads_of<V, TO8>(sc), m_nv = division_magic(nv);
    const int rp = divided(TPB, m_nv);
    const Lane<V> l(t, nv, m_nv, rp, sc);
    const int R = (int)p.R;
    const T *base = (const T *)p.x + (int64_t)img * R * p.ldx + s0;
    D d[NB];
    auto load = [&](int r) {
#pragma unroll
        for (int k = 0; k < NB; ++k) d[k] = load_lane<T, V, TO8>(base + (int64_t)min(r + k * rp, R - 1) * p.ldx, l);
    };
    load(l.rt);
    Affine<V> f;
    load_channels<V, TO8>(p.w ? p.w + s0 : nullptr, l, sc, 1.f, f.a);
    load_channels<V, TO8>(p.b ? p.b + s0 : nullptr, l, sc, 0.f, f.b);
    constexpr int CH = kChains<V, HOW>;
    double s1[CH] = {}, s2[CH] = {};
    W *at = data;
    for (int r = l.rt; r < R;) {
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            put(at + k * Q * TPB, d[k]);
            const bool on = r + k * rp < R;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double x = on ? to_f32(d[k].v[j]) : 0.f;
                s1[j % CH] += x;
                s2[j % CH] = fma(x, x, s2[j % CH]);
            }
        }
        at += NB * Q * TPB;
        r += NB * rp;
        if (r < R) load(r);
    }
    const int per = divided_any(R, rp), rem = R - per * rp;
    Lane<V> le = l;                                            // (the 8-bit form's padding lanes own nothing and take no part in the sums)
    le.live = l.live && l.cv * V < sc;
    unit_sums<TPB, V, HOW>(s1, s2, per > 0 ? rp : rem, le, nv, sc, uw, p.m_uw, p.m_w, nu, dyn, [&](int u) { return (double *)&stat[u]; },
                           [&](int u, double a, double b) { stat[u] = moments(a, b, (double)R * uw, p.eps); });
    __syncthreads();
    if (!l.live) return;
    int un[V];
    l.template units<HOW == ONE>(uw, p.m_uw, nu, un);
#pragma unroll
    for (int j = 0; j < V; ++j) f.set(j, stat[un[j]]);
    // this workgroup's share of the rows
    const int its = per + (rem ? 1 : 0), share = (its + p.parts - 1) / p.parts, from = part * share, end = min(R, (from + share) * rp);
    at = data + from * (Q * TPB);
    int64_t row = (int64_t)img * R + l.rt + from * rp;
    for (int r = l.rt + from * rp; r < end; r += rp, at += Q * TPB, row += rp) {     // (the 16 lanes of a block share r)
        float y[V];
        finish<T, V>(get(at), f, p, y);
        if constexpr (TO8) store_lane_fp8(p.q + row * p.ldq + s0, p.qs + row * p.ldqs + s0 / kFp8Block, l, sc, y);
        else store_lane<T, V>((T *)p.y + row * p.ldy + s0, l, y, true);
    }
}

// ---- which form, with which split ---------------------------------------------------------------------------------------------------
struct NormPlan {
    bool resident;
    int tpb;                 // resident
    size_t lds;
    int V;
    int slice, nslices, P, piece, S;
    int64_t chunk;
    Sums sums;
    bool join;               // split: the normalising pass adds up the chunks itself
};
static int gcd_i(int a, int b) { return b ? gcd_i(b, a % b) : a; }
constexpr int kMergeMax = 2048;          // chunks x pieces: what one merging workgroup adds up
constexpr int kResidentBytes = 159 * 1024;   // of the CU's 160 KB (a workgroup's own 128 bytes beside)

static NormPlan norm_plan(int64_t R, int images, int C, int G, int es, bool to8) {
    NormPlan q{};
    const int cg = C / G;
    int V = to8 ? 8 : 16 / es;
    // Resident: the narrowest slice of whole groups whose rows are 32 contiguous bytes (a slice of 8-bit rows starts at a block: a multiple
    // of 128 columns, or the whole row), if the LDS holds it
    const int64_t unit = to8 ? (int64_t)cg / gcd_i(cg, kFp8Block) * kFp8Block : cg;
    int64_t slice = unit * ((32 / es + unit - 1) / unit);
    if (slice > C) slice = C;
    const auto last = [&](int64_t w) { return C % w ? C % w : w; };
    if (!to8 && last(slice) < V) V = 1;
    q.V = V;
    q.sums = sums_of(cg, V);
    const int64_t nv = to8 ? (slice + kFp8Block - 1) / kFp8Block * (kFp8Block / 8) : (slice + V - 1) / V;
    if (nv <= 512 && R <= kResidentBytes) {
        q.tpb = nv <= 256 && R <= 8 * (256 / nv) ? 256 : 512;
        const int64_t rp = q.tpb / nv, its = (R + kResidentRows * rp - 1) / (kResidentRows * rp) * kResidentRows;
        q.slice = (int)slice;
        const size_t map = 16 * (size_t)(slice / cg) + (size_t)(its * q.tpb * V * es);
        if (q.sums == EACH && entry_bytes(q.tpb, EACH, V) + map > kResidentBytes) q.sums = TURNS;
        q.lds = entry_bytes(q.tpb, q.sums, V) + map;
        if (q.lds <= kResidentBytes) {
            q.resident = true;
            q.nslices = (int)((C + slice - 1) / slice);
            return q;
        }
    }
    for (V = 16 / es, q.piece = kSliceMax;; V = 1, q.piece = 256) {
        q.P = (cg + q.piece - 1) / q.piece;
        q.slice = q.P == 1 ? std::min(q.piece / cg * cg, C) : q.piece;
        q.nslices = q.P == 1 ? (C + q.slice - 1) / q.slice : G * q.P;
        if (V == 1 || (q.P == 1 ? last(q.slice) : (cg - 1) % q.piece + 1) >= V) break;
    }
    q.V = V;
    q.sums = sums_of(cg, V);
    // about 4 workgroups per CU, each with at least 8 rows per thread
    const int64_t rp = 256 / ((q.slice + V - 1) / V);
    int64_t S = std::min<int64_t>(1024 / std::max<int64_t>(1, std::min<int64_t>((int64_t)images * q.nslices, 1024)), std::max(1, kMergeMax / q.P));
    int64_t chunk = (R + S - 1) / S;
    if (chunk < 8 * rp) chunk = 8 * rp;
    q.chunk = chunk;
    q.S = (int)((R + chunk - 1) / chunk);
    // joining costs every workgroup of the last pass what it reads; a launch costs 3 us of the device's time and as much of the host's
    q.join = (int64_t)q.S * q.P * G <= 1024;
    return q;
}

// Sizes within which the plan's and the workspace's arithmetic holds (an image's rows are counted in 32 bits; more images x columns than 2^40 values
// fit no memory)
static bool norm_range(int64_t rows, int64_t images, int64_t cols) {
    return rows < (1LL << 40) && cols <= (1 << 30) && rows / images <= (1LL << 30) && images * cols <= (1LL << 40);
}
static int64_t norm_ws(const NormPlan &q, int images, int C, int G) {
    return q.resident ? 0 : 16 * (int64_t)images * q.S * G * q.P + (q.join ? 0 : 12 * (int64_t)images * C);
}

template <typename T, int V, int TPB, Sums HOW, bool TO8> static int launch_resident(const NormP &p, const NormPlan &q, int images, hipStream_t s) {
    static LdsGrant grant;
    if (q.lds > 64 * 1024)                                       // (all there is, once: two threads' calls never lower each other's limit)
        if (int rc = grant.ensure((const void *)norm_resident_kernel<T, V, TPB, HOW, TO8>, kResidentBytes, 64 * 1024)) return rc;
    NormP n = p;
    const int rp = TPB / threads_of<V, TO8>(q.slice), its = (int)((p.R + rp - 1) / rp);
    n.parts = p.in_place ? 1 : std::max(1, std::min(std::min(12, its), 256 / (int)std::min<int64_t>(256, (int64_t)images * q.nslices)));
    n.nv = threads_of<V, TO8>(q.slice), n.m_nv = division_magic(n.nv);
    n.m_uw = division_magic(p.cg), n.m_w = division_magic(entries_of(HOW, p.cg, V));
    const int64_t workgroups = (int64_t)images * q.nslices * n.parts;
    LSSVC_CHECK(fits_launch(workgroups, TPB), "group_norm: %lld workgroups do not fit one launch", (long long)workgroups);
    norm_resident_kernel<T, V, TPB, HOW, TO8><<<(unsigned)workgroups, TPB, q.lds, s>>>(n);
    return launch_status("group_norm");
}
template <typename T, int TPB> static int launch_resident(const NormP &p, const NormPlan &q, int images, bool to8, hipStream_t s) {
    auto form = [&](auto v, auto to8_) {
        constexpr int V = decltype(v)::value;
        constexpr bool TO8 = decltype(to8_)::value;
        if (q.sums == ONE) return launch_resident<T, V, TPB, ONE, TO8>(p, q, images, s);
        if constexpr (V > 1) {                                 // (1 divides every width)
            if (q.sums == TWO) return launch_resident<T, V, TPB, TWO, TO8>(p, q, images, s);
            if (q.sums == EACH) return launch_resident<T, V, TPB, EACH, TO8>(p, q, images, s);
        }
        return launch_resident<T, V, TPB, TURNS, TO8>(p, q, images, s);
    };
    if (to8) return form(std::integral_constant<int, 8>{}, std::true_type{});
    if (q.V == 1) return form(std::integral_constant<int, 1>{}, std::false_type{});
    return form(std::integral_constant<int, kVecOf<T>>{}, std::false_type{});
}

template <typename T> static int launch_norm(const NormP &p, const NormPlan &q, int images, bool to8, hipStream_t s) {
    if (q.resident) return q.tpb == 256 ? launch_resident<T, 256>(p, q, images, to8, s) : launch_resident<T, 512>(p, q, images, to8, s);
    constexpr int V = kVecOf<T>;
    const int64_t g1 = (int64_t)images * q.S * q.nslices;
    NormP n = p;
    const int uw = q.P == 1 ? p.cg : q.piece;
    n.nv = q.V == 1 ? q.slice : threads_of<V, false>(q.slice), n.m_nv = division_magic(n.nv);
    n.m_uw = division_magic(uw), n.m_w = division_magic(entries_of(q.sums, uw, q.V));
    // the normalising pass: slices of columns that need not hold whole groups
    const int tail = p.C % kSliceMax, V2 = to8 ? 8 : tail && tail < V ? 1 : V, width = V2 == 1 ? 256 : kSliceMax;
    const int nsl = (p.C + width - 1) / width, sc = std::min(p.C, width);
    const int nv = to8 ? threads_of<8, true>(sc) : (sc + V2 - 1) / V2;
    const int64_t rp = 256 / nv;
    int64_t S2 = std::max<int64_t>(1, 4096 / std::max<int64_t>(1, (int64_t)images * nsl));
    int64_t chunk2 = (p.R + S2 - 1) / S2;
    if (chunk2 < (to8 ? 2 : 3) * rp) chunk2 = (to8 ? 2 : 3) * rp;         // (with 4 rows to a thread 10 % slower, with 8 20 %)
    S2 = (p.R + chunk2 - 1) / chunk2;
    const int64_t g2 = images * S2 * nsl;
    const int64_t g_merge = (int64_t)images * p.G;
    LSSVC_CHECK(fits_launch(std::max(std::max(g1, g2), g_merge), 256), "group_norm: %d images of %lld rows do not fit one launch", images, (long long)p.R);
    if (q.V == 1) norm_stats_kernel<T, 1, ONE><<<(unsigned)g1, 256, 0, s>>>(n);
    else if (q.sums == ONE) norm_stats_kernel<T, V, ONE><<<(unsigned)g1, 256, 0, s>>>(n);
    else if (q.sums == TWO) norm_stats_kernel<T, V, TWO><<<(unsigned)g1, 256, 0, s>>>(n);
    else norm_stats_kernel<T, V, EACH><<<(unsigned)g1, 256, 0, s>>>(n);
    const bool join = q.join;
    if (!join) norm_merge_kernel<<<(unsigned)g_merge, 256, 0, s>>>(p);
    n.nv = nv, n.m_nv = division_magic(nv);
    auto apply = [&](auto kernel) { kernel<<<(unsigned)g2, 256, 0, s>>>(n, sc, nsl, (int)S2, chunk2); };
    if (to8) join ? apply(norm_apply_kernel<T, 8, true, true>) : apply(norm_apply_kernel<T, 8, true, false>);
    else if (V2 == 1) join ? apply(norm_apply_kernel<T, 1, false, true>) : apply(norm_apply_kernel<T, 1, false, false>);
    else join ? apply(norm_apply_kernel<T, V, false, true>) : apply(norm_apply_kernel<T, V, false, false>);
    return launch_status("group_norm");
}

// All images: as many at a time as one launch's threads can be counted for (one-row images of 8 narrow slices: 2 million)
template <typename T> static int launch_images(const NormP &p, const NormPlan &q, int images, bool to8, hipStream_t s) {
    const int64_t sl2 = (p.C + 255) / 256;                     // (at least the last pass's slices)
    const int64_t per = q.resident ? q.nslices : std::max<int64_t>(std::max<int64_t>((int64_t)q.nslices * q.S, sl2), q.join ? 0 : p.G);
    const int most = (int)std::min<int64_t>(images, std::max<int64_t>(1, ((1LL << 32) - 1) / (q.resident ? q.tpb : 256) / per));
    for (int64_t i = 0; i < images; i += most) {
        NormP n = p;
        const int64_t rows = i * p.R;
        n.x = (const T *)p.x + rows * p.ldx;
        if (to8) n.q = p.q + rows * p.ldq, n.qs = p.qs + rows * p.ldqs;
        else n.y = (T *)p.y + rows * p.ldy;
        n.part = p.part + i * q.S * p.G * q.P;
        n.mean = p.mean + i * p.C, n.scale = p.scale + i * p.C, n.shift = p.shift + i * p.C;
        if (int rc = launch_norm<T>(n, q, (int)std::min<int64_t>(most, images - i), to8, s)) return rc;
    }
    return 0;
}

int fp8_out_check(const char *what, const lssvc_fp8 *y, int64_t rows, int cols) {
    LSSVC_CHECK(y && (rows == 0 || (y->values && y->scale)), "%s: no 8-bit output", what);
    LSSVC_CHECK(y->rows == rows && y->cols == cols, "%s: 8-bit output is %lld x %d, expected %lld x %d", what, (long long)y->rows, y->cols, (long long)rows, cols);
    LSSVC_CHECK(y->scale_e8m0 == 1 && y->reserved == 0, "%s: 8-bit outputs have e8m0 scales", what);
    LSSVC_CHECK(aligned(y->values, 16) && y->ld % 16 == 0 && y->ld >= (cols + 15) / 16 * 16, "%s: 8-bit values need a 16-byte aligned base and a pitch that is a multiple of 16", what);
    LSSVC_CHECK(aligned(y->scale, 4) && y->scale_ld % 4 == 0 && y->scale_ld >= (cols + kFp8Block - 1) / kFp8Block, "%s: e8m0 scales need a 4-byte aligned base and a pitch that is a multiple of 4", what);
    return 0;
}

int rows_check(const char *what, const lssvc_rows *x) {
    LSSVC_CHECK(x && x->rows >= 0 && (x->ptr || x->rows == 0) && x->cols > 0 && x->ld >= x->cols, "%s: bad rows", what);
    LSSVC_CHECK(rows_type_ok(x->dtype), "%s: unknown element type %d", what, x->dtype);
    LSSVC_CHECK(aligned(x->ptr, rows_type_size(x->dtype)), "%s: rows are not aligned to their element", what);
    LSSVC_CHECK(x->rows < (1LL << 40) && x->ld < (1LL << 32) && x->cols <= (1 << 30), "%s: %lld rows x %d, pitch %lld, is out of range", what, (long long)x->rows, x->cols, (long long)x->ld);
    return 0;
}

}  // namespace lssvc

using namespace lssvc;

extern "C" int64_t lssvc_group_norm_workspace_bytes(int64_t rows, int32_t images, int32_t cols, int32_t groups, int32_t dtype, int32_t to_fp8) {
    if (rows <= 0 || images <= 0 || cols <= 0 || groups <= 0 || cols % groups || rows % images || !rows_type_ok(dtype) || !norm_range(rows, images, cols)) return 0;
    return norm_ws(norm_plan(rows / images, images, cols, groups, rows_type_size(dtype), to_fp8 != 0), images, cols, groups);
}

extern "C" int lssvc_group_norm(const lssvc_rows *x, int32_t images, int32_t groups, const float *weight, const float *bias, float eps,
                                int32_t act, float slope, const lssvc_rows *y, const lssvc_fp8 *y8, void *workspace, int64_t workspace_bytes,
                                void *stream) {
    if (int rc = rows_check("group_norm", x)) return rc;
    LSSVC_CHECK(images > 0 && x->rows % images == 0, "group_norm: %lld rows are not %d images", (long long)x->rows, images);
    LSSVC_CHECK(groups > 0 && x->cols % groups == 0, "group_norm: %d channels are not %d groups", x->cols, groups);
    LSSVC_CHECK(eps >= 0.f, "group_norm: eps %g", eps);
    LSSVC_CHECK(act_ok(act), "group_norm: unknown activation %d", act);
    LSSVC_CHECK((y != nullptr) != (y8 != nullptr), "group_norm: exactly one of the outputs is given");
    LSSVC_CHECK(norm_range(x->rows, images, x->cols), "group_norm: %d images of %lld rows x %d channels are too large", images, (long long)(x->rows / images), x->cols);
    const int64_t R = x->rows / images;
    const NormPlan q = norm_plan(R, images, x->cols, groups, rows_type_size(x->dtype), y8 != nullptr);
    const int64_t need = x->rows ? norm_ws(q, images, x->cols, groups) : 0;
    const Span ws{(uintptr_t)workspace, workspace ? (uint64_t)need : 0};
    if (y) {
        if (int rc = rows_check("group_norm", y)) return rc;
        LSSVC_CHECK(y->rows == x->rows && y->cols == x->cols && y->dtype == x->dtype, "group_norm: the output's shape or type is not the input's");
        if (x->rows) LSSVC_CHECK(rows_disjoint_or_same(x, y), "group_norm: input and output overlap in part");
        LSSVC_CHECK(apart({span_of(y), ws}, {span_of(weight, x->cols), span_of(bias, x->cols)}), "group_norm: the output overlaps weight, bias or workspace");
    } else if (int rc = fp8_out_check("group_norm", y8, x->rows, x->cols)) return rc;
    if (y8) {
        LSSVC_CHECK(y8->block_rows == 1, "group_norm: 8-bit output has 1 x 128 blocks");
        LSSVC_CHECK(apart({values_of(y8), scales_of(y8), ws}, {span_of(x), span_of(weight, x->cols), span_of(bias, x->cols)}), "group_norm: the output overlaps an input or the workspace");
    } else LSSVC_CHECK(apart({ws}, {span_of(x)}), "group_norm: the workspace overlaps the input");
    if (x->rows == 0) return 0;
    LSSVC_CHECK(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), "group_norm: workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)need, (long long)workspace_bytes);
    LSSVC_CHECK(q.P <= kMergeMax, "group_norm: an image of %lld rows x %d channels in %d groups is too large", (long long)R, x->cols, groups);
    NormP p{};
    p.x = x->ptr;
    p.ldx = x->ld;
    if (y) p.y = y->ptr, p.ldy = y->ld;
    else p.q = (uint8_t *)y8->values, p.ldq = y8->ld, p.qs = (uint8_t *)y8->scale, p.ldqs = y8->scale_ld;
    p.R = R;
    p.w = weight, p.b = bias;
    p.C = x->cols, p.G = groups, p.cg = x->cols / groups;
    p.S = q.S, p.P = q.P, p.piece = q.piece, p.chunk = q.chunk, p.slice = q.slice, p.nslices = q.nslices;
    p.act = Act{act, slope}, p.eps = eps;
    p.in_place = y && y->ptr == x->ptr;
    p.part = (double2 *)workspace;
    p.mean = (float *)(p.part + (int64_t)images * q.S * groups * q.P);
    p.scale = p.mean + (int64_t)images * x->cols;
    p.shift = p.scale + (int64_t)images * x->cols;
    hipStream_t s = (hipStream_t)stream;
    if (x->dtype == LSSVC_F32) return launch_images<float>(p, q, images, y8 != nullptr, s);
    if (x->dtype == LSSVC_F16) return launch_images<f16_t>(p, q, images, y8 != nullptr, s);
    return launch_images<bf16_t>(p, q, images, y8 != nullptr, s);
}
