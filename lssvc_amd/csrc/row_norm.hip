// row_norm.hip -- group norm with an activation over channels-last rows, optionally straight into 8-bit blocks.
//
// y = act((x - mu) * rsqrt(var + eps) * w_c + b_c), mu / var over the rows of an image and the cg = C / G channels of a group. The
// operator is bound by memory: one read and one write of the map if it stays on the chip between the statistics and their use, two reads
// otherwise. Two forms:
//   resident  a workgroup owns all rows of a slice of whole groups and holds the slice in registers (up to 256 KB): one read, one write,
//             one launch.
//   split     rows are split over workgroups that write (mean, M2) per chunk and group; one wave per group merges the chunks; the
//             normalising pass reads the map again, in the opposite order, so that what the first pass read last comes from the caches.
// Every sum is taken of differences to a value of the group itself (a pivot), and squares of differences to a mean, never E[x^2] - E[x]^2:
// a map whose offset is a thousand times its spread keeps the digits of its spread.
//
// One thread handles 8 consecutive channels (16 or 32 bytes, at any alignment). Where 8 does not divide the slice, a row's last thread
// loads the LAST 8 channels -- wide loads only -- and owns those that its neighbour does not.
#include "rows.h"

namespace lssvc {

struct NormP {
    const void *x;
    void *y;                     // T rows (to_fp8: unused)
    uint8_t *q, *qs;             // 8-bit values and scale bytes (to_fp8)
    int64_t ldx, ldy, ldq, ldqs;
    int64_t R;                   // rows of an image
    const float *w, *b;
    float2 *part, *stat;         // split form: [image][chunk][unit] (mean, M2); [image][group] (mean, 1 / sqrt(var + eps))
    int64_t chunk;               // rows of a chunk
    int C, G, cg;
    int S;                       // chunks of an image
    int P;                       // pieces of a group (1, or slices of kSliceMax where a group is wider than that)
    int slice, nslices;          // columns of a slice (P = 1), slices of a row
    int act;
    float eps, slope;
};

constexpr int kVec = 8;
constexpr int kSliceMax = 2048;

// a thread's 8 channels of a slice that is `sc` columns wide
struct Lane {
    int cv, rt;        // which 8 channels, which of the rows in flight
    int lo;            // first channel that is loaded
    int own;           // loaded channels from `own` on are this thread's (below `end`)
    int end;
    bool live;
    __device__ __forceinline__ Lane(int t, int nv, int rp, int sc) {
        rt = t / nv;
        cv = t - rt * nv;
        live = rt < rp;
        const int c0 = cv * kVec;
        lo = sc >= kVec ? min(c0, sc - kVec) : 0;
        own = c0 - lo;
        end = sc >= kVec ? kVec : sc;
        if (c0 >= sc) own = end = 0, lo = 0;         // padding lane of the 8-bit form: owns nothing
    }
    __device__ __forceinline__ bool owns(int j) const { return j >= own && j < end; }
};

template <typename T> __device__ __forceinline__ Pack<T, kVec> load_lane(const T *row, const Lane &l) {
    if (l.end == kVec) return load_pack<T, kVec>(row + l.lo);
    Pack<T, kVec> r;
#pragma unroll
    for (int j = 0; j < kVec; ++j) r.v[j] = j < l.end ? row[l.lo + j] : from_f32<T>(0.f);
    return r;
}

// Sums over (rows in flight x channels) per unit (a group, or a piece of one): v[j] is the thread's sum for channel lo + j. Entries go to
// the LDS, each unit is added up by `lpu` lanes of one wave in a fixed order, totals come back in `tot`. ONE: 8 divides the unit width, so a
// thread's channels lie in one unit and are added before.
template <int TPB, bool ONE>
__device__ __forceinline__ void unit_sums(const float (&v)[kVec], const Lane &l, int nv, int rp, int sc, int uw, int nu, float *ebuf, float *tot) {
    const int t = threadIdx.x;
    if (l.live) {
        if constexpr (ONE) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) s += v[j];
            ebuf[l.rt * nv + l.cv] = s;
        } else {
#pragma unroll
            for (int j = 0; j < kVec; ++j)
                if (l.owns(j)) ebuf[l.rt * sc + l.lo + j] = v[j];
        }
    }
    __syncthreads();
    const int W = ONE ? uw / kVec : uw, pitch = ONE ? nv : sc;
    int lpu = 64;
    while (lpu > 1 && lpu * nu > TPB) lpu >>= 1;
    const int li = t & (lpu - 1), dr = lpu / W, dc = lpu - dr * W;
    for (int u = t / lpu; u < nu; u += TPB / lpu) {
        float s = 0.f;
        int r = li / W, c = li - r * W;
        while (r < rp) {
            s += ebuf[r * pitch + u * W + c];
            r += dr;
            c += dc;
            if (c >= W) c -= W, ++r;
        }
        for (int o = lpu >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (li == 0) tot[u] = s;
    }
    __syncthreads();
}

// ---- split form, first pass: (mean, M2) of each chunk and unit ---------------------------------------------------------------------
template <typename T, bool ONE>
__global__ __launch_bounds__(256) void norm_stats_kernel(NormP p) {
    constexpr int TPB = 256, NB = 4;
    __shared__ float ebuf[TPB * kVec];
    __shared__ float tot[kSliceMax], piv[kSliceMax];
    unsigned id = blockIdx.x;
    const int sl = id % (unsigned)p.nslices;
    id /= (unsigned)p.nslices;
    const int chunk = id % (unsigned)p.S, img = id / (unsigned)p.S;
    int s0, sc, nu, uw;
    if (p.P == 1) {
        s0 = sl * p.slice;
        sc = min(p.slice, p.C - s0);
        uw = p.cg;
        nu = sc / uw;
    } else {
        const int g = sl / p.P, k = sl - g * p.P;
        s0 = g * p.cg + k * kSliceMax;
        sc = uw = min(kSliceMax, p.cg - k * kSliceMax);
        nu = 1;
    }
    const int nv = (sc + kVec - 1) / kVec, rp = TPB / nv, t = threadIdx.x;
    const Lane l(t, nv, rp, sc);
    const int64_t r0 = chunk * p.chunk, r1 = min(r0 + p.chunk, p.R);
    const T *base = (const T *)p.x + ((int64_t)img * p.R + r0) * p.ldx + s0;
    const int rows = (int)(r1 - r0);
    for (int u = t; u < nu; u += TPB) piv[u] = to_f32(base[u * uw]);

    float n = 0.f, mean[kVec] = {}, m2[kVec] = {};
    if (l.live) {
        int r = l.rt;
        const T *q = base + (int64_t)r * p.ldx;
        const int64_t step = (int64_t)rp * p.ldx;
        for (; r + (NB - 1) * rp < rows; r += NB * rp) {
            Pack<T, kVec> d[NB];
#pragma unroll
            for (int k = 0; k < NB; ++k) d[k] = load_lane(q + k * step, l);
            q += NB * step;
            const float f = (float)NB / (n + NB), nf = n * f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                float x[NB], m = 0.f, s = 0.f;
#pragma unroll
                for (int k = 0; k < NB; ++k) x[k] = to_f32(d[k].v[j]), m += x[k];
                m *= 1.f / NB;
#pragma unroll
                for (int k = 0; k < NB; ++k) s = fmaf(x[k] - m, x[k] - m, s);
                const float dm = m - mean[j];
                mean[j] = fmaf(dm, f, mean[j]);
                m2[j] += fmaf(dm * dm, nf, s);
            }
            n += NB;
        }
        for (; r < rows; r += rp, q += step) {
            const Pack<T, kVec> d = load_lane(q, l);
            const float f = 1.f / (n + 1.f), nf = n * f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float dm = to_f32(d.v[j]) - mean[j];
                mean[j] = fmaf(dm, f, mean[j]);
                m2[j] = fmaf(dm * dm, nf, m2[j]);
            }
            n += 1.f;
        }
    }
    __syncthreads();             // piv
    float v[kVec];
    int un[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) un[j] = min((l.lo + j) / uw, nu - 1);
#pragma unroll
    for (int j = 0; j < kVec; ++j) v[j] = n * (mean[j] - piv[un[j]]);
    if (n == 0.f)
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] = 0.f;
    unit_sums<TPB, ONE>(v, l, nv, rp, sc, uw, nu, ebuf, tot);
    const float inv = 1.f / ((float)rows * (float)uw);
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        const float d = mean[j] - fmaf(tot[un[j]], inv, piv[un[j]]);
        v[j] = n == 0.f ? 0.f : fmaf(n * d, d, m2[j]);
    }
    float um[(kSliceMax + TPB - 1) / TPB];       // this thread's units' means, before `tot` is written again
#pragma unroll
    for (int k = 0; k < (kSliceMax + TPB - 1) / TPB; ++k)
        if (t + k * TPB < nu) um[k] = fmaf(tot[t + k * TPB], inv, piv[t + k * TPB]);
    __syncthreads();
    unit_sums<TPB, ONE>(v, l, nv, rp, sc, uw, nu, ebuf, tot);
    const int U = p.G * p.P, u0 = p.P == 1 ? s0 / p.cg : sl;
    float2 *out = p.part + ((int64_t)img * p.S + chunk) * U + u0;
#pragma unroll
    for (int k = 0; k < (kSliceMax + TPB - 1) / TPB; ++k)
        if (t + k * TPB < nu) out[t + k * TPB] = make_float2(um[k], tot[t + k * TPB]);
}

// ---- split form, merge: one wave per image and group --------------------------------------------------------------------------------
__device__ __forceinline__ float wave_sum(float s) {
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    return s;
}
__global__ __launch_bounds__(64) void norm_merge_kernel(NormP p) {
    const int img = blockIdx.x / (unsigned)p.G, g = blockIdx.x - img * p.G, t = threadIdx.x;
    const int U = p.G * p.P, E = p.S * p.P;
    const float2 *src = p.part + (int64_t)img * p.S * U + g * p.P;
    const float pivot = src[0].x;
    const float inv = 1.f / ((float)p.R * (float)p.cg);
    auto weight = [&](int c, int k) {
        const float rows = (float)min(p.chunk, p.R - (int64_t)c * p.chunk);
        return rows * (float)(p.P == 1 ? p.cg : min(kSliceMax, p.cg - k * kSliceMax));
    };
    float s = 0.f;
    for (int e = t; e < E; e += 64) {
        const int c = e / p.P, k = e - c * p.P;
        s += weight(c, k) * (src[(int64_t)c * U + k].x - pivot);
    }
    const float mean = fmaf(wave_sum(s), inv, pivot);
    s = 0.f;
    for (int e = t; e < E; e += 64) {
        const int c = e / p.P, k = e - c * p.P;
        const float2 v = src[(int64_t)c * U + k];
        const float d = v.x - mean;
        s += fmaf(weight(c, k) * d, d, v.y);
    }
    const float var = wave_sum(s) * inv;
    if (t == 0) p.stat[blockIdx.x] = make_float2(mean, 1.f / sqrtf(var + p.eps));
}

// ---- normalise, activate, store: shared by both forms -------------------------------------------------------------------------------
struct Affine {
    float mean[kVec], a[kVec], b[kVec];
};
__device__ __forceinline__ void finish_row(const float (&x)[kVec], const Affine &f, const NormP &p, float (&y)[kVec]) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) y[j] = apply_act(fmaf(x[j] - f.mean[j], f.a[j], f.b[j]), p.act, p.slope);
}
template <typename T> __device__ __forceinline__ void store_lane(T *row, const Lane &l, const float (&y)[kVec]) {
    if (l.own == 0 && l.end == kVec) {
        Pack<T, kVec> r;
#pragma unroll
        for (int j = 0; j < kVec; ++j) r.v[j] = from_f32<T>(y[j]);
        store_pack(row + l.lo, r);
        return;
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j)
        if (l.owns(j)) row[l.lo + j] = from_f32<T>(y[j]);
}
// 8-bit store of a row's slice (its first column a multiple of 128): 16 consecutive lanes hold one block of 128 columns. `y` of channels that
// the thread does not own is not looked at; a tail thread's own channels start at `own`, its bytes at column cv * 8.
__device__ __forceinline__ void store_lane_fp8(uint8_t *qrow, uint8_t *srow, const Lane &l, int sc, bool row_live, const float (&y)[kVec]) {
    float z[kVec];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        z[j] = 0.f;
        if (l.own == 0) z[j] = j < l.end ? y[j] : 0.f;
        else
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                if (i == j + l.own) z[j] = y[i];
        m = max(m, finite_abs_bits(z[j]));
    }
    const uint32_t byte = fp8_scale_byte(row16_max(m));
    const float inv = scale_inverse(byte);
    if (!row_live) return;
    const int c0 = l.cv * kVec;
    if (c0 < ((sc + 15) & ~15)) {
        uint2 o;
        o.x = to_e4m3x4(z[0] * inv, z[1] * inv, z[2] * inv, z[3] * inv);
        o.y = to_e4m3x4(z[4] * inv, z[5] * inv, z[6] * inv, z[7] * inv);
        *reinterpret_cast<uint2 *>(qrow + c0) = o;
    }
    if ((l.cv & 15) == 0) srow[l.cv >> 4] = (uint8_t)byte;
}

template <typename T, bool TO8>
__global__ __launch_bounds__(256) void norm_apply_kernel(NormP p, int nsl, int S2, int64_t chunk2) {
    constexpr int TPB = 256, NB = 4;
    unsigned id = gridDim.x - 1 - blockIdx.x;                  // the opposite order of the first pass
    const int sl = id % (unsigned)nsl;
    id /= (unsigned)nsl;
    const int chunk = id % (unsigned)S2, img = id / (unsigned)S2;
    const int s0 = sl * kSliceMax, sc = min(kSliceMax, p.C - s0), t = threadIdx.x;
    const int nv = TO8 ? (sc + kFp8Block - 1) / kFp8Block * (kFp8Block / kVec) : (sc + kVec - 1) / kVec, rp = TPB / nv;
    const Lane l(t, nv, rp, sc);
    if (!l.live) return;
    Affine f;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        const int c = s0 + min(l.lo + j, sc - 1);
        const float2 st = p.stat[img * p.G + c / p.cg];
        f.mean[j] = st.x;
        f.a[j] = p.w ? st.y * p.w[c] : st.y;
        f.b[j] = p.b ? p.b[c] : 0.f;
    }
    const int64_t r0 = chunk * chunk2;
    const int rows = (int)(min(r0 + chunk2, p.R) - r0);
    const int64_t at = (int64_t)img * p.R + r0 + l.rt;
    const T *q = (const T *)p.x + at * p.ldx + s0;
    T *o = TO8 ? nullptr : (T *)p.y + at * p.ldy + s0;
    uint8_t *oq = TO8 ? p.q + at * p.ldq + s0 : nullptr, *os = TO8 ? p.qs + at * p.ldqs + s0 / kFp8Block : nullptr;
    const int64_t sx = (int64_t)rp * p.ldx;
    auto emit = [&](const Pack<T, kVec> &d, int64_t k) {
        float x[kVec], y[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[j] = to_f32(d.v[j]);
        finish_row(x, f, p, y);
        if constexpr (TO8) store_lane_fp8(oq + k * rp * p.ldq, os + k * rp * p.ldqs, l, sc, true, y);
        else store_lane(o + k * rp * p.ldy, l, y);
    };
    int r = l.rt;
    int64_t k = 0;
    // (lanes of a row of 16 share rt: they enter and leave these loops together, so the block maximum sees all of them)
    for (; r + (NB - 1) * rp < rows; r += NB * rp, k += NB) {
        Pack<T, kVec> d[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) d[i] = load_lane(q + (k + i) * sx, l);
#pragma unroll
        for (int i = 0; i < NB; ++i) emit(d[i], k + i);
    }
    for (; r < rows; r += rp, ++k) emit(load_lane(q + k * sx, l), k);
}

// ---- resident form --------------------------------------------------------------------------------------------------------------------
template <typename T, int TPB, int NIT, bool ONE, bool TO8>
__global__ __launch_bounds__(TPB) void norm_resident_kernel(NormP p) {
    __shared__ float ebuf[TPB * kVec];
    extern __shared__ float dyn[];                             // tot[units of the slice], piv[...]
    const int sl = blockIdx.x % (unsigned)p.nslices, img = blockIdx.x / (unsigned)p.nslices, t = threadIdx.x;
    const int s0 = sl * p.slice, sc = min(p.slice, p.C - s0), uw = p.cg, nu = sc / uw;
    float *tot = dyn, *piv = dyn + p.slice / p.cg;
    const int nv = TO8 ? (sc + kFp8Block - 1) / kFp8Block * (kFp8Block / kVec) : (sc + kVec - 1) / kVec, rp = TPB / nv;
    const Lane l(t, nv, rp, sc);
    const T *base = (const T *)p.x + (int64_t)img * p.R * p.ldx + s0;
    const int R = (int)p.R;
    Pack<T, kVec> d[NIT];
#pragma unroll
    for (int k = 0; k < NIT; ++k) {
        const int r = l.rt + k * rp;
        d[k] = load_lane(base + (int64_t)min(r, R - 1) * p.ldx, l);
    }
    for (int u = t; u < nu; u += TPB) piv[u] = to_f32(base[u * uw]);
    __syncthreads();
    int un[kVec];
    float pv[kVec], v[kVec] = {};
#pragma unroll
    for (int j = 0; j < kVec; ++j) un[j] = min((l.lo + j) / uw, nu - 1), pv[j] = piv[un[j]];
#pragma unroll
    for (int k = 0; k < NIT; ++k)
        if (l.rt + k * rp < R)
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[j] += to_f32(d[k].v[j]) - pv[j];
    const float inv = 1.f / ((float)R * (float)uw);
    const int ev = (sc + kVec - 1) / kVec;
    Lane le = l;                                               // (the 8-bit form's padding lanes own nothing and take no part in the sums)
    le.live = l.live && l.cv < ev;
    unit_sums<TPB, ONE>(v, le, nv, rp, sc, uw, nu, ebuf, tot);
    Affine f;
#pragma unroll
    for (int j = 0; j < kVec; ++j) f.mean[j] = fmaf(tot[un[j]], inv, pv[j]), v[j] = 0.f;
#pragma unroll
    for (int k = 0; k < NIT; ++k)
        if (l.rt + k * rp < R)
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float x = to_f32(d[k].v[j]) - f.mean[j];
                v[j] = fmaf(x, x, v[j]);
            }
    __syncthreads();                                           // every thread has its means
    unit_sums<TPB, ONE>(v, le, nv, rp, sc, uw, nu, ebuf, tot);
    if (!l.live) return;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        const int c = s0 + min(l.lo + j, sc - 1);
        const float rstd = 1.f / sqrtf(fmaf(tot[un[j]], inv, p.eps));
        f.a[j] = p.w ? rstd * p.w[c] : rstd;
        f.b[j] = p.b ? p.b[c] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < NIT; ++k) {
        const int r = l.rt + k * rp;
        if (r >= R) break;
        float x[kVec], y[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[j] = to_f32(d[k].v[j]);
        finish_row(x, f, p, y);
        const int64_t at = (int64_t)img * p.R + r;
        if constexpr (TO8) store_lane_fp8(p.q + at * p.ldq + s0, p.qs + at * p.ldqs + s0 / kFp8Block, l, sc, true, y);
        else store_lane((T *)p.y + at * p.ldy + s0, l, y);
    }
}

// ---- which form, with which split ---------------------------------------------------------------------------------------------------
struct NormPlan {
    bool resident;
    int tpb, nit;            // resident
    int slice, nslices, P, S;
    int64_t chunk;
    bool one;
};
static int gcd_i(int a, int b) { return b ? gcd_i(b, a % b) : a; }

static NormPlan norm_plan(int64_t R, int images, int C, int G, int es, bool to8) {
    NormPlan q{};
    const int cg = C / G;
    // resident: the narrowest slice of whole groups whose rows are 64 contiguous bytes (a slice of 8-bit rows starts at a block: a multiple
    // of 128 columns, or the whole row), if 1024 threads can hold it: 64 VGPRs of data each
    int64_t unit = to8 ? (int64_t)cg / gcd_i(cg, kFp8Block) * kFp8Block : cg;
    int64_t slice = unit * ((64 / es + unit - 1) / unit);
    if (slice > C) slice = C;
    const int maxit = es == 4 ? 8 : 16;
    const int64_t nv = to8 ? (slice + kFp8Block - 1) / kFp8Block * (kFp8Block / kVec) : (slice + kVec - 1) / kVec;
    if (nv <= 1024 && R <= (int64_t)maxit * (1024 / nv)) {
        q.resident = true;
        q.slice = (int)slice;
        q.nslices = (int)((C + slice - 1) / slice);
        q.tpb = nv <= 256 && R <= 4 * (256 / nv) ? 256 : 1024;
        const int64_t rp = q.tpb / nv, need = (R + rp - 1) / rp;
        q.nit = 1;
        while (q.nit < need) q.nit *= 2;
        q.one = cg % kVec == 0;
        return q;
    }
    q.P = cg > kSliceMax ? (cg + kSliceMax - 1) / kSliceMax : 1;
    q.slice = q.P == 1 ? kSliceMax / cg * cg : kSliceMax;
    if (q.P == 1 && q.slice > C) q.slice = C;
    q.nslices = q.P == 1 ? (C + q.slice - 1) / q.slice : G * q.P;
    q.one = cg % kVec == 0;
    // about 4 workgroups per CU, each with at least 8 rows per thread
    const int64_t rp = 256 / ((std::min(q.slice, C) + kVec - 1) / kVec);
    int64_t S = 1024 / ((int64_t)images * q.nslices);
    if (S < 1) S = 1;
    int64_t chunk = (R + S - 1) / S;
    if (chunk < 8 * rp) chunk = 8 * rp;
    if (chunk > 0x40000000) chunk = 0x40000000;
    q.chunk = chunk;
    q.S = (int)((R + chunk - 1) / chunk);
    return q;
}

static int64_t norm_ws(const NormPlan &q, int images, int G) {
    return q.resident ? 0 : 8 * ((int64_t)images * q.S * G * q.P + (int64_t)images * G);
}

template <typename T, int TPB, int NIT>
static void launch_resident(const NormP &p, const NormPlan &q, int images, bool to8, hipStream_t s) {
    const unsigned grid = (unsigned)(images * q.nslices);
    const size_t dyn = 8 * (size_t)(q.slice / p.cg);
    if (to8) {
        if (q.one) norm_resident_kernel<T, TPB, NIT, true, true><<<grid, TPB, dyn, s>>>(p);
        else norm_resident_kernel<T, TPB, NIT, false, true><<<grid, TPB, dyn, s>>>(p);
    } else {
        if (q.one) norm_resident_kernel<T, TPB, NIT, true, false><<<grid, TPB, dyn, s>>>(p);
        else norm_resident_kernel<T, TPB, NIT, false, false><<<grid, TPB, dyn, s>>>(p);
    }
}

template <typename T> static int launch_norm(const NormP &p, const NormPlan &q, int images, bool to8, hipStream_t s) {
    if (q.resident) {
        if (q.tpb == 256) switch (q.nit) {
            case 1: launch_resident<T, 256, 1>(p, q, images, to8, s); break;
            case 2: launch_resident<T, 256, 2>(p, q, images, to8, s); break;
            default: launch_resident<T, 256, 4>(p, q, images, to8, s); break;
        } else switch (q.nit) {
            case 1: launch_resident<T, 1024, 1>(p, q, images, to8, s); break;
            case 2: launch_resident<T, 1024, 2>(p, q, images, to8, s); break;
            case 4: launch_resident<T, 1024, 4>(p, q, images, to8, s); break;
            case 8: launch_resident<T, 1024, 8>(p, q, images, to8, s); break;
            default:
                if constexpr (sizeof(T) == 2) launch_resident<T, 1024, 16>(p, q, images, to8, s);
                break;
        }
        return launch_status("group_norm");
    }
    const unsigned g1 = (unsigned)((int64_t)images * q.S * q.nslices);
    if (q.one) norm_stats_kernel<T, true><<<g1, 256, 0, s>>>(p);
    else norm_stats_kernel<T, false><<<g1, 256, 0, s>>>(p);
    norm_merge_kernel<<<(unsigned)(images * p.G), 64, 0, s>>>(p);
    const int nsl = (p.C + kSliceMax - 1) / kSliceMax;
    const int sc = std::min(p.C, kSliceMax);
    const int nv = to8 ? (sc + kFp8Block - 1) / kFp8Block * (kFp8Block / kVec) : (sc + kVec - 1) / kVec;
    const int64_t rp = 256 / nv;
    int64_t S2 = 4096 / ((int64_t)images * nsl);
    if (S2 < 1) S2 = 1;
    int64_t chunk2 = (p.R + S2 - 1) / S2;
    if (chunk2 < 4 * rp) chunk2 = 4 * rp;
    if (chunk2 > 0x40000000) chunk2 = 0x40000000;
    S2 = (p.R + chunk2 - 1) / chunk2;
    const unsigned g2 = (unsigned)((int64_t)images * S2 * nsl);
    if (to8) norm_apply_kernel<T, true><<<g2, 256, 0, s>>>(p, nsl, (int)S2, chunk2);
    else norm_apply_kernel<T, false><<<g2, 256, 0, s>>>(p, nsl, (int)S2, chunk2);
    return launch_status("group_norm");
}

int fp8_out_check(const char *what, const lssvc_fp8 *y, int64_t rows, int cols) {
    LSSVC_CHECK(y && (rows == 0 || (y->values && y->scale)), "%s: no 8-bit output", what);
    LSSVC_CHECK(y->rows == rows && y->cols == cols, "%s: 8-bit output is %lld x %d, expected %lld x %d", what, (long long)y->rows, y->cols, (long long)rows, cols);
    LSSVC_CHECK(y->scale_e8m0 == 1 && y->reserved == 0, "%s: 8-bit outputs have e8m0 scales", what);
    LSSVC_CHECK(aligned(y->values, 16) && y->ld % 16 == 0 && y->ld >= (cols + 15) / 16 * 16, "%s: 8-bit values need a 16-byte aligned base and a pitch that is a multiple of 16", what);
    LSSVC_CHECK(aligned(y->scale, 4) && y->scale_ld % 4 == 0 && y->scale_ld >= (cols + kFp8Block - 1) / kFp8Block, "%s: e8m0 scales need a 4-byte aligned base and a pitch that is a multiple of 4", what);
    return 0;
}

static int rows_check(const char *what, const lssvc_rows *x) {
    LSSVC_CHECK(x && x->rows >= 0 && (x->ptr || x->rows == 0) && x->cols > 0 && x->ld >= x->cols, "%s: bad rows", what);
    LSSVC_CHECK(rows_type_ok(x->dtype), "%s: unknown element type %d", what, x->dtype);
    LSSVC_CHECK(aligned(x->ptr, rows_type_size(x->dtype)), "%s: rows are not aligned to their element", what);
    LSSVC_CHECK(x->rows < (1LL << 40) && x->ld < (1LL << 32), "%s: rows %lld x pitch %lld is out of range", what, (long long)x->rows, (long long)x->ld);
    return 0;
}

}  // namespace lssvc

using namespace lssvc;

extern "C" int64_t lssvc_group_norm_workspace_bytes(int64_t rows, int32_t images, int32_t cols, int32_t groups, int32_t dtype, int32_t to_fp8) {
    if (rows <= 0 || images <= 0 || cols <= 0 || groups <= 0 || cols % groups || rows % images || !rows_type_ok(dtype)) return 0;
    return norm_ws(norm_plan(rows / images, images, cols, groups, rows_type_size(dtype), to_fp8 != 0), images, groups);
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
    if (y) {
        if (int rc = rows_check("group_norm", y)) return rc;
        LSSVC_CHECK(y->rows == x->rows && y->cols == x->cols && y->dtype == x->dtype, "group_norm: the output's shape or type is not the input's");
        if (x->rows) LSSVC_CHECK(rows_disjoint_or_same(x, y), "group_norm: input and output overlap in part");
    } else if (int rc = fp8_out_check("group_norm", y8, x->rows, x->cols)) return rc;
    if (y8) LSSVC_CHECK(y8->block_rows == 1, "group_norm: 8-bit output has 1 x 128 blocks");
    if (x->rows == 0) return 0;
    const int64_t R = x->rows / images;
    const int es = rows_type_size(x->dtype);
    const NormPlan q = norm_plan(R, images, x->cols, groups, es, y8 != nullptr);
    const int64_t need = norm_ws(q, images, groups);
    LSSVC_CHECK(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), "group_norm: workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)need, (long long)workspace_bytes);
    LSSVC_CHECK((int64_t)images * std::max<int64_t>(groups, (int64_t)q.nslices * std::max(q.S, 1)) < (1LL << 31), "group_norm: too many images or groups for one launch");
    NormP p{};
    p.x = x->ptr;
    p.ldx = x->ld;
    if (y) p.y = y->ptr, p.ldy = y->ld;
    else p.q = (uint8_t *)y8->values, p.ldq = y8->ld, p.qs = (uint8_t *)y8->scale, p.ldqs = y8->scale_ld;
    p.R = R;
    p.w = weight, p.b = bias;
    p.C = x->cols, p.G = groups, p.cg = x->cols / groups;
    p.S = q.S, p.P = q.P, p.chunk = q.chunk, p.slice = q.slice, p.nslices = q.nslices;
    p.act = act, p.eps = eps, p.slope = slope;
    p.stat = (float2 *)workspace;
    p.part = p.stat + (int64_t)images * groups;
    hipStream_t s = (hipStream_t)stream;
    if (x->dtype == LSSVC_F32) return launch_norm<float>(p, q, images, y8 != nullptr, s);
    if (x->dtype == LSSVC_F16) return launch_norm<f16_t>(p, q, images, y8 != nullptr, s);
    return launch_norm<bf16_t>(p, q, images, y8 != nullptr, s);
}
