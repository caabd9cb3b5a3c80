// Attention of a batch's rows over a paged KV cache: new rows of many
// sequences, one each (a decode step) or chunks of prompts, in one launch and
// a second that joins what the first split.
//
// A sequence's new rows and the heads that share a kv head are its columns:
// column c is row c / group, head kv head * group + c % group. A work item is
// (sequence, kv head, 16 or 128 columns, run of positions), so a key or value is
// read once for as many columns. Both products are MFMAs whose terms keep fp32's
// accuracy (see Ops); the softmax runs with one pass over the positions, a
// running maximum and sum in fp32.
//
// The lengths are in device memory, so every workgroup forms the plan itself
// (Plan): the positions of all columns over the workgroups the card holds at
// once give a run's length, a sequence's positions are cut into runs of about
// that many, and blockIdx.x is looked up in the running number of items.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged.hpp"
#include "wave.hpp"

namespace em {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kCols = 16;       // columns of a narrow item, and of a unit of partials
constexpr int kWideCols = 128;  // columns of a wide one
// Sequences of more columns than this take wide items: us at 48 / 32 / 16, five
// of 32 to 40 rows of 32 heads (fp32, 1456 positions) 193 / 125 / 126, 47 of 5 to
// 6 rows of 24 heads on 8 (fp16, 4927 positions) 239 / 235 / 346.
constexpr int kNarrowMost = 32;
constexpr int kStep = 32;       // positions a wave takes at a time
constexpr int kWaves = 4;
constexpr int kMinRun = 128;    // positions of a narrow item at least: one step a wave
constexpr uint32_t kNoSlot = 0xffffffffu;

struct PagedAttnArgs {
    PagedArgs p;
    const float* q;
    const void *kc, *vc;
    float* out;
    long long q_stride, out_stride;
    float scale2;  // scale times log2 e: weights are 2^(x - max)
    int window;
    int wide;       // sequences may take wide items
    int slots;      // workgroups to spread the positions over
    int min_wide;   // positions of a wide item at least
    float wide_cost;  // what a position costs a wide item, in a narrow one's
    float* part_o;  // [unit][16 columns][head_size], a unit an item's 16 columns
    float2* part_ml;
    int part_units;
};

// --- the plan -----------------------------------------------------------------

// What a sequence asks for, from the batch's arrays.
struct SeqWork {
    int row0, n;         // its rows
    int p0;              // position of the first of them
    int first, end;      // positions that any row sees
    int width, tiles;    // columns of a tile; tiles of a kv head
    int span;            // positions of a tile, at most
};

__device__ __forceinline__ SeqWork seq_work(const PagedAttnArgs& a, int s) {
    const PagedArgs& p = a.p;
    SeqWork w;
    w.row0 = p.row_start[s];
    const int r1 = p.row_start[s + 1];
    w.n = rows_exist(p, w.row0, r1) ? r1 - w.row0 : 0;
    const int len = max(p.lengths[s], -(1 << 29));
    const int cap = p.page_size * p.max_pages;
    w.p0 = len - w.n;
    w.end = min(max(len, 0), cap);
    w.first = a.window ? min(w.end, max(0, w.p0 + 1 - a.window)) : 0;
    w.width = a.wide && w.n * p.group > kNarrowMost ? kWideCols : kCols;
    w.tiles = (w.n * p.group + w.width - 1) / w.width;
    w.span = max(1, w.end - w.first);
    if (a.window) w.span = min(w.span, a.window + (w.width + p.group - 1) / p.group);
    return w;
}

// The work of a lane's sequence of 64, kept from one pass over them to the next
// (all of a batch of up to 64 is then read once).
struct LaneWork {
    SeqWork w;
    int at = -1;
    __device__ __forceinline__ const SeqWork& of(const PagedAttnArgs& a, int s0) {
        if (at != s0) {
            const int s = s0 + static_cast<int>(threadIdx.x) % kWave;
            w = s < a.p.n_seqs ? seq_work(a, s) : SeqWork{};
            at = s0;
        }
        return w;
    }
};

// What all columns' positions cost over the slots. Narrow items take half of that where a
// sequence would be only a few of them: rounding leaves items of up to one and
// a half lengths, which twice as many even out (64 sequences of 500 to 4000
// positions 167 / 146 us, 2 of 100000 189 / 195; a cut costs a wide item its
// queries' terms again, 2048 rows at 8148 717 / 752).
// No contraction: both kernels have to come to the same plan.
struct RunLength {
    float narrow, wide;
};
__device__ __forceinline__ RunLength run_length(const PagedAttnArgs& a, LaneWork& lanes) {
#pragma clang fp contract(off)
    float total = 0.0f, tiles = 0.0f;
    for (int s0 = 0; s0 < a.p.n_seqs; s0 += kWave) {
        const SeqWork& w = lanes.of(a, s0);
        const float n = static_cast<float>(w.tiles);
        const float t = n * static_cast<float>(w.span) * (w.width == kWideCols ? a.wide_cost : 1.0f);
        total += last_lane(wave_scan(t));
        tiles += last_lane(wave_scan(n));
    }
    const float kv = static_cast<float>(a.p.n_kv_heads), slots = static_cast<float>(a.slots);
    const float run = total * kv / slots;
    const float part = tiles * kv * 16.0f > slots ? 0.5f : 1.0f;
    return {fmaxf(run * part, static_cast<float>(kMinRun)),
            fmaxf(run / a.wide_cost, static_cast<float>(a.min_wide))};
}

// Runs of a sequence: its positions over a run's length, to the nearest whole
// number.
__device__ __forceinline__ int runs_of(const SeqWork& w, const RunLength& run) {
#pragma clang fp contract(off)
    const float n = static_cast<float>(w.span) / (w.width == kWideCols ? run.wide : run.narrow);
    return max(1, min(1 << 16, static_cast<int>(n + 0.5f)));
}

// Where a sequence's items and partials are. Items of wide sequences come
// first: they take longest and the narrow ones fill in beside and behind them.
// Sequences of one run need no partials, and none is split past the partials'
// memory.
struct Found {
    int seq, runs, item0, unit0;
    SeqWork w;
};
// By wave: the sequence for which hit(s, items before, items of it) holds.
template <class Hit>
__device__ __forceinline__ bool find(const PagedAttnArgs& a, LaneWork& lanes, const RunLength& run,
                                     Hit hit, Found& f) {
    const int lane = threadIdx.x % kWave;
    int items = 0, units = 0;
    for (int width = a.wide ? kWideCols : kCols; width; width = width == kWideCols ? kCols : 0) {
        for (int s0 = 0; s0 < a.p.n_seqs; s0 += kWave) {
            const SeqWork& w = lanes.of(a, s0);
            const int cells = w.width == width ? w.tiles * a.p.n_kv_heads : 0;
            int runs = runs_of(w, run);
            // Units by the runs wanted; a sequence that would pass the partials'
            // memory stays whole (its units stay counted: all after it do too).
            const int want = runs > 1 ? cells * runs * (width / kCols) : 0;
            const int ahead = units + wave_scan(want) - want;
            if (ahead + want > a.part_units) runs = min(runs, 1);
            const int mine = cells * runs;
            const int before = items + wave_scan(mine) - mine;
            const unsigned long long got = __ballot(mine > 0 && hit(s0 + lane, before, mine));
            if (got) {
                const int src = __ffsll(got) - 1;
                auto its = [&](int v) { return __builtin_amdgcn_readlane(v, src); };
                f.seq = s0 + src;
                f.runs = its(runs);
                f.item0 = its(before);
                f.unit0 = its(ahead);
                f.w.row0 = its(w.row0);
                f.w.n = its(w.n);
                f.w.p0 = its(w.p0);
                f.w.first = its(w.first);
                f.w.end = its(w.end);
                f.w.width = width;
                f.w.tiles = its(w.tiles);
                return true;
            }
            items = last_lane(before + mine);
            units = last_lane(ahead + want);
        }
    }
    return false;
}

// --- types ----------------------------------------------------------------------

// The MFMA terms of each cache type. Queries and weights are fp32, so each is
// held as a sum of 16-bit terms and the products are added in fp32:
//   bf16 caches: three bf16 terms, exact down to 2^-109, times the value as it
//     is: three products.
//   fp32 caches: both sides three bf16 terms; the three products of the
//     smallest (below 2^-24 of the whole) are left out: six products.
//   fp16 caches: two fp16 terms of a column scaled to a largest query value
//     of 2^14 (weights: 2^14 for 1), off by 2^-22 of the value or, where that is
//     more, 2^-39 of the largest; fp16 keys and values are at most 2^16: two
//     products. Of queries the second is held below 2^-20 in a score (small_dims),
//     of weights it is 2^-39 of a value each.
template <class T>
struct Ops;

template <>
struct Ops<__bf16> {
    using Frag = bf16x8;
    static constexpr int kTerms = 3, kCacheTerms = 1;
    static constexpr float kWeight = 1.0f;
};
template <>
struct Ops<float> {
    using Frag = bf16x8;
    static constexpr int kTerms = 3, kCacheTerms = 3;
    static constexpr float kWeight = 1.0f;
};
template <>
struct Ops<_Float16> {
    using Frag = f16x8;
    static constexpr int kTerms = 2, kCacheTerms = 1;
    static constexpr float kWeight = 16384.0f;
};

typedef float floatx16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ floatx4 mma(f16x8 a, f16x8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mma(bf16x8 a, bf16x8 b, floatx4 c) {
    return mfma16x16x32(a, b, c);
}
__device__ __forceinline__ floatx16 mma(f16x8 a, f16x8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mma(bf16x8 a, bf16x8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

typedef short bf16x4 __attribute__((ext_vector_type(4)));  // bits of four bf16
__device__ __forceinline__ floatx4 mma(bf16x4 a, bf16x4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
}
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
// (a, b) rounded to nearest bf16, a in the low half. A conversion that the
// compiler knows: the terms go straight into MFMAs, and it keeps the wait states
// that an MFMA needs behind a VALU write, which it does not behind inline asm.
__device__ __forceinline__ uint32_t pair_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, bf16x2));
}
// N fp32 values as three terms of N bf16, each the remainder so far rounded to
// nearest: their sum is v exactly for |v| >= 2^-109. `lost` gets bits in its low
// half when a last term is not the whole remainder.
template <int N, class F>
__device__ __forceinline__ void split_terms(const float (&v)[N], F (&t)[3], uint32_t& lost) {
#pragma clang fp contract(off)
    typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
    words w[3];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            w[n][i] = pair_bf16(a, b);
            if (n == 2) break;
            a -= from_bits(w[n][i] << 16);
            b -= from_bits(w[n][i] & 0xffff0000u);
            if (n == 1) lost |= bits(a) | bits(b);
        }
    }
#pragma unroll
    for (int n = 0; n < 3; ++n) t[n] = __builtin_bit_cast(F, w[n]);
}
__device__ __forceinline__ void split_terms(const float (&v)[8], f16x8 (&t)[2], uint32_t&) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        t[0][e] = static_cast<_Float16>(v[e]);
        t[1][e] = static_cast<_Float16>(v[e] - static_cast<float>(t[0][e]));
    }
}

// What two fp16 terms leave of the values past 2^-22 of each: of those so far
// below a column's largest that their second term is subnormal. bf16's terms say
// by `lost` what they leave.
template <class F, int NT>
__device__ __forceinline__ float small_dims(const float (&)[8], const F (&)[NT]) {
    return 0.0f;
}
__device__ __forceinline__ float small_dims(const float (&v)[8], const f16x8 (&t)[2]) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float left =
            fabsf(v[e] - static_cast<float>(t[0][e]) - static_cast<float>(t[1][e]));
        sum += left > 0x1p-22f * fabsf(v[e]) ? left : 0.0f;
    }
    return sum;
}
// The score that a column's left bits make at most with keys of 65504, in log2
// units, may be 2^-20 (fp32's rounding of a score of 16); a column that may pass it is
// done plainly. A query of ordinary size (largest dim times scale log2 e below 2)
// passes with eight such dims.
constexpr float kMostLeft = 0x1p-20f / 65504.0f;

// 16-bit caches are loaded as they are (four dwords for eight values), fp32 as
// two vectors.
template <class T>
struct Raw8 {
    uint4 x;
    __device__ void load(const T* p) { x = *reinterpret_cast<const uint4*>(p); }
    __device__ void zero() { x = make_uint4(0, 0, 0, 0); }
};
template <>
struct Raw8<float> {
    float v[8];
    __device__ void load(const float* p) {
        const floatx4 a = *reinterpret_cast<const floatx4*>(p);
        const floatx4 b = *reinterpret_cast<const floatx4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    }
    __device__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
};

__device__ __forceinline__ uint32_t word(const uint4& x, int i) {
    return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w;
}

// d += A x B over the pairs of terms kept.
template <class F, int NT, class D>
__device__ __forceinline__ void mma_terms(const F (&k)[1], const F (&q)[NT], D& d) {
#pragma unroll
    for (int t = NT - 1; t >= 0; --t) d = mma(k[0], q[t], d);
}
template <class F, class D>
__device__ __forceinline__ void mma_terms(const F (&k)[3], const F (&q)[3], D& d) {
    d = mma(k[2], q[0], d);
    d = mma(k[1], q[1], d);
    d = mma(k[0], q[2], d);
    d = mma(k[1], q[0], d);
    d = mma(k[0], q[1], d);
    d = mma(k[0], q[0], d);
}

// --- one column, plainly ------------------------------------------------------------

// The slot of position t in units of eight elements, or kNoSlot.
__device__ __forceinline__ uint32_t slot_unit(const PagedArgs& p, int seq, int t) {
    const long long off = slot_offset(p, seq, t);
    return off < 0 ? kNoSlot : static_cast<uint32_t>(off >> 3);
}

template <class T>
struct __attribute__((aligned(16))) Eight {
    T v[8];
};

// One wave, one column over positions lo .. lo + width - 1 of every stride
// before hi, in fp32 operations on what the column sees alone: for columns
// whose operands the terms do not hold, and for those beside a position that
// is not finite and that they do not see (its zero weight would not hide it).
// m, l: maximum (of log2 weights) and sum; o[i]: head dim lane + 64 i,
// unnormalised. Where a sum passes kLargest they are formed again with m higher by
// 60: the same weights, l and o 2^60 lower, so that the sums behind a mean of values
// near fp32's largest are finite, here and when runs are added.
constexpr float kLargest = 0x1p100f;  // 2^18 runs and waves of it still add up
template <class T, int N>
__device__ __forceinline__ void plain_column(const PagedAttnArgs& a, int seq, int row, int head,
                                          int pq, int lo, int hi, int width, int stride, float& m,
                                          float& l,
                                          float (&o)[N]) {
    const PagedArgs& p = a.p;
    const int lane = threadIdx.x % kWave, D = p.head_size;
    const float* q = a.q + row * a.q_stride + head * D;
    const long long hoff = (head / p.group) * p.head_stride;
    const T* kc = static_cast<const T*>(a.kc) + hoff;
    const T* vc = static_cast<const T*>(a.vc) + hoff;
    float pre = 1.0f;  // on the weights of o
    while (true) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = 0.0f;
        for (int t0 = lo; t0 < hi; t0 += stride) {
            const int t = t0 + lane;
            uint32_t unit = kNoSlot;
            if (lane < width && t < hi && t <= pq && !(a.window && t <= pq - a.window))
                unit = slot_unit(p, seq, t);
            float x = -INFINITY;
            if (unit != kNoSlot) {
                const T* k = kc + static_cast<std::size_t>(unit) * 8;
                float dot = 0.0f;
                for (int d = 0; d < D; d += 8) {
                    const auto y = *reinterpret_cast<const Eight<T>*>(k + d);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot = fmaf(q[d + e], static_cast<float>(y.v[e]), dot);
                }
                x = dot * a.scale2;
            }
            const float mn = fmaxf(m, wave_max(x));
            const float alpha = mn == -INFINITY ? 1.0f : exp2f(m - mn);
            const float w = unit == kNoSlot || x == -INFINITY ? 0.0f : exp2f(x - mn);
            m = mn;
            l = l * alpha + wave_sum(w);
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] *= alpha;
            // Eight positions' values in flight; those not seen read slot 0 and count
            // for nothing, whatever it holds.
            for (int i = 0; i < width; i += 8) {
                float v[8][N], wi[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t u = __shfl(unit, i + e, kWave);
                    wi[e] = __shfl(w * pre, i + e, kWave);
                    const T* src = vc + static_cast<std::size_t>(u == kNoSlot ? 0 : u) * 8;
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        const float y = static_cast<float>(src[min(lane + kWave * n, D - 1)]);
                        v[e][n] = u == kNoSlot ? 0.0f : y;
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int n = 0; n < N; ++n) o[n] = fmaf(wi[e], v[e][n], o[n]);
            }
        }
        if (std::is_same_v<T, _Float16>) break;  // at most 2^46
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(o[i]));
        if (pre < 1.0f || !(wave_max(top) >= kLargest)) break;
        pre = 0x1p-60f;
    }
    if (pre < 1.0f) {
        // m + 60 is rounded; what that adds to 60 the weights leave off again.
        const float raised = m + 60.0f;
        const double off = static_cast<double>(m) - static_cast<double>(raised) + 60.0;
        const float by = __builtin_amdgcn_exp2f(static_cast<float>(off));
        m = raised;
        l *= by * pre;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] *= by;
    }
}

// --- 16 columns ---------------------------------------------------------------------

// An item: 16 columns over positions [lo, hi), its four waves taking every
// fourth 32 of them. In lane (g, j) of a wave, per 32 positions:
//  * S^T = K Q^T: position j (16 + j) of the first operand, head dims 8g .. of
//    each 32, loaded from the cache as the MFMA takes them; Q's terms stay in
//    registers.
//  * The lane ends with column j's scores at positions 4g + r and 16 + 4g + r:
//    its eight k values of O^T += V^T P^T once V's operand takes positions in
//    that order.
//  * V: a lane loads VU head dims VU j .. of its eight positions, 256 bytes of
//    a position by 16 lanes, and eight-position columns of them are put
//    together by byte permutes (fp32: by the split).
//  * O^T: column j, head dims VU (4g + r) + u.
// Nothing is staged in LDS: 16 KB a wave are in flight (keys are loaded again
// right after their product, values after theirs), which 8 waves a CU need to
// keep HBM busy. Bound by the cache's bytes: 64 rows at 500 to 4000 positions (32
// heads on 8 of 128, bf16) 136 us for 641 MB, 2 at 70001 to 131070 (fp16) 171 us
// for 954 MB.
template <class T, int DP>
struct Few {
    static constexpr int C = DP / 32, VU = DP / 16, NV = (VU + 7) / 8;
    using O = Ops<T>;
    // Positions of a step, and of them those whose values a lane holds.
    static constexpr int KS = O::kCacheTerms == 3 ? 16 : 32, NE = KS / 4;
    using Frag = typename O::Frag;
    static constexpr int NT = O::kTerms, KT = O::kCacheTerms;
    static constexpr int kQueryAt = kWaves * kCols * ((DP + 4) * 4 + 8);
    static constexpr bool kQueryLds = NT == 3;
    static constexpr int kLds = kQueryAt + (kQueryLds ? C * NT * kWave * 16 : 0);
};

// A 16-bit value operand: element u of eight positions.
template <class F, class T, int NV>
__device__ __forceinline__ void value_terms(const Raw8<T> (&v)[8][NV], int u, F (&t)[1], uint32_t&) {
    const uint32_t sel = u & 1 ? 0x07060302u : 0x05040100u;
    const int n = u / 8, wd = (u % 8) / 2;
    uint4 x;
    x.x = __builtin_amdgcn_perm(word(v[1][n].x, wd), word(v[0][n].x, wd), sel);
    x.y = __builtin_amdgcn_perm(word(v[3][n].x, wd), word(v[2][n].x, wd), sel);
    x.z = __builtin_amdgcn_perm(word(v[5][n].x, wd), word(v[4][n].x, wd), sel);
    x.w = __builtin_amdgcn_perm(word(v[7][n].x, wd), word(v[6][n].x, wd), sel);
    t[0] = __builtin_bit_cast(F, x);
}
template <int NV>
__device__ __forceinline__ void value_terms(const Raw8<float> (&v)[4][NV], int u, bf16x4 (&t)[3],
                                            uint32_t& lost) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = v[e][u / 8].v[u % 8];
    split_terms(x, t, lost);
}
template <class F, class T>
__device__ __forceinline__ void key_terms(const Raw8<T>& k, F (&t)[1]) {
    t[0] = __builtin_bit_cast(F, k.x);
}
template <class F>
__device__ __forceinline__ void key_terms(const Raw8<float>& k, F (&t)[3]) {
    uint32_t lost = 0;  // a query too large for it to matter is found with the query
    split_terms(k.v, t, lost);
}

// The operands of O^T += V^T P^T: as many positions a lane as a step has.
template <class F, int NE>
struct WeightFrag {
    using type = F;
};
template <class F>
struct WeightFrag<F, 4> {
    using type = bf16x4;
};

// An item of the plan: columns [col0, col0 + cols) of kv head kvh of the
// found sequence over positions [lo, hi), its partials' first unit.
struct Item {
    Found f;
    int kvh, col0, cols, lo, hi, unit;
};

template <class T, int DP>
__device__ __forceinline__ void narrow_item(const PagedAttnArgs& a, const Item& it, char* smem) {
    using F = Few<T, DP>;
    constexpr int C = F::C, VU = F::VU, NV = F::NV, NT = F::NT, KT = F::KT;
    constexpr int KS = F::KS, NE = F::NE, NY = KS / 16;
    constexpr int kRow = DP + 4;  // floats of a column in LDS
    // The waves' outputs; before them the query terms of fp32 caches, whose
    // keys and values take the registers (148 spilled with them): they are the
    // same in every wave.
    auto* o_s = reinterpret_cast<float(*)[kCols][kRow]>(smem);
    auto* ml_s = reinterpret_cast<float2(*)[kCols]>(smem + sizeof(float) * kWaves * kCols * kRow);
    constexpr bool kQueryLds = F::kQueryLds;
    auto* q_s = reinterpret_cast<typename F::Frag*>(smem + F::kQueryAt);
    const PagedArgs& p = a.p;
    const int tid = threadIdx.x, lane = tid % kWave, g = lane >> 4, j = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int D = p.head_size;
    const Found& f = it.f;
    const int kvh = it.kvh, cols = it.cols, lo = it.lo, hi = it.hi;
    const int col = it.col0 + min(j, cols - 1);
    const int i = col / p.group, row = f.w.row0 + i, head = kvh * p.group + col % p.group;
    const int pq = f.w.p0 + i;
    const int i0 = it.col0 / p.group, i1 = (it.col0 + cols - 1) / p.group;
    // Every column sees positions [all_lo, all_hi].
    const int all_lo = a.window ? f.w.p0 + i1 + 1 - a.window : 0, all_hi = f.w.p0 + i0;

    // The column's query terms.
    typename F::Frag q[kQueryLds ? 1 : C][NT];
    uint32_t lost_q = 0, lost_v = 0;
    float top_q = 0.0f, unscale = 1.0f, left_q = 0.0f;
    {
        float v[C][8];
        const float* src = a.q + row * a.q_stride + head * D;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = 32 * c + 8 * g;
            const bool in = d < D;
            const floatx4 x0 = *reinterpret_cast<const floatx4*>(src + (in ? d : 0));
            const floatx4 x1 = *reinterpret_cast<const floatx4*>(src + (in ? d : 0) + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[c][e] = in ? x0[e] * a.scale2 : 0.0f;
                v[c][4 + e] = in ? x1[e] * a.scale2 : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) top_q = fmaxf(top_q, fabsf(v[c][e]));
        }
        top_q = max32(max16(top_q));
        if constexpr (NT == 2) {
            // To a largest value of 2^14 .. 2^15.
            const int ex = top_q > 0.0f && top_q < INFINITY ? 14 - ilogbf(top_q) : 0;
            const float up = ldexpf(1.0f, min(ex, 120));
            unscale = ldexpf(1.0f, -min(ex, 120));
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] *= up;
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            split_terms(v[c], q[kQueryLds ? 0 : c], lost_q);
            left_q += small_dims(v[c], q[kQueryLds ? 0 : c]);
            if (kQueryLds && w == 0) {
#pragma unroll
                for (int t = 0; t < NT; ++t) q_s[(c * NT + t) * kWave + lane] = q[0][t];
            }
        }
        if (kQueryLds) __syncthreads();
    }
    // fp32 keys below 2^-109 drop bits worth up to 2^-134 each: nothing for a
    // query below 2^90. fp16's scale reaches down to 2^-106.
    bool bad = KT == 3   ? (lost_q & 0xffffu) != 0 || !(top_q < 0x1p90f)
               : NT == 3 ? (lost_q & 0xffffu) != 0
                         : top_q != 0.0f && !(top_q >= 0x1p-100f && top_q < INFINITY);
    if constexpr (NT == 2) bad |= sum32(sum16(left_q)) * unscale > kMostLeft;

    const T* kc = static_cast<const T*>(a.kc) + kvh * p.head_stride;
    const T* vc = static_cast<const T*>(a.vc) + kvh * p.head_stride;
    // Lane l holds position l % KS of a step. Positions that are not there
    // read slot 0 and count for nothing.
    auto units = [&](int t0) {
        const int t = t0 + (lane & (KS - 1));
        return t < hi ? slot_unit(p, f.seq, t) : kNoSlot;
    };
    auto place = [&](int e) { return 4 * g + (e < 4 ? e : 12 + e); };  // of a lane's e-th position
    using Values = Raw8<T>[NE][NV];
    Raw8<T> k[NY][C];
    auto load_k = [&](uint32_t u) {
#pragma unroll
        for (int y = 0; y < NY; ++y) {
            const uint32_t x = __shfl(u, 16 * y + j, kWave);
            const T* src = kc + static_cast<std::size_t>(x == kNoSlot ? 0 : x) * 8;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int d = 32 * c + 8 * g;
                k[y][c].load(src + (d < D ? d : 0));
            }
        }
    };
    auto load_v = [&](uint32_t u, Values& v) {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const uint32_t x = __shfl(u, place(e), kWave);
            const T* src = vc + static_cast<std::size_t>(x == kNoSlot ? 0 : x) * 8;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int d = VU * j + 8 * n;
                if constexpr (VU == 4) {
                    // Four head dims a lane: half a vector.
                    const T* s4 = src + (d < D ? d : 0);
                    if constexpr (sizeof(T) == 4) {
                        const floatx4 y = *reinterpret_cast<const floatx4*>(s4);
#pragma unroll
                        for (int z = 0; z < 4; ++z) v[e][n].v[z] = y[z];
                    } else {
                        const uint2 y = *reinterpret_cast<const uint2*>(s4);
                        v[e][n].x = make_uint4(y.x, y.y, 0, 0);
                    }
                } else {
                    v[e][n].load(src + (d < D ? d : 0));
                }
            }
        }
    };

    float m = -INFINITY, l = 0.0f;
    floatx4 o[VU];
#pragma unroll
    for (int u = 0; u < VU; ++u) o[u] = floatx4{0.f, 0.f, 0.f, 0.f};

    constexpr int kStride = KS * kWaves;
    int t0 = lo + w * KS;
    uint32_t u = kNoSlot;
    // One step with its values in v; the next one's keys are loaded after the
    // scores, its values into vn before them or, where vn is v, after their
    // products. False: it was the last.
    auto step = [&](Values& v, Values& vn, auto ahead) {
        const uint32_t un = units(t0 + kStride);
        const bool more = t0 + kStride < hi;
        if (ahead && more) load_v(un, vn);
        floatx4 s[NY];
#pragma unroll
        for (int y = 0; y < NY; ++y) {
            s[y] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                typename F::Frag kt[KT];
                key_terms(k[y][c], kt);
                if constexpr (kQueryLds) {
                    typename F::Frag qt[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) qt[t] = q_s[(c * NT + t) * kWave + lane];
                    mma_terms(kt, qt, s[y]);
                } else {
                    mma_terms(kt, q[c], s[y]);
                }
            }
        }
        if (more) load_k(un);
        float x[NE];
#pragma unroll
        for (int e = 0; e < NE; ++e) x[e] = NT == 2 ? s[e / 4][e % 4] * unscale : s[e / 4][e % 4];
        // Positions that are there, of the step's.
        constexpr uint32_t kAll = KS == 32 ? 0xffffffffu : (1u << (KS & 31)) - 1;
        const uint32_t there = static_cast<uint32_t>(__ballot(u != kNoSlot)) & kAll;
        if (there != kAll || t0 < all_lo || t0 + KS - 1 > all_hi) {
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                const int r = place(e), t = t0 + r;
                const bool seen = (there >> r & 1) && t <= pq && !(a.window && t <= pq - a.window);
                x[e] = seen ? x[e] : -INFINITY;
            }
            if (there != kAll) {
#pragma unroll
                for (int e = 0; e < NE; ++e)
                    if (!(there >> place(e) & 1)) {
#pragma unroll
                        for (int n = 0; n < NV; ++n) v[e][n].zero();
                    }
            }
        }
        float mb = x[0];
#pragma unroll
        for (int e = 1; e < NE; ++e) mb = fmaxf(mb, x[e]);
        const float mn = fmaxf(m, max32(max16(mb)));
        if (__ballot(mn > m)) {
            const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
#pragma unroll
            for (int y = 0; y < VU; ++y) o[y] *= alpha;
            m = mn;
        }
        const float base = mn == -INFINITY ? 0.0f : mn;
        float pw[NE];
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            pw[e] = __builtin_amdgcn_exp2f(x[e] - base);
            l += pw[e];
            pw[e] *= F::O::kWeight;
        }
        typename WeightFrag<typename F::Frag, NE>::type pt[NT];
        uint32_t lost_p = 0;
        split_terms(pw, pt, lost_p);
#pragma unroll
        for (int y = 0; y < VU; ++y) {
            typename WeightFrag<typename F::Frag, NE>::type vt[KT];
            value_terms(v, y, vt, lost_v);
            mma_terms(vt, pt, o[y]);
        }
        if (!more) return false;
        if (!ahead) load_v(un, vn);
        u = un;
        t0 += kStride;
        return true;
    };
    if (t0 < hi) {
        Raw8<T> v[NE][NV];
        u = units(t0);
        load_k(u);
        load_v(u, v);
        if constexpr (KT == 3 && DP <= 128) {
            Raw8<T> v2[NE][NV];
            while (step(v, v2, std::true_type{}) && step(v2, v, std::true_type{})) {
            }
        } else {
            while (step(v, v, std::false_type{})) {
            }
        }
    }
    l = sum32(sum16(l));
    constexpr float kMost = NT == 3 ? kLargest : INFINITY;  // fp16's sums stay below 2^61
    float low = INFINITY;
#pragma unroll
    for (int y = 0; y < VU; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = VU * (4 * g + r) + y;
            const float x = fabsf(o[y][r]);
            bad |= d < D && !(x < kMost);
            low = d < D ? fminf(low, x) : low;
        }
    // fp32 values that dropped bits, worth up to 2^-134 each, beside a sum so
    // small that it could show.
    if constexpr (KT == 3) bad |= __ballot((lost_v & 0xffffu) != 0) != 0 && low < 0x1p-50f;
    bad |= !(l < INFINITY);
    // A column's lanes together.
    unsigned long long redo = __ballot(bad);
    redo |= redo >> 32;
    redo = (redo | redo >> 16) & 0xffffu;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int y = 0; y < VU; ++y)
            o_s[w][j][VU * (4 * g + r) + y] = o[y][r] * (1.0f / F::O::kWeight);
    if (g == 0) ml_s[w][j] = make_float2(m, l);
    while (redo) {
        const int c = __ffsll(redo) - 1;
        redo &= redo - 1;
        float po[DP / kWave], pm, pl;
        plain_column<T, DP / kWave>(a, f.seq, __shfl(row, c, kWave), __shfl(head, c, kWave),
                                    __shfl(pq, c, kWave), lo + w * KS, hi, KS, kStride, pm, pl, po);
#pragma unroll
        for (int n = 0; n < DP / kWave; ++n) o_s[w][c][lane + kWave * n] = po[n];
        if (lane == 0) ml_s[w][c] = make_float2(pm, pl);
    }
    __syncthreads();

    // The four waves' sums, in wave order.
    for (int x = tid; x < cols * (D / 4); x += kThreads) {
        const int c = x / (D / 4), d = x % (D / 4) * 4;
        float mm = -INFINITY, ll = 0.0f;
#pragma unroll
        for (int y = 0; y < kWaves; ++y) mm = fmaxf(mm, ml_s[y][c].x);
        floatx4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < kWaves; ++y) {
            const float2 ml = ml_s[y][c];
            // A wave whose sum is NaN has no maximum to go by.
            const float fac = ml.x == mm || ml.y != ml.y ? 1.0f
                              : ml.x == -INFINITY        ? 0.0f
                                                         : __builtin_amdgcn_exp2f(ml.x - mm);
            ll += fac * ml.y;
            sum += fac * *reinterpret_cast<const floatx4*>(&o_s[y][c][d]);
        }
        const int cc = it.col0 + c;
        if (f.runs > 1) {
            const std::size_t pc = static_cast<std::size_t>(it.unit) * kCols + c;
            *reinterpret_cast<floatx4*>(a.part_o + pc * D + d) = sum;
            if (d == 0) a.part_ml[pc] = make_float2(mm, ll);
        } else {
            float* dst = a.out + (f.w.row0 + cc / p.group) * a.out_stride +
                         (kvh * p.group + cc % p.group) * D + d;
            *reinterpret_cast<floatx4*>(dst) = ll == 0.0f ? floatx4{0.f, 0.f, 0.f, 0.f} : sum * (1.0f / ll);
        }
    }
}

// --- 128 columns --------------------------------------------------------------------

// A wide item: 128 columns, 32 a wave, over positions [lo, hi), 32 at a time
// staged in LDS for the four waves. In lane (h, j), h = lane / 32:
//  * S^T = K Q^T, 32 positions x 32 columns: the keys from LDS, Q's terms from
//    registers (of three the last from LDS: with all in registers two
//    workgroups a CU do not fit). The 16-byte units of a key's row are permuted
//    by the key, so that 16 keys' reads of one unit fall into different banks.
//  * The lane ends with column j's scores at positions 8 (r / 4) + 4h + r % 4,
//    r < 16: per 16 positions the k values of O^T += V^T P^T, for which V's
//    operand takes the positions in that order, DP / 32 head dims of eight
//    positions read from LDS and put together by byte permutes.
//  * O^T: column j, head dims DP / 32 (8 (r / 4) + 4h + r % 4) + u.
// The next 32 positions are loaded into registers beside the products and
// written to LDS after them (fp32: split into its three terms there). Bound by
// the matrix cores, three products a multiply-add for bf16 and six for fp32,
// beside the softmax of the other workgroup on the CU: 2048 rows of 32 heads on 8
// of 128 behind 6100 positions (bf16) 667 us, 1070 TFLOP/s of products (16 columns
// an item: 1119 us).
template <class T, int DP>
struct Wide {
    using O = Ops<T>;
    using Frag = typename O::Frag;
    static constexpr int NT = O::kTerms, KT = O::kCacheTerms;
    static constexpr int C = DP / 16, DU = DP / 32;  // k steps of S; head dims a lane
    static constexpr int kRowBytes = DP * 2, kPlane = kStep * kRowBytes;
    static constexpr int kStage = 2 * KT * kPlane;  // keys' planes, then values'
    static constexpr int kBufs = 2 * kStage <= 64 * 1024 || KT == 3 ? (KT == 3 && DP > 64 ? 1 : 2) : 1;
    static constexpr bool kQueryLds = NT == 3;
    static constexpr int kQueryAt = kBufs * kStage;
    static constexpr int kLds = kQueryAt + (kQueryLds ? kWaves * C * kWave * 16 : 0);
    static_assert(kWaves * 32 * (8 * DU + 4) * 4 <= kLds);
    static constexpr int kLoads = kStep * (DP / 8) / kThreads;  // units a thread, of K and of V
};

// DU elements (DU / 2 words) of a value row for eight positions, and operand u.
template <int DU>
struct ValueRun {
    uint32_t x[DU / 2];
};

template <class T, int DP>
__device__ __forceinline__ void wide_item(const PagedAttnArgs& a, const Item& it, char* smem) {
    using W = Wide<T, DP>;
    using Frag = typename W::Frag;
    constexpr int NT = W::NT, KT = W::KT, C = W::C, DU = W::DU, L = W::kLoads;
    constexpr int NQ = W::kQueryLds ? 2 : NT;  // terms in registers
    const PagedArgs& p = a.p;
    const Found& f = it.f;
    const int tid = threadIdx.x, lane = tid % kWave, h = lane >> 5, j = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int D = p.head_size, kvh = it.kvh, lo = it.lo, hi = it.hi;
    const int wc = 32 * w;  // the wave's first column in the tile
    const bool idle = wc >= it.cols;
    const int cin = min(wc + j, it.cols - 1), col = it.col0 + cin;
    const int i = col / p.group, row = f.w.row0 + i, head = kvh * p.group + col % p.group;
    const int pq = f.w.p0 + i;
    // The wave's first and last row.
    const int i0 = (it.col0 + min(wc, it.cols - 1)) / p.group;
    const int i1 = (it.col0 + min(wc + 31, it.cols - 1)) / p.group;
    const int all_lo = a.window ? f.w.p0 + i1 + 1 - a.window : 0, all_hi = f.w.p0 + i0;
    const int wave_lo = a.window ? f.w.p0 + i0 + 1 - a.window : 0, wave_hi = f.w.p0 + i1;
    const T* kc = static_cast<const T*>(a.kc) + kvh * p.head_stride;
    const T* vc = static_cast<const T*>(a.vc) + kvh * p.head_stride;
    auto* q_s = reinterpret_cast<Frag*>(smem + W::kQueryAt) + w * C * kWave;

    // Head dims past the head size stay zero.
    if (D < DP)
        for (int x = tid; x < W::kBufs * W::kStage / 16; x += kThreads)
            reinterpret_cast<uint4*>(smem)[x] = make_uint4(0, 0, 0, 0);

    Frag q[C][NQ];
    uint32_t lost_q = 0, lost_v = 0;
    float top_q = 0.0f, unscale = 1.0f, left_q = 0.0f;
    {
        const float* src = a.q + row * a.q_stride + head * D;
        auto load = [&](int c, float (&v)[8]) {
            const int d = 16 * c + 8 * h;
            const bool in = d < D;
            const floatx4 x0 = *reinterpret_cast<const floatx4*>(src + (in ? d : 0));
            const floatx4 x1 = *reinterpret_cast<const floatx4*>(src + (in ? d : 0) + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = in ? x0[e] * a.scale2 : 0.0f;
                v[4 + e] = in ? x1[e] * a.scale2 : 0.0f;
            }
        };
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float v[8];
            load(c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) top_q = fmaxf(top_q, fabsf(v[e]));
            if constexpr (NT == 3) {
                Frag t[3];
                split_terms(v, t, lost_q);
                q[c][0] = t[0];
                q[c][1] = t[1];
                if constexpr (W::kQueryLds)
                    q_s[c * kWave + lane] = t[2];
                else
                    q[c][2] = t[2];
            }
        }
        top_q = max32(top_q);
        if constexpr (NT == 2) {
            // To a largest value of 2^14 .. 2^15.
            const int ex = top_q > 0.0f && top_q < INFINITY ? min(120, 14 - ilogbf(top_q)) : 0;
            const float up = ldexpf(1.0f, ex);
            unscale = ldexpf(1.0f, -ex);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float v[8];
                load(c, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= up;
                split_terms(v, q[c], lost_q);
                left_q += small_dims(v, q[c]);
            }
        }
    }
    bool bad = KT == 3   ? (lost_q & 0xffffu) != 0 || !(top_q < 0x1p90f)
               : NT == 3 ? (lost_q & 0xffffu) != 0
                         : top_q != 0.0f && !(top_q >= 0x1p-100f && top_q < INFINITY);
    if constexpr (NT == 2) bad |= sum32(left_q) * unscale > kMostLeft;

    // Unit x = tid + 256 y of a stage: position x / (DP / 8), head dims 8 (x % (DP / 8)).
    constexpr int UR = DP / 8;
    Raw8<T> kr[L], vr[L];
    auto load = [&](uint32_t units) {
#pragma unroll
        for (int y = 0; y < L; ++y) {
            const int x = tid + kThreads * y, c = x % UR;
            const uint32_t u = __shfl(units, x / UR, kWave);
            if (8 * c < D) {
                const std::size_t at = static_cast<std::size_t>(u == kNoSlot ? 0 : u) * 8 + 8 * c;
                kr[y].load(kc + at);
                vr[y].load(vc + at);
            }
        }
    };
    auto permuted = [](int key, int c) {
        return c ^ (DP == 64 ? (key >> 1) & 7 : key & 15);
    };
    auto store = [&](uint32_t there, char* buf) {
#pragma unroll
        for (int y = 0; y < L; ++y) {
            const int x = tid + kThreads * y, c = x % UR, key = x / UR;
            if (8 * c < D) {
                if (!(there >> key & 1)) vr[y].zero();
                char* kd = buf + key * W::kRowBytes + permuted(key, c) * 16;
                char* vd = buf + KT * W::kPlane + key * W::kRowBytes + c * 16;
                Frag t[KT];
                key_terms(kr[y], t);
#pragma unroll
                for (int n = 0; n < KT; ++n) *reinterpret_cast<Frag*>(kd + n * W::kPlane) = t[n];
                if constexpr (KT == 3)
                    split_terms(vr[y].v, t, lost_v);
                else
                    key_terms(vr[y], t);
#pragma unroll
                for (int n = 0; n < KT; ++n) *reinterpret_cast<Frag*>(vd + n * W::kPlane) = t[n];
            }
        }
    };
    // Lane l holds the slot of position t0 + l % 32; the stage's positions that
    // are there.
    auto look = [&](int t0) {
        const int t = t0 + j;
        return t < hi ? slot_unit(p, f.seq, t) : kNoSlot;
    };
    auto mask = [](uint32_t units) { return static_cast<uint32_t>(__ballot(units != kNoSlot)); };

    float m = -INFINITY, l = 0.0f;
    floatx16 o[DU];
#pragma unroll
    for (int u = 0; u < DU; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[u][r] = 0.0f;

    auto use = [&](int t0, uint32_t there, const char* buf) {
        floatx16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            Frag k[KT], qt[NT];
#pragma unroll
            for (int n = 0; n < KT; ++n)
                k[n] = *reinterpret_cast<const Frag*>(buf + n * W::kPlane + j * W::kRowBytes +
                                                      permuted(j, 2 * c + h) * 16);
#pragma unroll
            for (int n = 0; n < NQ; ++n) qt[n] = q[c][n];
            if constexpr (W::kQueryLds) qt[2] = q_s[c * kWave + lane];
            mma_terms(k, qt, s);
        }
        if constexpr (NT == 2) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= unscale;
        }
        if (there != 0xffffffffu || t0 < all_lo || t0 + kStep - 1 > all_hi) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int x = 8 * (r / 4) + 4 * h + r % 4, t = t0 + x;
                const bool seen = (there >> x & 1) && t <= pq && !(a.window && t <= pq - a.window);
                s[r] = seen ? s[r] : -INFINITY;
            }
        }
        float mb = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mb = fmaxf(mb, s[r]);
        const float mn = fmaxf(m, max32(mb));
        if (__ballot(mn > m)) {
            const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
#pragma unroll
            for (int u = 0; u < DU; ++u) o[u] *= alpha;
            m = mn;
        }
        const float base = mn == -INFINITY ? 0.0f : mn;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            float pw[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                pw[e] = __builtin_amdgcn_exp2f(s[8 * y + e] - base);
                l += pw[e];
                pw[e] *= W::O::kWeight;
            }
            Frag pt[NT];
            uint32_t lost_p = 0;
            split_terms(pw, pt, lost_p);
            // A plane at a time, the smallest first.
#pragma unroll
            for (int n = KT - 1; n >= 0; --n) {
                ValueRun<DU> v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = *reinterpret_cast<const ValueRun<DU>*>(
                        buf + (KT + n) * W::kPlane +
                        (16 * y + 4 * h + (e < 4 ? e : 4 + e)) * W::kRowBytes + j * DU * 2);
#pragma unroll
                for (int u = 0; u < DU; ++u) {
                    const uint32_t sel = u & 1 ? 0x07060302u : 0x05040100u;
                    uint4 x;
                    x.x = __builtin_amdgcn_perm(v[1].x[u / 2], v[0].x[u / 2], sel);
                    x.y = __builtin_amdgcn_perm(v[3].x[u / 2], v[2].x[u / 2], sel);
                    x.z = __builtin_amdgcn_perm(v[5].x[u / 2], v[4].x[u / 2], sel);
                    x.w = __builtin_amdgcn_perm(v[7].x[u / 2], v[6].x[u / 2], sel);
                    const Frag vt = __builtin_bit_cast(Frag, x);
#pragma unroll
                    for (int t = NT - 1 - n; t >= 0; --t) o[u] = mma(vt, pt[t], o[u]);
                }
            }
        }
    };

    if (lo < hi) {
        uint32_t units = look(lo), next = look(lo + kStep);
        if (D < DP) __syncthreads();  // the zeros
        load(units);
        store(mask(units), smem);
        for (int t0 = lo, s = 0; t0 < hi; t0 += kStep, ++s) {
            char* buf = smem + (W::kBufs == 2 ? (s & 1) * W::kStage : 0);
            __syncthreads();  // this stage is in LDS, the one before has been read
            const bool more = t0 + kStep < hi;
            const uint32_t there = mask(units);
            units = next;
            if (more) load(units);
            next = look(t0 + 2 * kStep);
            if (!idle && t0 <= wave_hi && t0 + kStep > wave_lo) use(t0, there, buf);
            if (W::kBufs == 1) __syncthreads();
            if (more) store(mask(units), smem + (W::kBufs == 2 ? ((s + 1) & 1) * W::kStage : 0));
        }
    }
    // Every wave is through with the stages in LDS. v_lost: whether any stored a
    // value that dropped bits.
    bool v_lost = false;
    if constexpr (KT == 3) {
        auto* flag = reinterpret_cast<int*>(smem);
        __syncthreads();
        if (tid == 0) *flag = 0;
        __syncthreads();
        if (lost_v & 0xffffu) *flag = 1;
        __syncthreads();
        v_lost = *flag != 0;
    }
    __syncthreads();
    if (idle) return;
    l = sum32(l);
    constexpr float kMost = NT == 3 ? kLargest : INFINITY;
    float low = INFINITY;
#pragma unroll
    for (int u = 0; u < DU; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int d = DU * (8 * (r / 4) + 4 * h + r % 4) + u;
            const float x = fabsf(o[u][r]);
            bad |= d < D && !(x < kMost);
            low = d < D ? fminf(low, x) : low;
        }
    if constexpr (KT == 3) bad |= v_lost && low < 0x1p-50f;
    bad |= !(l < INFINITY);
    unsigned long long redo = __ballot(bad);
    redo = (redo | redo >> 32) & 0xffffffffull;
    // Head dims DU 8 y .. DU 8 (y + 1) of the wave's columns at a time through
    // LDS, so that a column's are written in whole lines (64 lanes' eight bytes of
    // as many rows: 15 us for 128 columns of 128 in every workgroup at once).
    constexpr int CH = 8 * DU, kChRow = CH + 4, kLanes = CH / 4;
    const float by = (f.runs > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l) * (1.0f / W::O::kWeight);
    float* o_s = reinterpret_cast<float*>(smem) + w * 32 * kChRow;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int u = 0; u < DU; ++u) o_s[j * kChRow + DU * (4 * h + r) + u] = o[u][4 * y + r] * by;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int x = 0; x < 32; x += kWave / kLanes) {
            const int c = x + lane / kLanes, at = lane % kLanes * 4, d = CH * y + at;
            const floatx4 z = *reinterpret_cast<const floatx4*>(o_s + c * kChRow + at);
            if (wc + c < it.cols && !(redo >> c & 1) && d < D) {
                const int cc = it.col0 + wc + c;
                float* dst = f.runs > 1
                                 ? a.part_o + (static_cast<std::size_t>(it.unit) * kCols + wc + c) * D
                                 : a.out + (f.w.row0 + cc / p.group) * a.out_stride +
                                       (kvh * p.group + cc % p.group) * D;
                *reinterpret_cast<floatx4*>(dst + d) = z;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    if (f.runs > 1 && h == 0 && wc + j < it.cols && !(redo >> j & 1))
        a.part_ml[static_cast<std::size_t>(it.unit) * kCols + cin] = make_float2(m, l);
    while (redo) {
        const int c = __ffsll(redo) - 1;
        redo &= redo - 1;
        if (wc + c >= it.cols) break;
        float po[DP / kWave], pm, pl;
        const int prow = __shfl(row, c, kWave), phead = __shfl(head, c, kWave);
        plain_column<T, DP / kWave>(a, f.seq, prow, phead, __shfl(pq, c, kWave), lo, hi, kStep,
                                    kStep, pm, pl, po);
        const std::size_t ppc = static_cast<std::size_t>(it.unit) * kCols + wc + c;
        float* pdst = f.runs > 1 ? a.part_o + ppc * D : a.out + prow * a.out_stride + phead * D;
        const float pby = f.runs > 1 ? 1.0f : pl == 0.0f ? 0.0f : 1.0f / pl;
#pragma unroll
        for (int n = 0; n < DP / kWave; ++n)
            if (lane + kWave * n < D) pdst[lane + kWave * n] = po[n] * pby;
        if (f.runs > 1 && lane == 0) a.part_ml[ppc] = make_float2(pm, pl);
    }
}

// Workgroups on a CU, four waves each: heads past 128 take a CU's registers.
// As many as the plan counts on: with a third one of narrow items of heads of 64
// beside the two, 15 rows of 8 heads at 12921 to 25843 positions (bf16) took 145
// us for 126.
constexpr int on_a_cu(int head_size) { return head_size <= 128 ? 2 : 1; }

// WIDE: for calls in which a sequence may have more than kNarrowMost columns.
template <class T, int DP, bool WIDE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(
    on_a_cu(DP), on_a_cu(DP)))) void paged_attn_kernel(PagedAttnArgs a) {
    constexpr int kNarrowLds = Few<T, DP>::kLds, kWideLds = Wide<T, DP>::kLds;
    __shared__ __attribute__((aligned(16))) char smem[WIDE && kWideLds > kNarrowLds ? kWideLds : kNarrowLds];
    const PagedArgs& p = a.p;
    const int item = blockIdx.x;
    Item it;
    LaneWork lanes;
    const RunLength run = run_length(a, lanes);
    if (!find(a, lanes, run, [&](int, int before, int mine) { return item >= before && item < before + mine; },
              it.f))
        return;
    // Item order in a sequence: kv heads fastest (the XCDs take blocks in
    // turn, so a kv head's tiles share an L2), the longest tiles first.
    const SeqWork& w = it.f.w;
    const int at = item - it.f.item0, tile = w.tiles - 1 - at / p.n_kv_heads % w.tiles;
    it.kvh = at % p.n_kv_heads;
    it.col0 = tile * w.width;
    it.cols = min(w.width, w.n * p.group - it.col0);
    it.unit = it.f.unit0 + at * (w.width / kCols);
    // The tile's positions, this item's run of them.
    const int i0 = it.col0 / p.group, i1 = (it.col0 + it.cols - 1) / p.group;
    const int first = max(w.first, a.window ? w.p0 + i0 + 1 - a.window : 0);
    const int end = min(w.end, w.p0 + i1 + 1);
    const int len =
        ((max(0, end - first) + it.f.runs - 1) / it.f.runs + kStep - 1) / kStep * kStep;
    it.lo = first + at / p.n_kv_heads / w.tiles * len;
    it.hi = min(end, it.lo + len);
    if (WIDE && w.width == kWideCols)
        wide_item<T, DP>(a, it, smem);
    else
        narrow_item<T, DP>(a, it, smem);
}

// Joins the runs of sequences that were split: rows blockIdx.x * each .. and
// kv head blockIdx.y. A thread takes four head dims of a column of one row;
// where a row leaves threads, they take other rows, or shares of the runs where
// there are many, which are added in order in LDS. Several rows a workgroup, so
// that a batch that was not split costs one plan per workgroup of a grid that
// the card holds at once (2048 rows of 8 kv heads: 19 us with a workgroup for
// each, 4 so).
// Bound by reads that wait for one another: starts, lengths, then the partials (64
// rows in 8 kv heads 5.8 us; 843 rows of 32, three chunks of them split, 13.4).
__global__ __launch_bounds__(kThreads) void paged_join_kernel(PagedAttnArgs a, int each) {
    const PagedArgs& p = a.p;
    __shared__ __attribute__((aligned(16))) float o_s[kThreads][4];
    __shared__ float2 ml_s[kThreads];
    const int kvh = blockIdx.y, D = p.head_size, tid = threadIdx.x;
    LaneWork lanes;
    const RunLength run = run_length(a, lanes);
    const int last = min(p.rows, (static_cast<int>(blockIdx.x) + 1) * each);
    const int units = p.group * (D / 4), width = min(units, kThreads);
    for (int r = blockIdx.x * each; r < last;) {
        const int seq = row_sequence(p, r);
        Found f;
        if (seq < 0 || !find(a, lanes, run, [&](int s, int, int) { return s == seq; }, f)) {
            ++r;
            continue;
        }
        const int stop = min(last, f.w.row0 + f.w.n);
        if (f.runs <= 1) {
            r = stop;
            continue;
        }
        const int of = f.w.width / kCols;  // units of an item
        const int step = f.w.tiles * p.n_kv_heads * of;
        const int shares = max(1, min(kThreads / width, f.runs / 8));
        const int abreast = kThreads / (width * shares);  // rows at a time
        const int share = tid / width % shares, mine = tid / (width * shares);
        for (; r < stop; r += abreast) {
            const int row = r + mine;
            for (int x0 = 0; x0 < units; x0 += width) {
                const int x = x0 + tid % width;
                const bool in = mine < abreast && row < stop && x < units;
                const int h = x / (D / 4), d = x % (D / 4) * 4;
                const int cc = (row - f.w.row0) * p.group + h, tile = cc / f.w.width;
                float m = -INFINITY, l = 0.0f;
                floatx4 sum{0.f, 0.f, 0.f, 0.f};
                auto add = [&](float2 ml, floatx4 o) {
                    // A run whose sum is NaN has no maximum to go by.
                    const float mn = fmaxf(m, ml.x);
                    const float old = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                    const float fac = ml.x == mn || ml.y != ml.y ? 1.0f
                                      : ml.x == -INFINITY        ? 0.0f
                                                                 : __builtin_amdgcn_exp2f(ml.x - mn);
                    l = l * old + fac * ml.y;
                    sum = sum * old + fac * o;
                    m = mn;
                };
                if (in) {
                    const std::size_t u0 = f.unit0 + ((f.w.tiles - 1 - tile) * p.n_kv_heads + kvh) * of +
                                           cc % f.w.width / kCols;
                    for (int y = share; y < f.runs; y += 4 * shares) {
                        float2 ml[4];
                        floatx4 o[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const std::size_t run_i = min(y + i * shares, f.runs - 1);
                            const std::size_t pc = (u0 + run_i * step) * kCols + cc % kCols;
                            ml[i] = a.part_ml[pc];
                            o[i] = *reinterpret_cast<const floatx4*>(a.part_o + pc * D + d);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (y + i * shares < f.runs) add(ml[i], o[i]);
                    }
                }
                if (shares > 1) {
                    __syncthreads();
                    ml_s[tid] = make_float2(m, l);
                    *reinterpret_cast<floatx4*>(o_s[tid]) = sum;
                    __syncthreads();
                    if (in && share == 0)
                        for (int y = 1; y < shares; ++y)
                            add(ml_s[y * width + tid], *reinterpret_cast<const floatx4*>(o_s[y * width + tid]));
                }
                if (in && share == 0)
                    *reinterpret_cast<floatx4*>(a.out + row * a.out_stride + (kvh * p.group + h) * D + d) =
                        l == 0.0f ? floatx4{0.f, 0.f, 0.f, 0.f} : sum * (1.0f / l);
            }
        }
        r = stop;
    }
}

// --- launch ---------------------------------------------------------------------------

// Workgroups the card holds at once.
int paged_slots(const em_paged_shape& s) { return on_a_cu(s.head_size) * cu_count(); }

// Whether any sequence of the shape can be split: it needs one and a half
// runs' positions.
bool can_split(const em_paged_shape& s) {
    return static_cast<long long>(s.page_size) * s.max_pages >= kMinRun * 3 / 2;
}

// Whether a sequence of the call may take wide items.
bool can_widen(const em_paged_shape& s, std::size_t rows) {
    return rows * static_cast<std::size_t>(s.n_heads / s.n_kv_heads) >
           static_cast<std::size_t>(kNarrowMost);
}

// Units of partials at most. All columns' positions over a run's length are at
// most the slots. A wide sequence that is split has 1.5 lengths or more, so no
// more than 4/3 runs a length; a narrow one twice that; one sixteenth is added
// for the float arithmetic of the plan.
int partial_units(const em_paged_shape& s, std::size_t rows) {
    if (!can_split(s)) return 0;
    return (paged_slots(s) * 17 / 12 + 1) * (can_widen(s, rows) ? kWideCols / kCols : 2);
}

std::size_t paged_attention_scratch(const em_paged_shape& s, std::size_t, std::size_t rows) {
    return static_cast<std::size_t>(partial_units(s, rows)) * kCols *
           (static_cast<std::size_t>(s.head_size) + 2);
}

// Items at most: column tiles (each sequence's last may be partly full;
// narrow ones and wide), and up to two runs more for each run length in all
// columns' positions.
long long paged_items(const em_paged_shape& s, long long n_seqs, long long rows) {
    const long long cols = rows * (s.n_heads / s.n_kv_heads), seqs = std::min(n_seqs, rows);
    const bool wide = can_widen(s, static_cast<std::size_t>(rows));
    long long tiles = cols / kCols + seqs;
    if (wide) {
        tiles = std::min(tiles, seqs * (kNarrowMost / kCols));
        tiles += cols / kWideCols + std::min(seqs, cols / (kNarrowMost + 1));
    }
    const int slots = paged_slots(s);
    return tiles * s.n_kv_heads + (can_split(s) ? 2 * slots + slots / 8 + 1 : 0);
}

template <class T, int DP>
void launch_attn(const PagedAttnArgs& a, dim3 grid, hipStream_t stream) {
    if (a.wide)
        hipLaunchKernelGGL((paged_attn_kernel<T, DP, true>), grid, dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((paged_attn_kernel<T, DP, false>), grid, dim3(kThreads), 0, stream, a);
}
template <class T>
void launch_attn(const PagedAttnArgs& a, dim3 grid, hipStream_t stream) {
    if (a.p.head_size <= 64)
        launch_attn<T, 64>(a, grid, stream);
    else if (a.p.head_size <= 128)
        launch_attn<T, 128>(a, grid, stream);
    else
        launch_attn<T, 256>(a, grid, stream);
}

void run_paged_attention(PagedAttnArgs a, const em_paged_shape& s, float* scratch,
                         hipStream_t stream) {
    const auto rows = static_cast<std::size_t>(a.p.rows);
    a.wide = can_widen(s, rows);
    a.slots = paged_slots(s);
    // A stage of fp32 takes twice the products and both splits: us at 192 /
    // 512 positions, three chunks of 200 rows of 8 heads of 64 (fp32) 45 / 62,
    // one of 1205 rows of 24 heads of 96 85 / 116; eight of up to 466 rows of 20
    // heads of 80 (fp16) 50 / 34.
    a.min_wide = s.type == EM_CACHE_F32 ? 192 : 512;
    // With two workgroups on a CU a wide item takes 175 ns a position of heads of
    // 128 (fp32; bf16 96, fp16 75), a narrow one that reads at HBM's rate 50 (fp32
    // 100, of which the cache holds some). Measured at that head size alone; at
    // others the ratio is assumed, both items' work being linear in it.
    a.wide_cost = s.type == EM_CACHE_F32 ? 3.0f : s.type == EM_CACHE_BF16 ? 2.0f : 1.5f;
    a.part_units = partial_units(s, rows);
    a.part_o = scratch;
    a.part_ml = reinterpret_cast<float2*>(
        scratch + static_cast<std::size_t>(a.part_units) * kCols * s.head_size);
    const dim3 grid(static_cast<unsigned>(paged_items(s, a.p.n_seqs, a.p.rows)));
    if (s.type == EM_CACHE_F32)
        launch_attn<float>(a, grid, stream);
    else if (s.type == EM_CACHE_F16)
        launch_attn<_Float16>(a, grid, stream);
    else
        launch_attn<__bf16>(a, grid, stream);
    if (a.part_units) {
        const int each = static_cast<int>(std::max(
            1LL, static_cast<long long>(a.p.rows) * a.p.n_kv_heads / (4 * cu_count())));
        hipLaunchKernelGGL(paged_join_kernel, dim3(ceil_div(a.p.rows, each), a.p.n_kv_heads),
                           dim3(kThreads), 0, stream, a, each);
    }
}

bool a16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace em

using em::fail;

extern "C" {

size_t em_paged_attention_scratch_floats(const em_paged_shape* s, size_t n_seqs, size_t rows) {
    if (!s || !em::paged_reject(*s).empty() || rows > (size_t{1} << 22) ||
        n_seqs > (size_t{1} << 20))
        return 0;
    return em::paged_attention_scratch(*s, n_seqs, rows);
}

int em_paged_attention(const em_paged_shape* s, const em_paged_batch* b, size_t rows,
                       const float* q, size_t q_stride, const void* key_cache,
                       const void* value_cache, float* out, size_t out_stride, float scale,
                       int window, float* scratch, void* stream) {
    if (const int rc = em_paged_check(s)) return rc;
    if (!b) return fail(EM_EINVAL, "paged_attention: null batch");
    const std::string why = em::paged_batch_reject(*s, *b, rows);
    if (!why.empty()) return fail(EM_EINVAL, why);
    if (window < 0 || window > (1 << 30))
        return fail(EM_EINVAL, "paged_attention: a window of 0 to 2^30 positions");
    if (!std::isfinite(scale * 1.4427f))
        return fail(EM_EINVAL, "paged_attention: scale is not finite, or its product with log2 e");
    if (rows == 0 || b->n_seqs == 0) return EM_OK;
    const size_t need =
        em::paged_attention_scratch(*s, static_cast<size_t>(b->n_seqs), rows);
    if (!q || !key_cache || !value_cache || !out || (need && !scratch))
        return fail(EM_EINVAL, "paged_attention: null pointer");
    const size_t dim = static_cast<size_t>(s->n_heads) * s->head_size;
    const size_t most = size_t{1} << 32;
    if (q_stride % 4 || out_stride % 4 || q_stride >= most || out_stride >= most ||
        (rows > 1 && (q_stride < dim || out_stride < dim)))
        return fail(EM_EINVAL, "paged_attention: row strides must be multiples of 4, no smaller "
                               "than a row");
    if (!em::a16(q) || !em::a16(key_cache) || !em::a16(value_cache) || !em::a16(out) ||
        (need && !em::a16(scratch)))
        return fail(EM_EINVAL, "paged_attention: pointers must be 16-byte aligned");
    if (!em::device_present()) return fail(EM_ENODEV, "paged_attention: no usable GPU");
    if (em::paged_items(*s, b->n_seqs, static_cast<long long>(rows)) >= (1LL << 24))
        return fail(EM_EINVAL, "paged_attention: more rows and heads than one launch takes");
    try {
        em::PagedAttnArgs a{};
        a.p = em::paged_args(*s, *b, rows);
        a.q = q;
        a.kc = key_cache;
        a.vc = value_cache;
        a.out = out;
        a.q_stride = static_cast<long long>(q_stride);
        a.out_stride = static_cast<long long>(out_stride);
        const double by = scale != 0.0f ? scale : 1.0 / std::sqrt(static_cast<double>(s->head_size));
        a.scale2 = static_cast<float>(by * 1.4426950408889634074);
        a.window = window;
        em::run_paged_attention(a, *s, scratch, static_cast<hipStream_t>(stream));
        em::hip_check(hipGetLastError(), "launch");
    } catch (const std::exception& e) {
        return fail(EM_EDEVICE, e.what());
    }
    return EM_OK;
}

}  // extern "C"
