// Sampling: the next token of each row of logits by temperature, top-k,
// top-p and min-p from a given uniform number.
//
// A token's weight w = exp((x - max) / T) is formed in 64 bits, so that which
// side of a border u falls on is off by some 2^-50 of the sum, where fp32 sums
// of 100000 weights lose 2^-20 of it. Where weights are added by atomics, in an
// order that changes, they are integers, w 2^bits rounded down, bits = 62 -
// ceil(log2 vocab), at most 52: the row's sum stays below 2^63 and is always the same.
//
// Both filters are thresholds on the logit: the last token kept is a value and
// a number of tokens of just that value, lowest index first. A histogram over
// the distance from the maximum (counts for top-k, weights for top-p) names the
// bin it lies in, and the few tokens of that bin are ranked against each other;
// a bin with too many (ties, or a maximum far above the rest) is resolved by
// radix selection on the logits' bits instead. The draw then adds the kept
// weights in index order: a total per wave, whose run of the row the whole
// workgroup then goes through.
//
// One workgroup a row, 16 waves each with its own run of consecutive logits;
// rows of up to 32765 are read once, into LDS, longer ones once a pass (greedy and
// unfiltered ones once in all). Not bound by the logits' bytes but by the passes
// of a workgroup one behind the other: 1 x 32000 with top-k of 40 15 us, with
// top-p of 0.9 32 (four passes over LDS, the 64-bit weights in two of them); 256 x
// 131072 unfiltered 43 us (weights, for the most part), with min-p 60, greedy 25,
// where a copy's rate would take 26.
#include <algorithm>
#include <cmath>

#include "internal.hpp"
#include "llm_engine_amd.h"
#include "wave.hpp"

namespace em {
namespace {

using u64 = unsigned long long;
constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / kWave;
constexpr int kChunk = 4 * kWave;  // logits a wave reads at once
constexpr int kMaxVocab = 1 << 20;
// Bins of a histogram: what LDS holds beside a row, and more where it need not.
constexpr int kHeldBins = 2048, kWideBins = 4096;
constexpr int kList = 512;   // tokens of a bin that are ranked against each other
constexpr int kShort = 128;  // a list that holds all that may be kept
constexpr int kMaxSlices = kWave;  // workgroups a row, where several share one: a lane each

struct SampleArgs {
    int rows, vocab, bits;
    const float* logits;
    long long stride;
    const float *u, *temperature, *top_p, *min_p;
    const int* top_k;
    int* tokens;
    float* logprobs;
};

// A logit as the sampler sees it: NaN is -inf, -0 is 0.
__device__ __forceinline__ float clean(float x) { return fmaxf(x + 0.0f, -INFINITY); }
// Its bits in an order that is the values'; -inf has the least.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}

// 2^(i / 32), then 2^((i + 1/2) / 32).
constexpr int kRoots = 32;
__device__ constexpr double kRoot[2 * kRoots] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
    1.0108892860517005, 1.0330248790212284, 1.0556451783605572, 1.0787607977571199,
    1.102382583307841, 1.1265216186082418, 1.1511892299529827, 1.1763969916502812,
    1.202156731452703, 1.22848053610687, 1.255380757024691, 1.2828700160787783,
    1.3109612115247644, 1.339667524053303, 1.3690024229745905, 1.3989796725383112,
    1.42961333839197, 1.460917794180647, 1.4929077282912648, 1.5255981507445384,
    1.559004400237837, 1.593142151342267, 1.6280274218573478, 1.6636765803267364,
    1.7001063537185235, 1.7373338352737062, 1.7753764925265212, 1.8142521755003989,
    1.8539791250833855, 1.8945759815869656, 1.9360617934922943, 1.978456026387951};

// A row's weights relative to its maximum: w = 2^(z / 32), z = (x - top) *
// 32 log2 e / T: a root from the table, the rest by its Taylor series (the
// first term left out is below 2^-48). The whole part of z is read from the
// low bits of z + 1.5 2^52 and added to the exponent's, so that of the
// instructions only the conversion of x is not a 64-bit add or multiply-add
// (floor, ldexp and a 16-entry table take half as long again).
struct Weigh {
    float top;
    bool endless;  // top is +inf: its tokens share all the weight
    float least;   // weights of lower logits (below e^-60) count as 0
    double c;      // 32 log2 e / T
    int bits;
    const double* roots;  // kRoot in LDS
    // 2^(y / 32), |y| <= 1/2.
    static __device__ __forceinline__ double small_power(double y) {
        constexpr double kL = 0.69314718055994530942 / kRoots;
        double p = fma(y, kL * kL * kL * kL * kL / 120, kL * kL * kL * kL / 24);
        p = fma(p, y, kL * kL * kL / 6);
        p = fma(p, y, kL * kL / 2);
        p = fma(p, y, kL);
        return fma(p, y, 1.0);
    }
    static constexpr double kMagic = 6755399441055744.0;
    __device__ __forceinline__ double below(float x) const {
        return static_cast<double>(x) - static_cast<double>(top);
    }
    // Weights side by side and without a branch, so that their chains and table
    // reads overlap (256 x 131072 unfiltered: 65 us, an element at a time 71; 64 x
    // 32000 of mixed settings 35 and 40). Not for an endless row; logits below `least`
    // weigh what it does and are the caller's to leave out.
    template <int N>
    __device__ __forceinline__ void several(const float (&x)[N], double (&w)[N]) const {
        double t[N], y[N], q[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const double d = below(fmaxf(x[i], least));
            t[i] = fma(d, c, kMagic);
            y[i] = fma(d, c, kMagic - t[i]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = roots[__double_as_longlong(t[i]) & (kRoots - 1)];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = static_cast<int>(__double_as_longlong(t[i]));
            q[i] *= small_power(y[i]);
            w[i] = __longlong_as_double(__double_as_longlong(q[i]) + (static_cast<u64>(n >> 5) << 52));
        }
    }
    __device__ __forceinline__ void whole_eight(const float (&x)[8], u64 (&w)[8]) const {
        double z[8], t[8], q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            z[i] = fma(below(fmaxf(x[i], least)), c, -0.5);
            t[i] = z[i] + kMagic;
            z[i] -= t[i] - kMagic;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = roots[kRoots + (__double_as_longlong(t[i]) & (kRoots - 1))];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int n = static_cast<int>(__double_as_longlong(t[i]));
            q[i] *= small_power(z[i]);
            w[i] = (__double_as_longlong(q[i]) - (u64{0x3fe} << 52)) >> min(52 - bits - (n >> 5), 63);
        }
    }
    __device__ __forceinline__ double operator()(float x) const {
        if (endless) return x == top ? 1.0 : 0.0;
        const double d = below(x), t = fma(d, c, kMagic), y = fma(d, c, kMagic - t);
        const int n = static_cast<int>(__double_as_longlong(t));
        const double q = small_power(y) * roots[n & (kRoots - 1)];
        const u64 w = __double_as_longlong(q) + (static_cast<u64>(n >> 5) << 52);
        return x < least ? 0.0 : __longlong_as_double(w);
    }
    // The weight as an integer of 2^-bits, rounded down: z - 1/2 to the nearest
    // whole number and a root half a step higher leave q in [1, 2] up to
    // rounding, whose bits less those of 1/2 are q 2^52.
    __device__ __forceinline__ u64 whole(float x) const {
        if (endless) return x == top ? u64{1} << bits : 0;
        const double z = fma(below(x), c, -0.5), t = z + kMagic, y = z - (t - kMagic);
        const int n = static_cast<int>(__double_as_longlong(t));
        const double q = small_power(y) * roots[kRoots + (n & (kRoots - 1))];
        const u64 w = (__double_as_longlong(q) - (u64{0x3fe} << 52)) >> min(52 - bits - (n >> 5), 63);
        return x < least ? 0 : w;
    }
};

// A share in [0, 1) of a sum of weights, exactly and rounded up.
__device__ __forceinline__ u64 share_up(u64 total, float share) {
    const u64 f = static_cast<u64>(static_cast<double>(share) * 0x1p64);
    return __umul64hi(total, f) + (total * f != 0);
}

__device__ __forceinline__ float wave_top(float v) {
    return last_lane(wave_scan(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); }));
}
__device__ __forceinline__ int wave_least(int v) {
    return last_lane(wave_scan(v, 0x7fffffff, [](int a, int b) { return min(a, b); }));
}

template <int BINS>
struct SampleShared {
    static constexpr int kBins = BINS;
    u64 weight[BINS];  // the bins'; once they have been read, the list's
    uint32_t count[BINS];
    uint32_t list[kList];
    int list_at[kList];
    double roots[2 * kRoots];
    double part[kSampleWaves], sums[kMaxSlices];
    u64 part64[kSampleWaves];
    float part_hi[kSampleWaves], part_lo[kSampleWaves];
    uint32_t part_n[kSampleWaves];
    uint32_t n, key, ties, bin, bin_end;
    u64 left;
    int token, last, keep;  // token, last: the drawing threads (draw_in_run)
};

// Chunks a wave whose row LDS (160 KB) holds beside SampleShared.
constexpr int kHeldChunks = 8;
static_assert(sizeof(SampleShared<kHeldBins>) + kHeldChunks * kSampleWaves * kChunk * sizeof(float) <= 160 * 1024);

template <class T>
__device__ __forceinline__ T shfl(T v, int lane) { return __shfl(v, lane, kWave); }

// Exclusive prefix of v over the workgroup's threads, and the total.
template <class T>
__device__ __forceinline__ T block_prefix(T v, T* part, T& total) {
    const T in = wave_scan(v);
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if (threadIdx.x % kWave == kWave - 1) part[wave] = in;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kSampleWaves; ++i) {
        const T p = part[i];
        before += i < wave ? p : T(0);
        total += p;
    }
    return before + in - v;
}

// Running sums of v over the workgroup's threads: a thread's own, and `before`
// its predecessor's, the same bits (own less v would lose what is 2^-53 of v).
__device__ __forceinline__ double block_running(double v, double* part, double& before) {
    const double in = wave_scan(v);
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    __syncthreads();
    if (lane == kWave - 1) part[wave] = in;
    __syncthreads();
    double base = 0.0;
#pragma unroll
    for (int i = 0; i < kSampleWaves; ++i) base += i < wave ? part[i] : 0.0;
    const double ahead = __shfl_up(in, 1, kWave);
    before = lane ? base + ahead : base;
    return base + in;
}

// A row's logits, cleaned. HELD: kept in LDS, read from memory once.
template <bool HELD>
struct Row {
    const float* x;
    float* held;
    int vocab, pre, chunks;  // pre: floats from 16 bytes' alignment to the row

    __device__ __forceinline__ int position(int c) const {
        return ((threadIdx.x / kWave) * chunks + c) * kChunk + 4 * (threadIdx.x % kWave);
    }
    __device__ __forceinline__ float load(int pos) const {
        const int i = pos - pre;
        const float v = clean(x[max(0, min(i, vocab - 1))]);
        return i >= 0 && i < vocab ? v : -INFINITY;
    }
    __device__ __forceinline__ float at(int pos) const {
        if constexpr (HELD) return held[pos];
        return load(pos);
    }
    static constexpr int U = 8;  // vectors in flight: a held row's eight chunks at once
    // f(vectors, first chunk) of this thread's logits, eight vectors at a
    // time (-inf past the end); KEEP: the pass that fills `held`.
    template <bool KEEP = false, class Fn>
    __device__ __forceinline__ void batches(Fn f) const {
        for (int c = 0; c < chunks; c += U) {
            float4 v[U];
            // All in the row, the same for the whole wave: loads without a
            // branch around each, so that they are in flight together.
            const int from = __builtin_amdgcn_readfirstlane(position(c) - 4 * (threadIdx.x % kWave));
            const int to = from + (min(c + U, chunks) - c) * kChunk;
            if (HELD && !KEEP) {
#pragma unroll
                for (int i = 0; i < U; ++i)
                    v[i] = *reinterpret_cast<const float4*>(held + position(min(c + i, chunks - 1)));
            } else if (from >= pre && to <= pre + vocab) {
                const float* src = x - pre;
#pragma unroll
                for (int i = 0; i < U; ++i)
                    v[i] = *reinterpret_cast<const float4*>(src + position(min(c + i, chunks - 1)));
#pragma unroll
                for (int i = 0; i < U; ++i)
                    v[i] = make_float4(clean(v[i].x), clean(v[i].y), clean(v[i].z), clean(v[i].w));
            } else {
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int pos = position(min(c + i, chunks - 1));
                    v[i] = make_float4(load(pos), load(pos + 1), load(pos + 2), load(pos + 3));
                }
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (c + i >= chunks)
                    v[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                else if constexpr (HELD && KEEP)
                    *reinterpret_cast<float4*>(held + position(c + i)) = v[i];
            }
            f(v, c);
        }
    }
    // f(x, position) of every logit of this thread.
    template <bool KEEP = false, class Fn>
    __device__ __forceinline__ void each(Fn f) const {
        batches<KEEP>([&](const float4 (&v)[U], int c) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (c + i >= chunks) break;
                const int pos = position(c + i);
                f(v[i].x, pos);
                f(v[i].y, pos + 1);
                f(v[i].z, pos + 2);
                f(v[i].w, pos + 3);
            }
        });
    }
};

// A row's settings; `top_k` 0: off.
struct Settings {
    float temperature, top_p;
    bool greedy;
    int top_k;
    double min_p, draw;
    __device__ __forceinline__ Settings(const SampleArgs& a, int r) {
        temperature = a.temperature ? a.temperature[r] : 1.0f;
        greedy = !(temperature > 0.0f);
        top_k = a.top_k && a.top_k[r] < a.vocab ? max(0, a.top_k[r]) : 0;
        top_p = a.top_p ? a.top_p[r] : 1.0f;
        const float mp = a.min_p ? a.min_p[r] : 0.0f, u = a.u[r];
        min_p = mp > 0.0f ? fmin(static_cast<double>(mp), 1.0) : 0.0;
        draw = u > 0.0f ? fmin(static_cast<double>(u), 0x1.fffffffffffffp-1) : 0.0;
    }
};

__device__ __forceinline__ Weigh weigh_of(const SampleArgs& a, const Settings& set, float top,
                                          const double* roots) {
    const float T = set.temperature;
    return {top, top == INFINITY, fmaxf(static_cast<float>(top - 60.0 * T), -3.4028235e38f),
            set.greedy ? 0.0 : kRoots * 1.4426950408889634074 / T, a.bits, roots};
}
// No logit below this weighs min_p (a thousandth of T and the fp32 roundings
// of the sum are left for the comparison in 64 bits), or anything.
__device__ __forceinline__ float cut_of(const Settings& set, const Weigh& weigh) {
    if (weigh.endless || set.min_p == 0.0) return weigh.least;
    return fmaxf(weigh.least, static_cast<float>(weigh.top + (log(set.min_p) - 1e-3) * set.temperature -
                                                 1e-6 * fabs(static_cast<double>(weigh.top))));
}
// The histogram's bin of x; inv: bins over the range they cover.
template <int BINS>
__device__ __forceinline__ int bin_at(float x, float top, float inv) {
    const float b = x == top ? 0.0f : (top - x) * inv;
    return b < BINS - 1 ? static_cast<int>(b) : BINS - 1;
}
// Bins of equal factors in weight, the last one from 2^-32.
template <int BINS>
__device__ __forceinline__ float weight_bins(const Weigh& weigh) {
    return static_cast<float>(fmin(weigh.c * (BINS / 32.0 / kRoots), 3e38));
}

// A lane a run of the row, `sum` its kept weight: the first run whose running
// sum passes draw times the total (the last with any weight where rounding
// leaves none), and what of that is wanted of the run.
__device__ __forceinline__ int pick_run(double sum, double draw, double& total, double& target) {
    const double run = wave_scan(sum);
    total = last_lane(run);
    target = draw * total;
    const u64 some = __ballot(sum > 0.0), past = __ballot(sum > 0.0 && run > target);
    const int pick = past ? __ffsll(past) - 1 : 63 - __clzll(some);
    const double ahead = __shfl_up(run, 1, kWave);  // the run before's
    target = fmax(0.0, target - (pick ? __shfl(ahead, pick, kWave) : 0.0));
    return pick;
}

// Draws from logits [begin, end) by the whole workgroup, consecutive ones a
// thread: those above thr and the first `left` at it, of weight wt, of which
// `target` is wanted; `total` is the row's.
template <class Shared, class At, class Kept>
__device__ __forceinline__ void draw_in_run(const SampleArgs& a, int r, Shared& s, At at,
                                            int begin, int end, Kept kept, float cut, float thr,
                                            uint32_t left, double wt, double target, double total) {
    const int tid = threadIdx.x, span = end - begin;
    const int each = (span + kSampleThreads - 1) / kSampleThreads;
    const int from = begin + tid * each, to = min(from + each, end);
    double mine = 0.0;
    uint32_t n = 0;
    for (int p = from; p < to; ++p) {
        const float x = at(p);
        if (x > thr && x >= cut) mine += kept(x);
        n += x == thr && wt > 0.0;
    }
    uint32_t here = 0;
    if (left > 0) {
        uint32_t all_n = 0;
        const uint32_t n_before = block_prefix(n, s.part_n, all_n);
        here = left > n_before ? min(left - n_before, n) : 0;
        mine += here * wt;
    }
    double before = 0.0;
    const double through = block_running(mine, s.part, before);
    // One thread draws: the first with any weight whose running sum passes the
    // target, the last with any where rounding leaves none. Running sums of equal
    // real value may round apart (a scan adds in another order for each lane), so
    // several may pass or none; the lowest index is the same on every call. At a
    // target of 0 it is the first thread with any weight, however small beside
    // what follows.
    const int lane = tid % kWave;
    const u64 some = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && through > target);
    if (past && lane == __ffsll(past) - 1) atomicMin(&s.token, tid);
    if (some && lane == 63 - __clzll(some)) atomicMax(&s.last, tid);
    __syncthreads();
    if (tid != (s.token < kSampleThreads ? s.token : s.last)) return;
    double run = before, w_token = 0.0;
    int token = -1;
    for (int p = from; p < to; ++p) {
        const float x = at(p);
        double w = 0.0;
        if (x > thr) {
            if (x >= cut) w = kept(x);
        } else if (x == thr && here > 0) {
            --here;
            w = wt;
        }
        if (!(w > 0.0)) continue;
        token = p;
        w_token = w;
        run += w;
        if (run > target) break;
    }
    a.tokens[r] = token;
    if (a.logprobs) a.logprobs[r] = static_cast<float>(log(w_token / total));
}

// Draws from the n tokens of the list (keys and positions, at most kShort), all
// that may be kept among them: ranks them, keeps the highest most_kept, of those what top-p
// (nucleus, by whole weights) and min-p leave, which are some of the highest
// ranks too.
template <class Shared>
__device__ __forceinline__ void draw_from_list(const SampleArgs& a, int r, Shared& s,
                                               const Settings& set, const Weigh& weigh, uint32_t n,
                                               uint32_t most_kept, bool nucleus) {
    const int tid = threadIdx.x;
    auto* weights = reinterpret_cast<double*>(s.weight + kShort);
    static_assert(kShort == 2 * kWave && Shared::kBins >= 2 * kShort);
    uint32_t key = 0, rank = 0, place = 0;  // place: rank by position
    int pos = 0;
    const bool mine = static_cast<uint32_t>(tid) < n;
    if (mine) {
        key = s.list[tid];
        pos = s.list_at[tid];
#pragma unroll 8
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t o = s.list[i];
            const int at = s.list_at[i];
            rank += (o > key) | ((o == key) & (at < pos));
            place += at < pos;
        }
    }
    most_kept = min(n, most_kept);
    const bool in = mine && rank < most_kept;
    const float x = key_value(key);
    const double w = in ? weigh(x) : 0.0;
    const u64 ww = in ? weigh.whole(x) : 0;
    if (tid == 0) s.keep = most_kept;
    __syncthreads();  // the list has been read
    if (in) s.weight[rank] = ww;
    if (mine) s.list_at[place] = pos;
    __syncthreads();
    if (in && nucleus) {
        u64 before = 0, total = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < most_kept; ++i) {
            const u64 o = s.weight[i];
            before += i < rank ? o : 0;
            total += o;
        }
        const u64 target = max(u64{1}, share_up(total, fmaxf(set.top_p, 0.0f)));
        if (rank > 0 && before >= target) atomicMin(&s.keep, static_cast<int>(rank));
    }
    if (in && w < set.min_p) atomicMin(&s.keep, static_cast<int>(rank));
    __syncthreads();
    // The draw: weights in 64 bits (whole ones would leave nothing of those below
    // 2^-bits) in the order of positions, two a lane of one wave.
    if (mine) weights[place] = rank < static_cast<uint32_t>(s.keep) ? w : 0.0;
    __syncthreads();
    if (tid >= kWave) return;
    const uint32_t at = 2 * tid;
    const double w0 = at < n ? weights[at] : 0.0, w1 = at + 1 < n ? weights[at + 1] : 0.0;
    double total = 0.0, target = 0.0;
    if (tid != pick_run(w0 + w1, set.draw, total, target)) return;
    const bool second = w1 > 0.0 && !(w0 > target);
    a.tokens[r] = s.list_at[at + second];
    if (a.logprobs) a.logprobs[r] = static_cast<float>(log((second ? w1 : w0) / total));
}

// The last token that top-p keeps, from the list's tokens of the border bin
// (in_bin): the value, and how many of just that value. left: what is wanted of
// the bin's weight; the first `ties` of thr alone count, where top-k set them.
template <class Shared, class InBin>
__device__ __forceinline__ void nucleus_end(Shared& s, const Weigh& weigh, uint32_t n,
                                            InBin in_bin, u64 left, float& thr, uint32_t& ties) {
    const int tid = threadIdx.x;
    uint32_t mine = 0;
    u64 w = 0;
    if (static_cast<uint32_t>(tid) < n) {
        mine = s.list[tid];
        w = in_bin(mine) ? weigh.whole(key_value(mine)) : 0;
        s.weight[tid] = w;
    }
    __syncthreads();
    if (w) {
        u64 above = 0;
        uint32_t equal = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t o = s.list[i];
            const u64 ow = s.weight[i];
            above += o > mine ? ow : 0;
            equal += o == mine;
        }
        if (ties && key_value(mine) == thr) equal = min(equal, ties);
        if (above < left && above + equal * w >= left) {
            s.key = mine;
            s.ties = static_cast<uint32_t>((left - above + w - 1) / w);
        }
    }
    __syncthreads();
    thr = key_value(s.key);
    ties = s.ties;
}

template <bool HELD, class Shared>
__device__ __forceinline__ void sample_row(const SampleArgs& a, int r, Shared& s, float* held) {
    constexpr int kBins = Shared::kBins;
    constexpr int E = kBins / kSampleThreads;  // bins a thread
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    Row<HELD> row;
    row.held = held;
    row.x = a.logits + r * a.stride;
    row.vocab = a.vocab;
    row.pre = static_cast<int>(reinterpret_cast<uintptr_t>(row.x) / 4 % 4);
    row.chunks = (a.vocab + row.pre + kSampleWaves * kChunk - 1) / (kSampleWaves * kChunk);
    if (tid < 2 * kRoots) s.roots[tid] = kRoot[tid];
    const Settings set(a, r);
    const float top_p = set.top_p;
    const int k = set.top_k;
    const double min_p = set.min_p;

    // The maximum, and the least of the threads' maxima.
    float most = -INFINITY;
    // A long row without a filter is read once: its weights are summed beside
    // the maximum, relative to the thread's own so far.
    const bool once = !HELD && !set.greedy && k == 0 && !(top_p < 1.0f) && min_p == 0.0;
    double sum = 0.0;
    int first = 0;  // greedy: the lowest position of the thread's maximum
    if (once) {
        __syncthreads();  // the roots
        row.batches([&](const float4 (&v)[Row<HELD>::U], int) {
            float m = most;
#pragma unroll
            for (int i = 0; i < Row<HELD>::U; ++i)
                m = fmaxf(fmaxf(m, fmaxf(v[i].x, v[i].y)), fmaxf(v[i].z, v[i].w));
            Weigh weigh = weigh_of(a, set, m, s.roots);
            weigh.endless = false;  // +inf: summed again
            if (__ballot(m > most)) sum *= m > most ? weigh(most) : 1.0;
#pragma unroll
            for (int i = 0; i < Row<HELD>::U; ++i) {
                const float x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                double w[4];
                weigh.several(x, w);
                if (__ballot(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])) < weigh.least)) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = x[e] < weigh.least ? 0.0 : w[e];
                }
                sum += (w[0] + w[1]) + (w[2] + w[3]);
            }
            most = m;
        });
    } else if (set.greedy) {
        row.template each<true>([&](float x, int pos) {
            first = x > most ? pos : first;
            most = fmaxf(most, x);
        });
    } else {
        row.template each<true>([&](float x, int) { most = fmaxf(most, x); });
    }
    float top = wave_top(most), low = -wave_top(-most);
    if (lane == 0) {
        s.part_hi[wave] = top;
        s.part_lo[wave] = low;
    }
    for (int i = tid; i < kBins; i += kSampleThreads) {
        s.count[i] = 0;
        s.weight[i] = 0;
    }
    if (tid == 0) {
        s.n = 0;
        s.token = kSampleThreads;
        s.last = -1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSampleWaves; ++i) {
        top = fmaxf(top, s.part_hi[i]);
        low = fminf(low, s.part_lo[i]);
    }
    if (top == -INFINITY) {
        if (tid == 0) {
            a.tokens[r] = -1;
            if (a.logprobs) a.logprobs[r] = -INFINITY;
        }
        return;
    }
    const Weigh weigh = weigh_of(a, set, top, s.roots);

    // The last token kept: value thr, the first `ties` of that value.
    float thr = -INFINITY;
    uint32_t ties = 0;

    // Radix selection from the top: the value at which the running sum of
    // amount(x) over falling values reaches `target`, and what is left of the
    // target for the tokens of just that value.
    auto radix = [&](u64 target, auto amount) {
        uint32_t prefix = 0;
        u64 left = target;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) s.weight[tid] = 0;
            __syncthreads();
            row.each([&](float x, int) {
                const uint32_t key = order_key(x);
                if (x > -INFINITY && (shift == 24 || key >> (shift + 8) == prefix))
                    atomicAdd(&s.weight[key >> shift & 255], amount(x));
            });
            __syncthreads();
            if (tid == 0) {
                u64 l = left;
                int b = 255;
                while (b > 0 && s.weight[b] < l) l -= s.weight[b--];
                s.left = l;
                s.key = prefix << 8 | b;
            }
            __syncthreads();
            prefix = s.key;
            left = s.left;
        }
        thr = key_value(prefix);
        return left;
    };
    auto bin_of = [&](float x, float inv) { return bin_at<kBins>(x, top, inv); };
    // Appends a token to the list (s.n counts past its end too).
    auto append = [&](float x, int pos) {
        const uint32_t i = atomicAdd(&s.n, 1u);
        if (i < kList) {
            s.list[i] = order_key(x);
            s.list_at[i] = pos - row.pre;
        }
    };

    if (set.greedy) {
        // The lowest index of the maximum.
        if (tid == 0) s.keep = 0x7fffffff;
        __syncthreads();
        if (most == top) atomicMin(&s.keep, first);
        __syncthreads();
        if (tid == 0) {
            a.tokens[r] = s.keep - row.pre;
            if (a.logprobs) a.logprobs[r] = 0.0f;
        }
        return;
    }
    if (k > 0) {
        // Where every thread has a maximum, k of them are at least the least
        // one, so only tokens from there on need be counted.
        float floor = low;
        if (low == -INFINITY || k > kSampleThreads) {
            float least = INFINITY;
            row.each([&](float x, int) { least = x > -INFINITY ? fminf(least, x) : least; });
            least = -wave_top(-least);
            __syncthreads();
            if (lane == 0) s.part_lo[wave] = least;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kSampleWaves; ++i) least = fminf(least, s.part_lo[i]);
            floor = least;
        }
        const float inv = fminf((kBins - 1) / (top - floor), 3e38f);
        row.each([&](float x, int) {
            if (x >= floor) atomicAdd(&s.count[bin_of(x, inv)], 1u);
        });
        __syncthreads();
        uint32_t bins[E], sum_n = 0, all = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            bins[i] = s.count[E * tid + i];
            sum_n += bins[i];
        }
        const uint32_t want = k;
        uint32_t before = block_prefix(sum_n, s.part_n, all);
        // Fewer tokens than k that can be drawn: the filter is off.
        if (all >= want) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                if (before < want && before + bins[i] >= want) {
                    s.bin = E * tid + i;
                    s.left = want - before;
                    s.bin_end = before + bins[i];
                }
                before += bins[i];
            }
            __syncthreads();
            const int bin = s.bin;
            const u64 left = s.left;
            // All of them from the border bin up, or that bin's alone.
            const bool whole = s.bin_end <= kShort;
            row.each([&](float x, int pos) {
                if (x >= floor) {
                    const int b = bin_of(x, inv);
                    if (b == bin || (whole && b < bin)) append(x, pos);
                }
            });
            __syncthreads();
            const uint32_t n = s.n;
            if (whole) {
                draw_from_list(a, r, s, set, weigh, n, want, top_p < 1.0f);
                return;
            }
            if (n <= kList) {
                if (static_cast<uint32_t>(tid) < n) {
                    const uint32_t mine = s.list[tid];
                    uint32_t above = 0, equal = 0;
#pragma unroll 8
                    for (uint32_t i = 0; i < n; ++i) {
                        const uint32_t o = s.list[i];
                        above += o > mine;
                        equal += o == mine;
                    }
                    if (above < left && above + equal >= left) {
                        s.key = mine;
                        s.ties = static_cast<uint32_t>(left) - above;
                    }
                }
                __syncthreads();
                thr = key_value(s.key);
                ties = s.ties;
            } else {
                ties = static_cast<uint32_t>(radix(want, [](float) { return u64{1}; }));
            }
            __syncthreads();
            for (int i = tid; i < kBins; i += kSampleThreads) {
                s.count[i] = 0;
                s.weight[i] = 0;
            }
            if (tid == 0) s.n = 0;
            __syncthreads();
        } else {
            __syncthreads();
            for (int i = tid; i < kBins; i += kSampleThreads) s.count[i] = 0;
            __syncthreads();
        }
    }

    if (top_p < 1.0f) {
        const float inv = weight_bins<kBins>(weigh);
        // The last bin holds most of a row at a low temperature: one add a thread.
        u64 rest = 0;
        uint32_t rest_n = 0;
        auto count = [&](float x, u64 w) {
            if (!(x > thr && x >= weigh.least)) return;
            const int b = bin_of(x, inv);
            if (b == kBins - 1) {
                rest += w;
                ++rest_n;
            } else {
                atomicAdd(&s.weight[b], w);
                atomicAdd(&s.count[b], 1u);
            }
        };
        if (weigh.endless) {
            row.each([&](float x, int) { count(x, weigh.whole(x)); });
        } else {
            row.batches([&](const float4 (&v)[Row<HELD>::U], int) {
#pragma unroll
                for (int i = 0; i < Row<HELD>::U; i += 2) {
                    const float x[8] = {v[i].x,     v[i].y,     v[i].z,     v[i].w,
                                        v[i + 1].x, v[i + 1].y, v[i + 1].z, v[i + 1].w};
                    float hi = x[0];
#pragma unroll
                    for (int e = 1; e < 8; ++e) hi = fmaxf(hi, x[e]);
                    if (!__ballot(hi > thr && hi >= weigh.least)) continue;
                    u64 w[8];
                    weigh.whole_eight(x, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) count(x[e], w[e]);
                }
            });
        }
        if (rest_n) {
            atomicAdd(&s.weight[kBins - 1], rest);
            atomicAdd(&s.count[kBins - 1], rest_n);
        }
        if (tid == 0 && ties) {
            const int b = bin_of(thr, inv);
            atomicAdd(&s.weight[b], ties * weigh.whole(thr));
            atomicAdd(&s.count[b], ties);
        }
        __syncthreads();
        u64 bins[E], sum_w = 0, total = 0;
        uint32_t counts[E], sum_n = 0, all = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            bins[i] = s.weight[E * tid + i];
            counts[i] = s.count[E * tid + i];
            sum_w += bins[i];
            sum_n += counts[i];
        }
        u64 before = block_prefix(sum_w, s.part64, total);
        uint32_t n_before = block_prefix(sum_n, s.part_n, all);
        const u64 target = max(u64{1}, share_up(total, fmaxf(top_p, 0.0f)));
#pragma unroll
        for (int i = 0; i < E; ++i) {
            n_before += counts[i];
            if (before < target && before + bins[i] >= target) {
                s.bin = E * tid + i;
                s.left = target - before;
                s.bin_end = n_before;
            }
            before += bins[i];
        }
        __syncthreads();
        const int bin = s.bin;
        const u64 left = s.left;
        const bool whole = k == 0 && s.bin_end <= kShort;
        // Logits that the border bin cannot hold, by a margin for the roundings of
        // its formula, are passed over (not where the bounds are no numbers).
        const float slack = 4e-7f * (fabsf(top) + (kBins + 1) / inv);
        float from = bin == kBins - 1 ? -INFINITY : top - (bin + 1) / inv - slack;
        float to = whole ? INFINITY : top - bin / inv + slack;
        from = from == from ? from : -INFINITY;
        to = to == to ? to : INFINITY;
        row.each([&](float x, int pos) {
            if (x >= from && x <= to && x >= thr && x >= weigh.least && x > -INFINITY) {
                const int b = bin_of(x, inv);
                if (b == bin || (whole && b < bin)) append(x, pos);
            }
        });
        __syncthreads();
        const uint32_t n = s.n;
        if (n <= kList) {
            nucleus_end(s, weigh, n, [&](uint32_t key) { return bin_of(key_value(key), inv) == bin; },
                        left, thr, ties);
            if (whole) {
                // What stays of the list: those above the last kept, and it.
                uint32_t above = 0;
                if (static_cast<uint32_t>(tid) < n) above = s.list[tid] > s.key;
                const uint32_t kept_above = __syncthreads_count(above);
                draw_from_list(a, r, s, set, weigh, n, kept_above + ties, false);
                return;
            }
        } else {
            const u64 rest = radix(target, [&](float x) { return weigh.whole(x); });
            const u64 w = max(u64{1}, weigh.whole(thr));
            ties = static_cast<uint32_t>((rest + w - 1) / w);
        }
    }

    const float cut = cut_of(set, weigh);
    auto kept = [&](float x) {  // the weight of a token that top-k and top-p keep
        const double w = weigh(x);
        return w >= min_p ? w : 0.0;
    };
    const double wt = thr > -INFINITY ? kept(thr) : 0.0;

    // Each wave's kept weight above the threshold and its tokens at it.
    uint32_t at_thr = 0;
    if (once && !weigh.endless) {
        sum = most > -INFINITY ? sum * weigh(most) : 0.0;
    } else if (weigh.endless) {
        sum = 0.0;
        row.each([&](float x, int) {
            if (x > thr && x >= cut) sum += kept(x);
            at_thr += x == thr && ties;
        });
    } else {
        sum = 0.0;
        row.batches([&](const float4 (&v)[Row<HELD>::U], int) {
#pragma unroll
            for (int i = 0; i < Row<HELD>::U; i += 2) {
                const float x[8] = {v[i].x,     v[i].y,     v[i].z,     v[i].w,
                                    v[i + 1].x, v[i + 1].y, v[i + 1].z, v[i + 1].w};
                uint32_t in = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    in |= x[e] > thr && x[e] >= cut ? 1u << e : 0;
                    at_thr += x[e] == thr && ties;
                }
                if (!__ballot(in)) continue;
                // Few: each lane its next one at a time (256 x 131072 with min-p of
                // 0.005 60 us, with eight a lane always 70; top-k of 1000 of 16 x
                // 160000 70 and 85; 56 x 16848 where most pass top-p 30.0 and 29.4).
                if (__popcll(__ballot(in & (in - 1))) <= 8) {
                    while (__ballot(in)) {
                        const uint32_t bit = in & (0u - in);
                        float y = x[0];
#pragma unroll
                        for (int e = 1; e < 8; ++e) y = bit == 1u << e ? x[e] : y;
                        const double w = weigh(y);
                        sum += in && w >= min_p ? w : 0.0;
                        in &= in - 1;
                    }
                    continue;
                }
                double w[8];
                weigh.several(x, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += in >> e & 1 && w[e] >= min_p ? w[e] : 0.0;
            }
        });
    }
    sum = last_lane(wave_scan(sum));
    at_thr = last_lane(wave_scan(at_thr));
    __syncthreads();
    if (lane == 0) {
        s.part[wave] = sum;
        s.part_n[wave] = at_thr;
    }
    __syncthreads();
    // The first wave whose running sum passes the target (the last with any
    // weight where rounding leaves none), a lane a wave.
    const bool is_wave = lane < kSampleWaves;
    const uint32_t n_here = is_wave ? s.part_n[lane] : 0, n_before = wave_scan(n_here) - n_here;
    const uint32_t n_kept = min(n_here, ties - min(ties, n_before));
    double total = 0.0, target = 0.0;
    const int pick = pick_run(is_wave ? s.part[lane] + n_kept * wt : 0.0, set.draw, total, target);
    const uint32_t left = ties - min(ties, __shfl(n_before, pick, kWave));
    // Of that wave's run of the row, positions as indexes.
    const int span = row.chunks * kChunk;
    draw_in_run(a, r, s, [&](int i) { return row.at(i + row.pre); }, max(0, pick * span - row.pre),
                min(a.vocab, (pick + 1) * span - row.pre), kept, cut, thr, left, wt, target, total);
}

template <bool HELD>
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ SampleShared<HELD ? kHeldBins : kWideBins> s;
    extern __shared__ __attribute__((aligned(16))) float held[];
    sample_row<HELD>(a, blockIdx.x, s, held);
}

// --- few rows of a large vocabulary: a row over several workgroups ------------------
//
// The same steps, a launch each, every row in slices of consecutive logits
// (blockIdx.x, a workgroup of 256 threads each), the histograms added up in
// the caller's scratch by integer atomics, and a last launch of one workgroup a
// row that draws. Rows that this does not fit (a logit of +inf, a border bin of
// more than kList) are done by that workgroup alone, as above. Calls without
// top-k only. 7 x 100003 with top-p: 3.8, 14, 8.9 and 17 us, waiting for the slices'
// atomics and, a workgroup a row, for its own reads and sums.

constexpr int kSliceThreads = 256;

struct SliceRow {
    u64 weight[kWideBins];
    uint32_t count[kWideBins];
    double sum[kMaxSlices];  // kept weights, but for the border bin's
    float top[kMaxSlices];
    int first[kMaxSlices];  // lowest index of the slice's maximum
    uint32_t list[kList];
    int list_at[kList];
    uint32_t n, pad[3];
};

struct SliceArgs {
    SampleArgs a;
    SliceRow* rows;
    int slices, length;
};

enum RowKind { kNothing, kGreedy, kPlain, kTopP, kAlone };

// What the slices' maxima say of the row.
struct SliceView {
    float top;
    int first;
    RowKind kind;
    // By wave: a lane a slice, so that the loads are in flight together.
    __device__ SliceView(const SliceArgs& b, const SliceRow& row, const Settings& set) {
        const int i = min(static_cast<int>(threadIdx.x % kWave), b.slices - 1);
        const float t = row.top[i];
        top = wave_top(t);
        first = wave_least(t == top ? row.first[i] : 0x7fffffff);
        kind = top == -INFINITY  ? kNothing
               : set.greedy      ? kGreedy
               : top == INFINITY ? kAlone
               : set.top_p < 1.0f ? kTopP
                                  : kPlain;
    }
};

// The slice's maximum; clears the row's histogram.
__global__ __launch_bounds__(kSliceThreads) void slice_top_kernel(SliceArgs b) {
    __shared__ float hi[kSliceThreads / kWave];
    __shared__ int at[kSliceThreads / kWave];
    const int s = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid % kWave;
    const float* x = b.a.logits + r * b.a.stride;
    SliceRow& row = b.rows[r];
    const int begin = s * b.length, end = min(begin + b.length, b.a.vocab);
    float top = -INFINITY;
    int first = 0x7fffffff;
#pragma unroll 8
    for (int i = begin + tid; i < end; i += kSliceThreads) {
        const float v = clean(x[i]);
        first = v > top ? i : first;
        top = fmaxf(top, v);
    }
    float m = wave_top(top);
    int f = top == m ? first : 0x7fffffff;
    f = wave_least(f);
    if (lane == 0) {
        hi[tid / kWave] = m;
        at[tid / kWave] = f;
    }
    for (int i = s * kSliceThreads + tid; i < kWideBins; i += b.slices * kSliceThreads) {
        row.weight[i] = 0;
        row.count[i] = 0;
    }
    if (s == 0 && tid == 0) row.n = 0;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kSliceThreads / kWave; ++i) {
            if (hi[i] > m || (hi[i] == m && at[i] < f)) f = at[i];
            m = fmaxf(m, hi[i]);
        }
        row.top[s] = m;
        row.first[s] = f;
    }
}

__device__ __forceinline__ double block_sum64(double v, double* part) {
    v = last_lane(wave_scan(v));
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// The slice's part of the row's histogram, or the sum of its weights.
__global__ __launch_bounds__(kSliceThreads) void slice_count_kernel(SliceArgs b) {
    __shared__ u64 weight[kWideBins];
    __shared__ uint32_t count[kWideBins];
    __shared__ double roots[2 * kRoots];
    __shared__ double part[kSliceThreads / kWave];
    const int s = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
    const SampleArgs& a = b.a;
    SliceRow& row = b.rows[r];
    const Settings set(a, r);
    const SliceView view(b, row, set);
    if (view.kind == kNothing || view.kind == kGreedy || view.kind == kAlone) return;
    if (tid < 2 * kRoots) roots[tid] = kRoot[tid];
    for (int i = tid; i < kWideBins; i += kSliceThreads) {
        weight[i] = 0;
        count[i] = 0;
    }
    __syncthreads();
    const Weigh weigh = weigh_of(a, set, view.top, roots);
    const float* x = a.logits + r * a.stride;
    const int begin = s * b.length, end = min(begin + b.length, a.vocab);
    if (view.kind == kPlain) {
        const float cut = cut_of(set, weigh);
        double sum = 0.0;
#pragma unroll 4
        for (int i = begin + tid; i < end; i += kSliceThreads) {
            const float v = clean(x[i]);
            if (v >= cut) {
                const double w = weigh(v);
                sum += w >= set.min_p ? w : 0.0;
            }
        }
        sum = block_sum64(sum, part);
        if (tid == 0) row.sum[s] = sum;
        return;
    }
    const float inv = weight_bins<kWideBins>(weigh);
    u64 rest = 0;  // the last bin's, one add a thread
    uint32_t rest_n = 0;
#pragma unroll 4
    for (int i = begin + tid; i < end; i += kSliceThreads) {
        const float v = clean(x[i]);
        if (v >= weigh.least) {
            const int bin = bin_at<kWideBins>(v, view.top, inv);
            const u64 w = weigh.whole(v);
            if (bin == kWideBins - 1) {
                rest += w;
                ++rest_n;
            } else {
                atomicAdd(&weight[bin], w);
                atomicAdd(&count[bin], 1u);
            }
        }
    }
    if (rest_n) {
        atomicAdd(&weight[kWideBins - 1], rest);
        atomicAdd(&count[kWideBins - 1], rest_n);
    }
    __syncthreads();
    for (int i = tid; i < kWideBins; i += kSliceThreads) {
        if (!count[i]) continue;
        atomicAdd(&row.count[i], count[i]);
        if (weight[i]) atomicAdd(&row.weight[i], weight[i]);
    }
}

// The bin at which top-p ends, from the row's histogram, by a
// workgroup of THREADS; part: two sums a wave.
struct Border {
    int bin;
    uint32_t count;  // tokens up to and with the bin
    u64 left;        // what is wanted of the bin's weight
};
template <int THREADS>
__device__ __forceinline__ Border border_of(const SliceRow& row, const Settings& set,
                                            u64 (&part)[2 * THREADS / kWave], Border* out) {
    constexpr int E = kWideBins / THREADS;
    const int tid = threadIdx.x, wave = tid / kWave;
    u64 w[E], sum = 0;
    uint32_t n[E], all = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        n[i] = row.count[E * tid + i];
        w[i] = row.weight[E * tid + i];
        sum += w[i];
        all += n[i];
    }
    const u64 scan = wave_scan(sum);
    const uint32_t scan_n = wave_scan(all);
    if (tid % kWave == kWave - 1) {
        part[2 * wave] = scan;
        part[2 * wave + 1] = scan_n;
    }
    __syncthreads();
    u64 before = scan - sum, total = 0;
    uint32_t count = scan_n - all;
#pragma unroll
    for (int i = 0; i < THREADS / kWave; ++i) {
        before += i < wave ? part[2 * i] : 0;
        count += i < wave ? static_cast<uint32_t>(part[2 * i + 1]) : 0;
        total += part[2 * i];
    }
    const u64 target = max(u64{1}, share_up(total, fmaxf(set.top_p, 0.0f)));
#pragma unroll
    for (int i = 0; i < E; ++i) {
        count += n[i];
        if (before < target && before + w[i] >= target) *out = Border{E * tid + i, count, target - before};
        before += w[i];
    }
    __syncthreads();
    return *out;
}

// The tokens of the border bin, or of all bins up to it where they are few;
// the sum of the slice's weights above it.
__global__ __launch_bounds__(kSliceThreads) void slice_list_kernel(SliceArgs b) {
    __shared__ double roots[2 * kRoots];
    __shared__ double part[kSliceThreads / kWave];
    __shared__ u64 part64[2 * kSliceThreads / kWave];
    __shared__ Border border;
    const int s = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
    const SampleArgs& a = b.a;
    SliceRow& row = b.rows[r];
    const Settings set(a, r);
    const SliceView view(b, row, set);
    if (view.kind != kTopP) return;
    if (tid < 2 * kRoots) roots[tid] = kRoot[tid];
    const Border end_at = border_of<kSliceThreads>(row, set, part64, &border);
    const Weigh weigh = weigh_of(a, set, view.top, roots);
    const bool whole = end_at.count <= kShort;
    const float inv = weight_bins<kWideBins>(weigh), cut = cut_of(set, weigh);
    const float* x = a.logits + r * a.stride;
    const int begin = s * b.length, end = min(begin + b.length, a.vocab);
    double sum = 0.0;
#pragma unroll 4
    for (int i = begin + tid; i < end; i += kSliceThreads) {
        const float v = clean(x[i]);
        if (!(v >= weigh.least)) continue;
        const int bin = bin_at<kWideBins>(v, view.top, inv);
        if (bin == end_at.bin || (whole && bin < end_at.bin)) {
            const uint32_t n = atomicAdd(&row.n, 1u);
            if (n < kList) {
                row.list[n] = order_key(v);
                row.list_at[n] = i;
            }
        } else if (bin < end_at.bin && v >= cut) {
            const double w = weigh(v);
            sum += w >= set.min_p ? w : 0.0;
        }
    }
    sum = block_sum64(sum, part);
    if (tid == 0) row.sum[s] = sum;
}

__global__ __launch_bounds__(kSampleThreads) void slice_draw_kernel(SliceArgs b) {
    __shared__ SampleShared<kWideBins> s;
    __shared__ u64 part64[2 * kSampleWaves];
    __shared__ Border border;
    const SampleArgs& a = b.a;
    const int r = blockIdx.x, tid = threadIdx.x;
    const SliceRow& row = b.rows[r];
    const Settings set(a, r);
    const SliceView view(b, row, set);
    if (view.kind == kNothing || view.kind == kGreedy) {
        if (tid == 0) {
            a.tokens[r] = view.kind == kGreedy ? view.first : -1;
            if (a.logprobs) a.logprobs[r] = view.kind == kGreedy ? 0.0f : -INFINITY;
        }
        return;
    }
    bool alone = view.kind == kAlone;
    Border end_at{};
    uint32_t n = 0;
    if (view.kind == kTopP) {
        end_at = border_of<kSampleThreads>(row, set, part64, &border);
        n = row.n;
        alone = n > kList;
    }
    if (alone) {
        __syncthreads();
        sample_row<false>(a, r, s, nullptr);
        return;
    }
    if (tid < 2 * kRoots) s.roots[tid] = kRoot[tid];
    if (tid == 0) {
        s.token = kSampleThreads;
        s.last = -1;
    }
    if (static_cast<uint32_t>(tid) < n) {
        s.list[tid] = row.list[tid];
        s.list_at[tid] = row.list_at[tid];
    }
    __syncthreads();
    const Weigh weigh = weigh_of(a, set, view.top, s.roots);
    float thr = -INFINITY;
    uint32_t ties = 0;
    const float cut = cut_of(set, weigh);
    auto kept = [&](float v) {
        const double w = weigh(v);
        return w >= set.min_p ? w : 0.0;
    };
    if (view.kind == kTopP) {
        const float inv = weight_bins<kWideBins>(weigh);
        nucleus_end(s, weigh, n,
                    [&](uint32_t key) { return bin_at<kWideBins>(key_value(key), view.top, inv) == end_at.bin; },
                    end_at.left, thr, ties);
        // The list by rank, so that the sums do not depend on its order.
        uint32_t key = 0, rank = 0, above = 0;
        int pos = 0;
        if (static_cast<uint32_t>(tid) < n) {
            key = s.list[tid];
            pos = s.list_at[tid];
            above = key > s.key;
#pragma unroll 8
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t o = s.list[i];
                const int at = s.list_at[i];
                rank += (o > key) | ((o == key) & (at < pos));
            }
        }
        const uint32_t kept_above = __syncthreads_count(above);
        if (end_at.count <= kShort) {
            draw_from_list(a, r, s, set, weigh, n, kept_above + ties, false);
            return;
        }
        n = kept_above + ties;  // of the list, by rank
        __syncthreads();  // the list has been read
        if (key && rank < n) {
            s.list_at[rank] = pos;
            s.weight[rank] = __double_as_longlong(kept(key_value(key)));
        }
        __syncthreads();
    }
    const double wt = ties ? kept(thr) : 0.0;
    // Slice sums with the list's kept tokens, a wave a slice, in a fixed pattern.
    for (int i = tid / kWave; i < b.slices; i += kSampleWaves) {
        const int begin = i * b.length, end = begin + b.length;
        double sum = 0.0;
        for (uint32_t y = tid % kWave; y < n; y += kWave) {
            const int at = s.list_at[y];
            sum += at >= begin && at < end ? __longlong_as_double(s.weight[y]) : 0.0;
        }
        sum = last_lane(wave_scan(sum));
        if (tid % kWave == 0) s.sums[i] = row.sum[i] + sum;
    }
    __syncthreads();
    double total = 0.0, target = 0.0;
    const int lane = tid % kWave;
    const int pick = pick_run(lane < b.slices ? s.sums[lane] : 0.0, set.draw, total, target);
    const int begin = pick * b.length;
    // Tokens at the threshold that slices before this one keep.
    uint32_t left = ties;
    if (ties)
        for (uint32_t i = n - ties; i < n; ++i) left -= s.list_at[i] < begin;
    const float* x = a.logits + r * a.stride;
    draw_in_run(a, r, s, [&](int i) { return clean(x[i]); }, begin, min(begin + b.length, a.vocab), kept,
                cut, thr, left, wt, target, total);
}

// Chunks a wave of the row kernel, for a row up to three floats off its 16 bytes.
int row_chunks(std::size_t vocab) {
    return ceil_div(static_cast<long long>(vocab) + 3, kSampleWaves * kChunk);
}

// Slices a row takes, 1: the row kernel, which has rows that LDS holds and many
// of them. us, row kernel / slices, top-p of 0.9: 1 x 32000 35 / 37, 1 x 50000
// 60 / 33, 32 x 50000 62 / 59, 1 x 100003 106 / 36, 7 x 100003 107 / 43, 32 x
// 100003 107 / 64, 64 x 100003 107 / 111; no filter: 41 / 17 at 1 x 100003, 25 /
// 28 at 64 x 50000. Not with a top-k, which leaves the row kernel little to do
// after its histogram: 39 / 48 at 7 x 100003, 15 / 27 at 1 x 32000. Of 2048
// logits and more: half as many take 40 at 1 x 100003.
int slices_of(std::size_t rows, std::size_t vocab) {
    if (row_chunks(vocab) <= kHeldChunks || rows > vocab / 2048) return 1;
    return static_cast<int>(std::min<std::size_t>({kMaxSlices, vocab / 2048, 512 / rows}));
}

std::size_t sample_scratch(std::size_t rows, std::size_t vocab) {
    return slices_of(rows, vocab) > 1 ? rows * sizeof(SliceRow) : 0;
}

void run_slices(const SampleArgs& a, int slices, void* scratch, hipStream_t stream) {
    SliceArgs b{a, static_cast<SliceRow*>(scratch), slices, 0};
    b.length = (ceil_div(a.vocab, slices) + kSliceThreads - 1) / kSliceThreads * kSliceThreads;
    b.slices = ceil_div(a.vocab, b.length);
    const dim3 grid(b.slices, a.rows), block(kSliceThreads);
    hipLaunchKernelGGL(slice_top_kernel, grid, block, 0, stream, b);
    hipLaunchKernelGGL(slice_count_kernel, grid, block, 0, stream, b);
    if (a.top_p) hipLaunchKernelGGL(slice_list_kernel, grid, block, 0, stream, b);
    hipLaunchKernelGGL(slice_draw_kernel, dim3(a.rows), dim3(kSampleThreads), 0, stream, b);
}

void run_sample(const SampleArgs& a, void* scratch, hipStream_t stream) {
    const int slices = slices_of(static_cast<std::size_t>(a.rows), static_cast<std::size_t>(a.vocab));
    if (slices > 1 && !a.top_k) {
        run_slices(a, slices, scratch, stream);
        return;
    }
    const int chunks = row_chunks(static_cast<std::size_t>(a.vocab));
    if (chunks <= kHeldChunks)
        hipLaunchKernelGGL(sample_row_kernel<true>, dim3(a.rows), dim3(kSampleThreads),
                           chunks * kSampleWaves * kChunk * sizeof(float), stream, a);
    else
        hipLaunchKernelGGL(sample_row_kernel<false>, dim3(a.rows), dim3(kSampleThreads), 0, stream, a);
}

}  // namespace
}  // namespace em

using em::fail;

extern "C" {

size_t em_sample_scratch_bytes(size_t rows, size_t vocab) {
    if (rows > (size_t{1} << 20) || vocab > static_cast<size_t>(em::kMaxVocab)) return 0;
    return em::sample_scratch(rows, vocab);
}

int em_sample(size_t rows, size_t vocab, const float* logits, size_t logits_stride, const float* u,
              const em_sampling* settings, int* tokens, float* logprobs, void* scratch,
              void* stream) {
    if (rows > (size_t{1} << 20)) return fail(EM_EINVAL, "sample: more than 2^20 rows");
    if (vocab == 0 || vocab > static_cast<size_t>(em::kMaxVocab))
        return fail(EM_EINVAL, "sample: a vocabulary of 1 to 2^20");
    if (rows > 1 && (logits_stride < vocab || logits_stride >= (size_t{1} << 40)))
        return fail(EM_EINVAL, "sample: logits_stride smaller than the vocabulary");
    if (!settings) return fail(EM_EINVAL, "sample: null settings");
    if (rows == 0) return EM_OK;
    const size_t need = em::sample_scratch(rows, vocab);
    if (!logits || !u || !tokens || (need && !scratch))
        return fail(EM_EINVAL, "sample: null pointer");
    if (need && reinterpret_cast<uintptr_t>(scratch) % 16)
        return fail(EM_EINVAL, "sample: scratch must be 16-byte aligned");
    if (!em::device_present()) return fail(EM_ENODEV, "sample: no usable GPU");
    try {
        em::SampleArgs a{};
        a.rows = static_cast<int>(rows);
        a.vocab = static_cast<int>(vocab);
        int log2 = 0;
        while ((size_t{1} << log2) < vocab) ++log2;
        a.bits = std::min(52, 62 - log2);
        a.logits = logits;
        a.stride = static_cast<long long>(logits_stride);
        a.u = u;
        a.temperature = settings->temperature;
        a.top_k = settings->top_k;
        a.top_p = settings->top_p;
        a.min_p = settings->min_p;
        a.tokens = tokens;
        a.logprobs = logprobs;
        em::run_sample(a, scratch, static_cast<hipStream_t>(stream));
        em::hip_check(hipGetLastError(), "launch");
    } catch (const std::exception& e) {
        return fail(EM_EDEVICE, e.what());
    }
    return EM_OK;
}

}  // extern "C"
