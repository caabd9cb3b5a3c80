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
// rows of up to 32765 are read once, into LDS, longer ones once a pass.
#include <algorithm>
#include <cmath>

#include "internal.hpp"
#include "llm_engine_amd.h"

namespace em {
namespace {

using u64 = unsigned long long;
constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / kWave;
constexpr int kChunk = 4 * kWave;  // logits a wave reads at once
constexpr int kMaxVocab = 1 << 20;
constexpr int kBins = 2048;
constexpr int kList = 512;   // tokens of a bin that are ranked against each other
constexpr int kShort = 128;  // a list that holds all that may be kept

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
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }
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
// (9 ns per 1024 weights a CU with floor, ldexp and a 16-entry table: 14).
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

// A share in [0, 1) of a sum of weights, exactly: rounded down, and up.
__device__ __forceinline__ u64 share_down(u64 total, float share) {
    return __umul64hi(total, static_cast<u64>(static_cast<double>(share) * 0x1p64));
}
__device__ __forceinline__ u64 share_up(u64 total, float share) {
    const u64 f = static_cast<u64>(static_cast<double>(share) * 0x1p64);
    return __umul64hi(total, f) + (total * f != 0);
}

template <class T>
__device__ __forceinline__ T wave_scan(T v) {  // inclusive
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const T o = __shfl_up(v, d, kWave);
        if (lane >= d) v += o;
    }
    return v;
}

struct SampleShared {
    u64 weight[kBins];  // the bins'; once they have been read, the list's
    uint32_t count[kBins];
    uint32_t list[kList];
    int list_at[kList];
    double roots[2 * kRoots];
    double part[kSampleWaves];
    u64 part64[kSampleWaves];
    float part_hi[kSampleWaves], part_lo[kSampleWaves];
    uint32_t part_n[kSampleWaves];
    uint32_t n, key, ties, bin, bin_end;
    u64 left;
    int token, last, keep;
};

// Chunks a wave whose row LDS (160 KB) holds beside SampleShared.
constexpr int kHeldChunks = 8;
static_assert(sizeof(SampleShared) + kHeldChunks * kSampleWaves * kChunk * sizeof(float) <= 160 * 1024);

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

template <bool HELD>
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ SampleShared s;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    extern __shared__ __attribute__((aligned(16))) float held[];
    Row<HELD> row;
    row.held = held;
    row.x = a.logits + r * a.stride;
    row.vocab = a.vocab;
    row.pre = static_cast<int>(reinterpret_cast<uintptr_t>(row.x) / 4 % 4);
    row.chunks = (a.vocab + row.pre + kSampleWaves * kChunk - 1) / (kSampleWaves * kChunk);
    if (tid < 2 * kRoots) s.roots[tid] = kRoot[tid];
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    const bool greedy = !(T > 0.0f);
    const int k = a.top_k && a.top_k[r] < a.vocab ? max(0, a.top_k[r]) : 0;
    const float top_p = a.top_p ? a.top_p[r] : 1.0f;
    const float mp = a.min_p ? a.min_p[r] : 0.0f;
    const double min_p = mp > 0.0f ? fmin(static_cast<double>(mp), 1.0) : 0.0;
    const float u = a.u[r];
    const double draw = u > 0.0f ? fmin(static_cast<double>(u), 1.0) : 0.0;

    // The maximum, and the least of the threads' maxima.
    float most = -INFINITY;
    const double c = greedy ? 0.0 : kRoots * 1.4426950408889634074 / T;
    // A long row without a filter is read once: its weights are summed beside
    // the maximum, relative to the thread's own so far.
    const bool once = !HELD && !greedy && k == 0 && !(top_p < 1.0f) && !(mp > 0.0f);
    double sum = 0.0;
    if (once) {
        __syncthreads();  // the roots
        row.batches([&](const float4 (&v)[Row<HELD>::U], int) {
            float m = most;
#pragma unroll
            for (int i = 0; i < Row<HELD>::U; ++i)
                m = fmaxf(fmaxf(m, fmaxf(v[i].x, v[i].y)), fmaxf(v[i].z, v[i].w));
            const Weigh weigh{m, false, static_cast<float>(m - 60.0 * T), c, a.bits, s.roots};
            if (__ballot(m > most)) sum *= m > most ? weigh(most) : 1.0;
#pragma unroll
            for (int i = 0; i < Row<HELD>::U; ++i)
                sum += (weigh(v[i].x) + weigh(v[i].y)) + (weigh(v[i].z) + weigh(v[i].w));
            most = m;
        });
    } else {
        row.template each<true>([&](float x, int) { most = fmaxf(most, x); });
    }
    float top = wave_max(most), low = -wave_max(-most);
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
        s.token = s.last = -1;
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
    const Weigh weigh{top, top == INFINITY, static_cast<float>(top - 60.0 * T), c, a.bits, s.roots};

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
    // The histogram's bin of x; inv: bins over the range they cover.
    auto bin_of = [&](float x, float inv) {
        const float b = x == top ? 0.0f : (top - x) * inv;
        return b < kBins - 1 ? static_cast<int>(b) : kBins - 1;
    };
    // Appends a token to the list (s.n counts past its end too).
    auto append = [&](float x, int pos) {
        const uint32_t i = atomicAdd(&s.n, 1u);
        if (i < kList) {
            s.list[i] = order_key(x);
            s.list_at[i] = pos;
        }
    };

    // Every token that may be kept is in the list: ranks them, keeps the
    // highest most_kept of them, of those what top-p (nucleus) and min-p leave,
    // which are some of the highest ranks too, and draws.
    auto draw_from_list = [&](uint32_t n, uint32_t most_kept, bool nucleus) {
        uint32_t key = 0, rank = 0;
        int pos = 0;
        const bool mine = static_cast<uint32_t>(tid) < n;
        if (mine) {
            key = s.list[tid];
            pos = s.list_at[tid];
#pragma unroll 8
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t o = s.list[i];
                rank += o > key || (o == key && s.list_at[i] < pos);
            }
        }
        n = min(n, most_kept);
        const bool in = mine && rank < n;
        const float x = key_value(key);
        const double w = in ? weigh(x) : 0.0;
        const u64 ww = in ? weigh.whole(x) : 0;
        if (tid == 0) s.keep = n;
        __syncthreads();  // the list has been read
        if (in) {
            s.weight[rank] = ww;
            s.list_at[rank] = pos;
        }
        __syncthreads();
        if (in) {
            u64 before = 0, total = 0;
#pragma unroll 8
            for (uint32_t i = 0; i < n; ++i) {
                const u64 o = s.weight[i];
                before += i < rank ? o : 0;
                total += o;
            }
            if (nucleus) {
                const u64 target = max(u64{1}, share_up(total, fmaxf(top_p, 0.0f)));
                if (rank > 0 && before >= target) atomicMin(&s.keep, static_cast<int>(rank));
            }
            if (w < min_p) atomicMin(&s.keep, static_cast<int>(rank));
        }
        __syncthreads();
        const uint32_t keep = s.keep;
        if (!in || rank >= keep) return;
        u64 before = 0, total = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < keep; ++i) {
            const u64 o = s.weight[i];
            before += s.list_at[i] < pos ? o : 0;
            total += o;
        }
        const u64 target = draw < 1.0 ? share_down(total, static_cast<float>(draw)) : total - 1;
        if (before <= target && before + ww > target) {
            a.tokens[r] = pos - row.pre;
            if (a.logprobs)
                a.logprobs[r] = static_cast<float>(log(ldexp(w, a.bits) / static_cast<double>(total)));
        }
    };

    if (greedy) {
        // The lowest index of the maximum.
        int first = 0x7fffffff;
        row.each([&](float x, int pos) { first = x == top ? min(first, pos) : first; });
        if (tid == 0) s.keep = 0x7fffffff;
        __syncthreads();
        if (first < 0x7fffffff) atomicMin(&s.keep, first);
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
            least = -wave_max(-least);
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
        const uint32_t b0 = s.count[2 * tid], b1 = s.count[2 * tid + 1];
        uint32_t all = 0;
        const uint32_t want = k, before = block_prefix(b0 + b1, s.part_n, all);
        // Fewer tokens than k that can be drawn: the filter is off.
        if (all >= want) {
            if (before < want && before + b0 + b1 >= want) {
                const bool second = before + b0 < want;
                s.bin = 2 * tid + second;
                s.left = want - before - (second ? b0 : 0);
                s.bin_end = before + b0 + (second ? b1 : 0);
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
                draw_from_list(n, want, top_p < 1.0f);
                return;
            }
            if (n <= kList) {
                if (static_cast<uint32_t>(tid) < n) {
                    const uint32_t mine = s.list[tid];
                    uint32_t above = 0, equal = 0;
#pragma unroll 8
                    for (uint32_t i = 0; i < n; ++i) {
                        above += s.list[i] > mine;
                        equal += s.list[i] == mine;
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
            s.count[2 * tid] = s.count[2 * tid + 1] = 0;
            __syncthreads();
        }
    }

    if (top_p < 1.0f) {
        // Bins of 1/64 of a factor of two in weight, the last one from 2^-32.
        const float inv = static_cast<float>(fmin(weigh.c * (64.0 / kRoots), 3e38));
        row.each([&](float x, int) {
            if (x > thr && x >= weigh.least) {
                const int b = bin_of(x, inv);
                atomicAdd(&s.weight[b], weigh.whole(x));
                atomicAdd(&s.count[b], 1u);
            }
        });
        if (tid == 0 && ties) {
            const int b = bin_of(thr, inv);
            atomicAdd(&s.weight[b], ties * weigh.whole(thr));
            atomicAdd(&s.count[b], ties);
        }
        __syncthreads();
        const u64 b0 = s.weight[2 * tid], b1 = s.weight[2 * tid + 1];
        const uint32_t n0 = s.count[2 * tid], n1 = s.count[2 * tid + 1];
        u64 total = 0;
        uint32_t all = 0;
        const u64 before = block_prefix(b0 + b1, s.part64, total);
        const uint32_t n_before = block_prefix(n0 + n1, s.part_n, all);
        const u64 target = max(u64{1}, share_up(total, fmaxf(top_p, 0.0f)));
        if (before < target && before + b0 + b1 >= target) {
            const bool second = before + b0 < target;
            s.bin = 2 * tid + second;
            s.left = target - before - (second ? b0 : 0);
            s.bin_end = n_before + n0 + (second ? n1 : 0);
        }
        __syncthreads();
        const int bin = s.bin;
        const u64 left = s.left;
        const bool whole = k == 0 && s.bin_end <= kShort;
        row.each([&](float x, int pos) {
            if (x >= thr && x >= weigh.least && x > -INFINITY) {
                const int b = bin_of(x, inv);
                if (b == bin || (whole && b < bin)) append(x, pos);
            }
        });
        __syncthreads();
        const uint32_t n = s.n;
        if (n <= kList) {
            uint32_t mine = 0;
            u64 w = 0;
            if (static_cast<uint32_t>(tid) < n) {
                mine = s.list[tid];
                w = weigh.whole(key_value(mine));
                s.weight[tid] = w;
            }
            __syncthreads();
            // In the border bin: a token's weight counts from the bins above.
            if (static_cast<uint32_t>(tid) < n && bin_of(key_value(mine), inv) == bin && w) {
                u64 above = 0;
                uint32_t equal = 0;
#pragma unroll 8
                for (uint32_t i = 0; i < n; ++i) {
                    const bool here = !whole || bin_of(key_value(s.list[i]), inv) == bin;
                    above += here && s.list[i] > mine ? s.weight[i] : 0;
                    equal += s.list[i] == mine;
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
            if (whole) {
                // What stays of the list: those above the last kept, and it.
                uint32_t above = 0;
                if (static_cast<uint32_t>(tid) < n) above = s.list[tid] > s.key;
                uint32_t kept_above = 0;
                (void)block_prefix(above, s.part_n, kept_above);
                draw_from_list(n, kept_above + ties, false);
                return;
            }
        } else {
            const u64 rest = radix(target, [&](float x) { return weigh.whole(x); });
            const u64 w = max(u64{1}, weigh.whole(thr));
            ties = static_cast<uint32_t>((rest + w - 1) / w);
        }
    }

    // No logit below `cut` weighs min_p (a thousandth of T and the fp32
    // roundings of the sum are left for the comparison in 64 bits).
    const float cut = weigh.endless ? -INFINITY : min_p > 0.0 ? static_cast<float>(top + (log(min_p) - 1e-3) * T -
                                                       1e-6 * fabs(static_cast<double>(top)))
                                  : weigh.least;
    auto kept = [&](float x) {  // the weight of a token that top-k and top-p keep
        const double w = weigh(x);
        return w >= min_p ? w : 0.0;
    };
    const double wt = thr > -INFINITY ? kept(thr) : 0.0;

    // Each wave's kept weight above the threshold and its tokens at it.
    uint32_t at_thr = 0;
    if (once && !weigh.endless) {
        sum = most > -INFINITY ? sum * weigh(most) : 0.0;
    } else {
        sum = 0.0;
        row.each([&](float x, int) {
            if (x > thr && x >= cut) sum += kept(x);
            at_thr += x == thr && ties;
        });
    }
    sum = __shfl(wave_scan(sum), kWave - 1, kWave);
    at_thr = __shfl(wave_scan(at_thr), kWave - 1, kWave);
    __syncthreads();
    if (lane == 0) {
        s.part[wave] = sum;
        s.part_n[wave] = at_thr;
    }
    __syncthreads();
    double total = 0.0;
    {
        uint32_t left = ties;
#pragma unroll
        for (int i = 0; i < kSampleWaves; ++i) {
            const uint32_t n = min(left, s.part_n[i]);
            left -= n;
            total += s.part[i] + n * wt;
        }
    }
    double target = draw * total;
    int pick = 0;
    uint32_t left = ties;
    {
        // The first wave whose running sum passes the target (the last with
        // any weight where rounding leaves none).
        double run = 0.0, pick_run = 0.0;
        uint32_t l = ties;
        bool found = false;
#pragma unroll
        for (int i = 0; i < kSampleWaves; ++i) {
            const uint32_t n = min(l, s.part_n[i]);
            const double w = s.part[i] + n * wt;
            if (!found && w > 0.0) {
                pick = i;
                pick_run = run;
                left = l;
                found = run + w > target;
            }
            l -= n;
            run += w;
        }
        target -= pick_run;
    }
    // That wave's run of the row, `each` consecutive logits a thread.
    const int span = row.chunks * kChunk, each = (span + kSampleThreads - 1) / kSampleThreads;
    const int from = pick * span + tid * each, to = min(from + each, (pick + 1) * span);
    double mine = 0.0;
    uint32_t n = 0;
    for (int p = from; p < to; ++p) {
        const float x = row.at(p);
        if (x > thr && x >= cut) mine += kept(x);
        n += x == thr && ties;
    }
    uint32_t all_n = 0;
    const uint32_t n_before = block_prefix(n, s.part_n, all_n);
    uint32_t here = left > n_before ? min(left - n_before, n) : 0;
    mine += here * wt;
    double all = 0.0;
    const double before = block_prefix(mine, s.part, all);
    const bool hit = mine > 0.0 && before <= target && before + mine > target;
    if (hit) s.token = 1;
    if (mine > 0.0) atomicMax(&s.last, tid);
    __syncthreads();
    // The scan's rounding may leave a gap that the target falls into: the
    // last thread with any weight then takes it.
    if (!(hit || (s.token < 0 && tid == s.last))) return;
    double run = before;
    int token = -1;
    double w_token = 0.0;
    for (int p = from; p < to; ++p) {
        const float x = row.at(p);
        double w = 0.0;
        if (x > thr) {
            if (x >= cut) w = kept(x);
        } else if (x == thr && here > 0) {
            --here;
            w = wt;
        }
        if (!(w > 0.0)) continue;
        token = p - row.pre;
        w_token = w;
        run += w;
        if (run > target) break;
    }
    a.tokens[r] = token;
    if (a.logprobs) a.logprobs[r] = static_cast<float>(log(w_token / total));
}

std::size_t sample_scratch(std::size_t, std::size_t) { return 0; }

void run_sample(const SampleArgs& a, hipStream_t stream) {
    // Rows that fit LDS beside the rest, up to three floats off their 16 bytes.
    const int per = kSampleWaves * kChunk, chunks = (a.vocab + 3 + per - 1) / per;
    if (chunks <= kHeldChunks)
        hipLaunchKernelGGL(sample_row_kernel<true>, dim3(a.rows), dim3(kSampleThreads),
                           chunks * per * sizeof(float), stream, a);
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
        em::run_sample(a, static_cast<hipStream_t>(stream));
        em::hip_check(hipGetLastError(), "launch");
    } catch (const std::exception& e) {
        return fail(EM_EDEVICE, e.what());
    }
    return EM_OK;
}

}  // extern "C"
