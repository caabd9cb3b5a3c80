// Sampling: the next token of each row of logits by temperature, top-k,
// top-p and min-p from a given uniform number.
//
// A token's weight w = exp((x - max) / T) is formed in 64 bits, so that which
// side of a border u falls on is off by some 2^-50 of the sum, where fp32 sums
// of 100000 weights lose 2^-20 of it. Where weights are added by atomics, in an
// order that changes, they are integers, round(w 2^bits) with bits = 62 -
// ceil(log2 vocab): the row's sum stays below 2^63 and is always the same.
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
constexpr int kList = 512;  // tokens of a bin that are ranked against each other

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

// 2^(i / 16).
__device__ constexpr double kRoots[16] = {
    1.0,                1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
    1.1892071150027210, 1.2418578120734840, 1.2968395546510096, 1.3542555469368927,
    1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
    1.6817928305074290, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

// A row's weights relative to its maximum: w = 2^(z / 16), z = (x - top) *
// 16 log2 e / T: a root from the table, the rest by its Taylor series (the
// first term left out is below 2^-51).
struct Weigh {
    float top;
    double c;  // 16 log2 e / T
    int bits;
    const double* roots;  // kRoots in LDS
    __device__ __forceinline__ double operator()(float x) const {
        const double d = x == top ? 0.0 : static_cast<double>(x) - static_cast<double>(top);
        const double z = fmax(d * c, -65536.0);  // 2^-4096 is 0
        const double n = rint(z);
        const double y = (z - n) * (0.69314718055994530942 / 16);
        double p = fma(y, 1.0 / 720.0, 1.0 / 120.0);
        p = fma(p, y, 1.0 / 24.0);
        p = fma(p, y, 1.0 / 6.0);
        p = fma(p, y, 0.5);
        p = fma(p, y, 1.0);
        p = fma(p, y, 1.0);
        const int i = static_cast<int>(n);
        return ldexp(p * roots[i & 15], i >> 4);
    }
    __device__ __forceinline__ u64 whole(float x) const {
        return static_cast<u64>(rint(ldexp((*this)(x), bits)));
    }
};

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
    u64 weight[kBins];
    uint32_t count[kBins];
    u64 list_w[kList];
    uint32_t list[kList];
    double roots[16];
    double part[kSampleWaves];
    u64 part64[kSampleWaves];
    float part_hi[kSampleWaves], part_lo[kSampleWaves];
    uint32_t part_n[kSampleWaves];
    uint32_t n, key, ties;
    u64 left;
    int token, last;
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
        return i >= 0 && i < vocab ? clean(x[i]) : -INFINITY;
    }
    __device__ __forceinline__ float4 load4(int pos) const {
        if (pos >= pre && pos + 4 <= pre + vocab) {
            const float4 v = *reinterpret_cast<const float4*>(x + (pos - pre));
            return make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
        }
        return make_float4(load(pos), load(pos + 1), load(pos + 2), load(pos + 3));
    }
    __device__ __forceinline__ float at(int pos) const {
        if constexpr (HELD) return held[pos];
        return load(pos);
    }
    // f(x) of every logit of this thread; KEEP: the pass that fills `held`.
    template <bool KEEP = false, class Fn>
    __device__ __forceinline__ void each(Fn f) const {
        constexpr int U = 4;  // vectors in flight
        for (int c = 0; c < chunks; c += U) {
            float4 v[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int pos = position(min(c + i, chunks - 1));
                if constexpr (HELD && !KEEP)
                    v[i] = *reinterpret_cast<const float4*>(held + pos);
                else
                    v[i] = load4(pos);
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (c + i >= chunks) break;
                if constexpr (HELD && KEEP)
                    *reinterpret_cast<float4*>(held + position(c + i)) = v[i];
                f(v[i].x);
                f(v[i].y);
                f(v[i].z);
                f(v[i].w);
            }
        }
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
    if (tid < 16) s.roots[tid] = kRoots[tid];

    // The maximum, and the least of the threads' maxima.
    float most = -INFINITY;
    row.template each<true>([&](float x) { most = fmaxf(most, x); });
    float top = wave_max(most), low = -wave_max(-most);
    if (lane == 0) {
        s.part_hi[wave] = top;
        s.part_lo[wave] = low;
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
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    const bool greedy = !(T > 0.0f);
    const Weigh weigh{top, greedy ? 0.0 : 16 * 1.4426950408889634074 / T, a.bits, s.roots};

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
            row.each([&](float x) {
                const uint32_t k = order_key(x);
                if (x > -INFINITY && (shift == 24 || k >> (shift + 8) == prefix))
                    atomicAdd(&s.weight[k >> shift & 255], amount(x));
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
    // The bin in which the running sum reaches `target` and what is left of
    // it there; two bins a thread.
    auto border = [&](const auto& bins, auto* part, u64 target, u64& left) {
        const auto b0 = bins[2 * tid], b1 = bins[2 * tid + 1];
        auto total = b0;
        const u64 before = block_prefix(b0 + b1, part, total);
        if (before < target && before + b0 + b1 >= target) {
            const bool second = before + b0 < target;
            s.n = 2 * tid + second;
            s.left = target - before - (second ? b0 : 0);
        }
        __syncthreads();
        const int bin = s.n;
        left = s.left;
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        return bin;
    };

    const int k = a.top_k ? a.top_k[r] : 0;
    if (greedy) {
        thr = top;
        ties = 1;
    } else if (k > 0 && k < a.vocab) {
        // Where every thread has a maximum, k of them are at least the least
        // one, so only tokens from there on need be counted.
        float floor = low;
        if (low == -INFINITY || k > kSampleThreads) {
            float least = INFINITY;
            row.each([&](float x) { least = x > -INFINITY ? fminf(least, x) : least; });
            least = -wave_max(-least);
            __syncthreads();
            if (lane == 0) s.part_lo[wave] = least;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kSampleWaves; ++i) least = fminf(least, s.part_lo[i]);
            floor = least;
        }
        const float inv = fminf((kBins - 1) / (top - floor), 3e38f);
        for (int i = tid; i < kBins; i += kSampleThreads) s.count[i] = 0;
        __syncthreads();
        row.each([&](float x) {
            if (x >= floor) atomicAdd(&s.count[bin_of(x, inv)], 1u);
        });
        __syncthreads();
        u64 left = 0;
        uint32_t all = 0;
        // Fewer tokens than k that can be drawn: the filter is off.
        (void)block_prefix(s.count[2 * tid] + s.count[2 * tid + 1], s.part_n, all);
        if (all >= static_cast<uint32_t>(k)) {
            const int bin = border(s.count, s.part_n, k, left);
            row.each([&](float x) {
                if (x >= floor && bin_of(x, inv) == bin) {
                    const uint32_t i = atomicAdd(&s.n, 1u);
                    if (i < kList) s.list[i] = order_key(x);
                }
            });
            __syncthreads();
            const uint32_t n = s.n;
            if (n <= kList) {
                if (static_cast<uint32_t>(tid) < n) {
                    const uint32_t mine = s.list[tid];
                    uint32_t above = 0, equal = 0;
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
                ties = static_cast<uint32_t>(radix(k, [](float) { return u64{1}; }));
            }
        }
    }

    const float top_p = a.top_p ? a.top_p[r] : 1.0f;
    if (!greedy && top_p < 1.0f) {
        // Bins of 1/64 of a factor of two in weight, the last one from 2^-32.
        const float inv = static_cast<float>(fmin(weigh.c * (64.0 / 16.0), 3e38));
        __syncthreads();
        for (int i = tid; i < kBins; i += kSampleThreads) s.weight[i] = 0;
        __syncthreads();
        row.each([&](float x) {
            if (x > thr) {
                const u64 w = weigh.whole(x);
                if (w) atomicAdd(&s.weight[bin_of(x, inv)], w);
            }
        });
        if (tid == 0 && ties) atomicAdd(&s.weight[bin_of(thr, inv)], ties * weigh.whole(thr));
        __syncthreads();
        u64 total = 0, left = 0;
        (void)block_prefix(s.weight[2 * tid] + s.weight[2 * tid + 1], s.part64, total);
        u64 target = static_cast<u64>(
            ceil(static_cast<double>(fmaxf(top_p, 0.0f)) * static_cast<double>(total)));
        target = max(u64{1}, min(target, total));
        const int bin = border(s.weight, s.part64, target, left);
        row.each([&](float x) {
            if (x >= thr && x > -INFINITY && bin_of(x, inv) == bin) {
                const u64 w = weigh.whole(x);
                if (w) {
                    const uint32_t i = atomicAdd(&s.n, 1u);
                    if (i < kList) {
                        s.list[i] = order_key(x);
                        s.list_w[i] = w;
                    }
                }
            }
        });
        __syncthreads();
        const uint32_t n = s.n;
        if (n <= kList) {
            if (static_cast<uint32_t>(tid) < n) {
                const uint32_t mine = s.list[tid];
                const u64 w = s.list_w[tid];
                u64 above = 0;
                uint32_t equal = 0;
                for (uint32_t i = 0; i < n; ++i) {
                    above += s.list[i] > mine ? s.list_w[i] : 0;
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
        } else {
            const u64 rest = radix(target, [&](float x) { return weigh.whole(x); });
            const u64 w = max(u64{1}, weigh.whole(thr));
            ties = static_cast<uint32_t>((rest + w - 1) / w);
        }
    }
    const float mp = a.min_p ? a.min_p[r] : 0.0f;
    const double min_p = mp > 0.0f ? fmin(static_cast<double>(mp), 1.0) : 0.0;
    auto kept = [&](float x) {  // the weight of a token that top-k and top-p keep
        const double w = weigh(x);
        return w >= min_p ? w : 0.0;
    };
    const double wt = thr > -INFINITY ? kept(thr) : 0.0;

    // Each wave's kept weight above the threshold and its tokens at it.
    double sum = 0.0;
    uint32_t at_thr = 0;
    row.each([&](float x) {
        if (x > thr) sum += kept(x);
        at_thr += x == thr && ties;
    });
    sum = shfl(wave_scan(sum), kWave - 1);
    at_thr = shfl(wave_scan(at_thr), kWave - 1);
    __syncthreads();
    if (lane == 0) {
        s.part[wave] = sum;
        s.part_n[wave] = at_thr;
    }
    if (tid == 0) s.token = s.last = -1;
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
    const float u = a.u[r];
    double target = u > 0.0f ? fmin(static_cast<double>(u), 1.0) * total : 0.0;
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
        if (x > thr) mine += kept(x);
        n += x == thr && ties;
    }
    uint32_t dummy_n = 0;
    const uint32_t n_before = block_prefix(n, s.part_n, dummy_n);
    uint32_t here = left > n_before ? min(left - n_before, n) : 0;
    mine += here * wt;
    double dummy = 0.0;
    const double before = block_prefix(mine, s.part, dummy);
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
            w = kept(x);
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
        a.bits = 62 - log2;
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
