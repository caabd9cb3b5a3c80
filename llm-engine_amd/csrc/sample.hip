// Sampling: the next token of each row of logits by temperature, top-k,
// top-p and min-p from a given uniform number.
//
// A token's weight w = exp((x - max) / T) is formed in 64 bits and summed as
// an integer, round(w 2^bits), bits = 62 - ceil(log2 vocab): the row's sum
// stays below 2^63, sums do not depend on the order they are formed in, and
// which side of a border u falls on is off by 2^-43 of a vocabulary's largest
// weight and less, where fp32 sums of 100000 weights lose 2^-20 of it.
//
// Both filters are thresholds on the logit: top-k's and top-p's last token
// kept is a value and a number of tokens of just that value, lowest index
// first, found by radix selection on the logits' ordered bits (top-k by
// counts, top-p by summed weights). The draw then adds the kept weights in
// index order.
#include <cmath>

#include "internal.hpp"
#include "llm_engine_amd.h"

namespace em {
namespace {

using u64 = unsigned long long;
constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / kWave;
constexpr int kSegment = 256;                 // values a wave takes at once
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxSegments = kMaxVocab / kSegment;

struct SampleArgs {
    int rows, vocab, bits;
    const float* logits;
    long long stride;
    const float *u, *temperature, *top_p, *min_p;
    const int* top_k;
    int* tokens;
    float* logprobs;
};

// A logit's bits in an order that is the values': -inf least, NaN as -inf, -0
// as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
    x = x == x ? x + 0.0f : -INFINITY;
    const uint32_t b = __float_as_uint(x);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t kLeastKey = 0x007fffffu;  // -inf's

// 2^z for z <= 0 in 64 bits: 2^f, |f| <= 1/2, by its Taylor series (the first
// term left out is below 2^-56), scaled by the whole part.
__device__ __forceinline__ double exp2_64(double z) {
    if (!(z > -1000.0)) return 0.0;
    const double n = rint(z), x = (z - n) * 0.69314718055994530942;
    double p = 1.0 / 6227020800.0;
    p = fma(p, x, 1.0 / 479001600.0);
    p = fma(p, x, 1.0 / 39916800.0);
    p = fma(p, x, 1.0 / 3628800.0);
    p = fma(p, x, 1.0 / 362880.0);
    p = fma(p, x, 1.0 / 40320.0);
    p = fma(p, x, 1.0 / 5040.0);
    p = fma(p, x, 1.0 / 720.0);
    p = fma(p, x, 1.0 / 120.0);
    p = fma(p, x, 1.0 / 24.0);
    p = fma(p, x, 1.0 / 6.0);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    p = fma(p, x, 1.0);
    return ldexp(p, static_cast<int>(n));
}

// A row's weights: of value v (its key not the least), relative to the row's
// maximum, T's reciprocal times log2 e in c.
struct Weigh {
    float top;
    double c;
    int bits;
    __device__ double exact(float v) const {
        if (v == top) return 1.0;  // +inf too
        return exp2_64((static_cast<double>(v) - static_cast<double>(top)) * c);
    }
    __device__ u64 whole(double w) const { return static_cast<u64>(rint(ldexp(w, bits))); }
    __device__ u64 operator()(uint32_t key) const {
        return key <= kLeastKey ? 0 : whole(exact(key_value(key)));
    }
};

__device__ __forceinline__ u64 shfl_up64(u64 v, int d) {
    const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), d, kWave);
    const uint32_t hi = __shfl_up(static_cast<uint32_t>(v >> 32), d, kWave);
    return static_cast<u64>(hi) << 32 | lo;
}
__device__ __forceinline__ u64 wave_scan64(u64 v) {  // inclusive
    const int lane = threadIdx.x % kWave;
    for (int d = 1; d < kWave; d *= 2) {
        const u64 o = shfl_up64(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// One workgroup a row.
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ u64 hist[256];
    __shared__ u64 seg_sum[kMaxSegments];
    __shared__ uint32_t seg_tie[kMaxSegments];
    __shared__ uint32_t s_key;
    __shared__ u64 s_left, s_total, s_target;
    __shared__ uint32_t s_ties;
    __shared__ int s_seg;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, V = a.vocab;
    const float* x = a.logits + r * a.stride;

    if (tid == 0) s_key = 0;
    __syncthreads();
    uint32_t mine = 0;
    for (int i = tid; i < V; i += kSampleThreads) mine = max(mine, order_key(x[i]));
    atomicMax(&s_key, mine);
    __syncthreads();
    const uint32_t top = s_key;
    if (top <= kLeastKey) {
        if (tid == 0) {
            a.tokens[r] = -1;
            if (a.logprobs) a.logprobs[r] = -INFINITY;
        }
        return;
    }
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    const bool greedy = !(T > 0.0f);
    const Weigh weigh{key_value(top), greedy ? 0.0 : 1.4426950408889634074 / T, a.bits};

    // The last token kept: value thr, `ties` of that value.
    uint32_t thr = kLeastKey + 1, ties = V;
    // Radix selection from the top: the value at which the running sum of
    // `amount` over falling values reaches `target`, and what is left of the
    // target for the tokens of just that value.
    auto select = [&](u64 target, auto amount) {
        uint32_t prefix = 0;
        u64 left = target;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += kSampleThreads) {
                const uint32_t k = order_key(x[i]);
                if (k > kLeastKey && (shift == 24 || k >> (shift + 8) == prefix))
                    atomicAdd(&hist[k >> shift & 255], amount(k));
            }
            __syncthreads();
            if (tid == 0) {
                u64 l = left;
                int b = 255;
                while (b > 0 && hist[b] < l) l -= hist[b--];
                s_left = l;
                s_key = prefix << 8 | b;
            }
            __syncthreads();
            prefix = s_key;
            left = s_left;
            __syncthreads();
        }
        thr = prefix;
        return left;
    };
    const int k = a.top_k ? a.top_k[r] : 0;
    if (greedy) {
        thr = top;
        ties = 1;
    } else if (k > 0 && k < V) {
        // Fewer than k tokens that can be drawn: the filter is off.
        if (tid == 0) s_total = 0;
        __syncthreads();
        u64 n = 0;
        for (int i = tid; i < V; i += kSampleThreads) n += order_key(x[i]) > kLeastKey;
        atomicAdd(&s_total, n);
        __syncthreads();
        const u64 all = s_total;
        __syncthreads();
        if (all > static_cast<u64>(k)) ties = select(k, [](uint32_t) { return u64{1}; });
    }
    const float top_p = a.top_p ? a.top_p[r] : 1.0f;
    if (!greedy && top_p < 1.0f) {
        if (tid == 0) s_total = 0;
        __syncthreads();
        u64 n = 0;
        for (int i = tid; i < V; i += kSampleThreads) {
            const uint32_t key = order_key(x[i]);
            if (key > thr) n += weigh(key);
        }
        atomicAdd(&s_total, n);
        // Every token of the threshold's value, up to the ties kept.
        if (tid == 0) s_ties = 0;
        __syncthreads();
        uint32_t c = 0;
        for (int i = tid; i < V; i += kSampleThreads) c += order_key(x[i]) == thr;
        atomicAdd(&s_ties, c);
        __syncthreads();
        const u64 total = s_total + min(ties, s_ties) * weigh(thr);
        __syncthreads();
        u64 target = static_cast<u64>(ceil(static_cast<double>(fmaxf(top_p, 0.0f)) *
                                           static_cast<double>(total)));
        target = max(u64{1}, min(target, total));
        const u64 left = select(target, weigh);
        const u64 w = max(u64{1}, weigh(thr));
        ties = static_cast<uint32_t>((left + w - 1) / w);
    }
    const float mp = a.min_p ? a.min_p[r] : 0.0f;
    const double min_p = mp > 0.0f ? fmin(static_cast<double>(mp), 1.0) : 0.0;
    auto kept = [&](uint32_t key) -> u64 {  // the weight of a token above the threshold
        if (key <= kLeastKey || key < thr) return 0;
        const double w = weigh.exact(key_value(key));
        return w >= min_p ? weigh.whole(w) : 0;
    };

    // Each segment's kept weight above the threshold and tokens at it.
    const int segs = (V + kSegment - 1) / kSegment;
    for (int s = tid / kWave; s < segs; s += kSampleWaves) {
        u64 sum = 0;
        uint32_t tie = 0;
        for (int i = 0; i < 4; ++i) {
            const int at = s * kSegment + 4 * lane + i;
            if (at >= V) continue;
            const uint32_t key = order_key(x[at]);
            if (key > thr) sum += kept(key);
            tie += key == thr;
        }
        sum = wave_scan64(sum);
        for (int d = 1; d < kWave; d *= 2) {
            const uint32_t o = __shfl_up(tie, d, kWave);
            if (lane >= d) tie += o;
        }
        if (lane == kWave - 1) {
            seg_sum[s] = sum;
            seg_tie[s] = tie;
        }
    }
    __syncthreads();
    const u64 wt = kept(thr);
    if (tid == 0) {
        u64 total = 0;
        uint32_t left = ties;
        for (int s = 0; s < segs; ++s) {
            const uint32_t n = min(left, seg_tie[s]);
            left -= n;
            total += seg_sum[s] + n * wt;
        }
        const float u = a.u[r];
        u64 target = u > 0.0f ? static_cast<u64>(static_cast<double>(u) * static_cast<double>(total)) : 0;
        target = min(target, total - 1);
        u64 sum = 0;
        left = ties;
        int s = 0;
        for (; s < segs - 1; ++s) {
            const uint32_t n = min(left, seg_tie[s]);
            const u64 w = seg_sum[s] + n * wt;
            if (sum + w > target) break;
            left -= n;
            sum += w;
        }
        s_seg = s;
        s_target = target - sum;
        s_ties = left;
        s_total = total;
    }
    __syncthreads();
    if (tid >= kWave) return;
    // The segment's values in order: one wave, four a lane.
    uint32_t key[4], tie[4], before = 0;
    for (int i = 0; i < 4; ++i) {
        const int at = s_seg * kSegment + 4 * lane + i;
        key[i] = at < V ? order_key(x[at]) : 0;
        tie[i] = key[i] == thr;
        before += tie[i];
    }
    uint32_t run = before;
    for (int d = 1; d < kWave; d *= 2) {
        const uint32_t o = __shfl_up(run, d, kWave);
        if (lane >= d) run += o;
    }
    run -= before;
    u64 w[4], sum = 0;
    for (int i = 0; i < 4; ++i) {
        w[i] = key[i] > thr ? kept(key[i]) : tie[i] && run < s_ties ? wt : 0;
        run += tie[i];
        sum += w[i];
    }
    u64 c = wave_scan64(sum) - sum;
    for (int i = 0; i < 4; ++i) {
        if (w[i] && c <= s_target && c + w[i] > s_target) {
            a.tokens[r] = s_seg * kSegment + 4 * lane + i;
            if (a.logprobs) {
                const double p = ldexp(weigh.exact(key_value(key[i])), a.bits);
                a.logprobs[r] = static_cast<float>(log(p / static_cast<double>(s_total)));
            }
        }
        c += w[i];
    }
}

std::size_t sample_scratch(std::size_t, std::size_t) { return 0; }

void run_sample(const SampleArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(sample_row_kernel, dim3(a.rows), dim3(kSampleThreads), 0, stream, a);
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
