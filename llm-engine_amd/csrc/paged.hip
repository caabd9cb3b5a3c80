// The paged KV cache: host-side checks of its operators, and the append of
// new rows with RoPE on the way.
#include <cmath>

#include "paged.hpp"

namespace em {

std::string paged_reject(const em_paged_shape& s) {
    if (s.n_heads <= 0 || s.n_kv_heads <= 0 || s.n_heads % s.n_kv_heads != 0)
        return "paged: n_heads must be a positive multiple of n_kv_heads";
    if (s.n_heads > 4096) return "paged: more than 4096 heads";
    if (s.head_size <= 0 || s.head_size > 256 || s.head_size % 8)
        return "paged: head_size must be a multiple of 8, at most 256";
    if (s.page_size <= 0 || s.n_pages <= 0 || s.max_pages <= 0)
        return "paged: page_size, n_pages and max_pages must be positive";
    if (static_cast<long long>(s.page_size) * s.max_pages > (1LL << 30))
        return "paged: a sequence of more than 2^30 positions";
    if (s.type != EM_CACHE_F32 && s.type != EM_CACHE_F16 && s.type != EM_CACHE_BF16)
        return "paged: unknown cache type";
    if (s.page_stride % 8 || s.slot_stride % 8 || s.head_stride % 8)
        return "paged: strides must be multiples of 8";
    constexpr std::size_t kMaxCache = std::size_t{1} << 34;
    const auto hs = static_cast<std::size_t>(s.head_size);
    if ((s.n_pages > 1 && s.page_stride < hs) || (s.page_size > 1 && s.slot_stride < hs) ||
        (s.n_kv_heads > 1 && s.head_stride < hs))
        return "paged: a stride smaller than head_size";
    // Offsets in units of eight elements are kept in 32 bits.
    std::size_t a = 0, b = 0, c = 0;
    if (__builtin_mul_overflow(static_cast<std::size_t>(s.n_pages), s.page_stride, &a) ||
        __builtin_mul_overflow(static_cast<std::size_t>(s.page_size), s.slot_stride, &b) ||
        __builtin_mul_overflow(static_cast<std::size_t>(s.n_kv_heads), s.head_stride, &c) ||
        a >= kMaxCache || b >= kMaxCache || c >= kMaxCache || a + b + c >= kMaxCache)
        return "paged: caches past 2^34 elements";
    return "";
}

std::string paged_batch_reject(const em_paged_shape& s, const em_paged_batch& b,
                               std::size_t rows) {
    if (b.n_seqs < 0 || b.n_seqs > (1 << 20)) return "paged: 0 to 2^20 sequences";
    if (rows > (std::size_t{1} << 22)) return "paged: more than 2^22 rows";
    if (b.n_seqs == 0 || rows == 0) return "";
    if (!b.row_start || !b.lengths || !b.page_table) return "paged: null batch pointer";
    if (b.table_stride < static_cast<std::size_t>(s.max_pages) ||
        b.table_stride >= (std::size_t{1} << 40))
        return "paged: table_stride smaller than max_pages";
    return "";
}

namespace {

struct AppendArgs {
    PagedArgs p;
    const float *q, *k, *v;
    const float* freq;
    float* q_out;
    void *kc, *vc;
    long long q_stride, k_stride, v_stride, q_out_stride;
    int rotary, halves;
};

// Cosine and sine of an angle formed in 64 bits, rounded to fp32 once: the
// angle less the nearest multiple of pi / 2 (held as a sum of two doubles, so
// that 2^31 quarter turns leave the remainder good to 2^-75), then the Taylor
// series of both, whose first terms left out are below 2^-36 of the sum's
// leading term at pi / 4, and the quarter's signs.
__device__ __forceinline__ void cos_sin(double angle, float& c, float& s) {
    constexpr double kTwoOverPi = 0.63661977236758134308;
    constexpr double kHi = 1.57079632679489661923, kLo = 6.12323399573676603587e-17;
    const double n = rint(angle * kTwoOverPi);
    double x = fma(-n, kHi, angle);
    x = fma(-n, kLo, x);
    const double z = x * x;
    double ps = -1.0 / 39916800.0;
    ps = fma(ps, z, 1.0 / 362880.0);
    ps = fma(ps, z, -1.0 / 5040.0);
    ps = fma(ps, z, 1.0 / 120.0);
    ps = fma(ps, z, -1.0 / 6.0);
    const double sn = fma(ps * z, x, x);
    double pc = 1.0 / 479001600.0;
    pc = fma(pc, z, -1.0 / 3628800.0);
    pc = fma(pc, z, 1.0 / 40320.0);
    pc = fma(pc, z, -1.0 / 720.0);
    pc = fma(pc, z, 1.0 / 24.0);
    pc = fma(pc, z, -0.5);
    const double cn = fma(pc, z, 1.0);
    const int quarter = static_cast<int>(static_cast<long long>(n)) & 3;
    const float fs = static_cast<float>(sn), fc = static_cast<float>(cn);
    const float a = quarter & 1 ? fs : fc, b = quarter & 1 ? fc : fs;
    c = (quarter == 1 || quarter == 2) ? -a : a;
    s = quarter >= 2 ? -b : b;
}

template <class T>
__device__ __forceinline__ void store4(T* dst, float a, float b, float c, float d) {
    typedef T vec __attribute__((ext_vector_type(4)));
    *reinterpret_cast<vec*>(dst) = vec{static_cast<T>(a), static_cast<T>(b), static_cast<T>(c),
                                       static_cast<T>(d)};
}

// Row blockIdx.x. A thread owns one unit of eight head dims (four pairs: two
// runs of four dims half a rotation apart, or one run of eight) of every
// step-th head of q, k and v, so its four angles are formed once for all of
// them; heads are spread over blockIdx.y where there are few rows. Bound by bytes
// (7167 rows of 32 + 32 + 32 heads of 128 into fp16: 114 us, 5.15 TB/s, a copy's
// rate), for few rows by three reads that depend on each other (64 rows of 32 + 8
// + 8: 4.2 us).
template <class T>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(AppendArgs a) {
    const PagedArgs& p = a.p;
    const int r = blockIdx.x, seq = row_sequence(p, r);
    if (seq < 0) return;
    const long long at =
        p.lengths[seq] - (static_cast<long long>(p.row_start[seq + 1]) - r);
    if (at < 0 || at >= static_cast<long long>(p.max_pages) * p.page_size) return;
    const int pos = static_cast<int>(at);
    const long long slot = slot_offset(p, seq, pos);

    const int units = p.head_size / 8, per = kThreads / units;
    const int unit = threadIdx.x % units, first = threadIdx.x / units;
    if (first >= per) return;
    const int heads = (a.q ? p.n_heads : 0), kv = p.n_kv_heads;
    // The unit's two runs of four dims; rot: rotated.
    const bool rot = unit < a.rotary / 8;
    const int d0 = rot && a.halves ? 4 * unit : 8 * unit;
    const int d1 = rot && a.halves ? d0 + a.rotary / 2 : d0 + 4;
    float c[4], s[4];
    if (rot) {
        const floatx4 f = *reinterpret_cast<const floatx4*>(a.freq + 4 * unit);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            cos_sin(static_cast<double>(pos) * static_cast<double>(f[i]), c[i], s[i]);
    }
    for (int h = first + per * blockIdx.y; h < heads + 2 * kv; h += per * gridDim.y) {
        const bool is_q = h < heads, is_k = !is_q && h < heads + kv;
        const float* src = is_q   ? a.q + r * a.q_stride + h * p.head_size
                           : is_k ? a.k + r * a.k_stride + (h - heads) * p.head_size
                                  : a.v + r * a.v_stride + (h - heads - kv) * p.head_size;
        if (!is_q && slot < 0) continue;
        // A value row's unit is the same pair of runs, unrotated.
        floatx4 x = *reinterpret_cast<const floatx4*>(src + d0);
        floatx4 y = *reinterpret_cast<const floatx4*>(src + d1);
        if (rot && (is_q || is_k)) {
            if (a.halves) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 z = rope_pair(x[i], y[i], c[i], s[i]);
                    x[i] = z.x;
                    y[i] = z.y;
                }
            } else {
                const float2 z0 = rope_pair(x[0], x[1], c[0], s[0]);
                const float2 z1 = rope_pair(x[2], x[3], c[1], s[1]);
                const float2 z2 = rope_pair(y[0], y[1], c[2], s[2]);
                const float2 z3 = rope_pair(y[2], y[3], c[3], s[3]);
                x = floatx4{z0.x, z0.y, z1.x, z1.y};
                y = floatx4{z2.x, z2.y, z3.x, z3.y};
            }
        }
        if (is_q) {
            float* dst = a.q_out + r * a.q_out_stride + h * p.head_size;
            *reinterpret_cast<floatx4*>(dst + d0) = x;
            *reinterpret_cast<floatx4*>(dst + d1) = y;
        } else {
            const int g = is_k ? h - heads : h - heads - kv;
            T* dst = static_cast<T*>(is_k ? a.kc : a.vc) + slot + g * p.head_stride;
            store4<T>(dst + d0, x[0], x[1], x[2], x[3]);
            store4<T>(dst + d1, y[0], y[1], y[2], y[3]);
        }
    }
}

void run_paged_append(const AppendArgs& a, int type, hipStream_t stream) {
    const int per = kThreads / (a.p.head_size / 8);
    const int heads = (a.q ? a.p.n_heads : 0) + 2 * a.p.n_kv_heads;
    // Heads are spread until the grid covers the CUs.
    const int most = ceil_div(heads, per), want = ceil_div(cu_count(), a.p.rows);
    const dim3 grid(a.p.rows, std::min(most, std::max(1, want))), block(kThreads);
    if (type == EM_CACHE_F32)
        hipLaunchKernelGGL(paged_append_kernel<float>, grid, block, 0, stream, a);
    else if (type == EM_CACHE_F16)
        hipLaunchKernelGGL(paged_append_kernel<_Float16>, grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL(paged_append_kernel<__bf16>, grid, block, 0, stream, a);
}

bool a16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace em

using em::fail;

extern "C" {

int em_paged_check(const em_paged_shape* s) {
    if (!s) return fail(EM_EINVAL, "paged: null shape");
    const std::string why = em::paged_reject(*s);
    return why.empty() ? EM_OK : fail(EM_EINVAL, why);
}

int em_paged_append(const em_paged_shape* s, const em_paged_batch* b, size_t rows, const float* q,
                    size_t q_stride, const float* k, size_t k_stride, const float* v,
                    size_t v_stride, const float* freq, int rotary, int halves, float* q_out,
                    size_t q_out_stride, void* key_cache, void* value_cache, void* stream) {
    if (const int rc = em_paged_check(s)) return rc;
    if (!b) return fail(EM_EINVAL, "paged_append: null batch");
    const std::string why = em::paged_batch_reject(*s, *b, rows);
    if (!why.empty()) return fail(EM_EINVAL, why);
    if (rotary < 0 || rotary > s->head_size || rotary % 8)
        return fail(EM_EINVAL, "paged_append: rotary must be a multiple of 8, at most head_size");
    if (rows == 0 || b->n_seqs == 0) return EM_OK;
    if (!k || !v || !key_cache || !value_cache || (q && !q_out) || (rotary && !freq))
        return fail(EM_EINVAL, "paged_append: null pointer");
    const size_t dim = static_cast<size_t>(s->n_heads) * s->head_size;
    const size_t kv = static_cast<size_t>(s->n_kv_heads) * s->head_size;
    const size_t most = size_t{1} << 32;
    auto bad = [&](size_t stride, size_t width) {
        return stride % 4 || stride >= most || (rows > 1 && stride < width);
    };
    if ((q && (bad(q_stride, dim) || bad(q_out_stride, dim))) || bad(k_stride, kv) ||
        bad(v_stride, kv))
        return fail(EM_EINVAL, "paged_append: row strides must be multiples of 4, no smaller "
                               "than a row");
    if ((q && (!em::a16(q) || !em::a16(q_out))) || !em::a16(k) || !em::a16(v) ||
        (rotary && !em::a16(freq)) || !em::a16(key_cache) || !em::a16(value_cache))
        return fail(EM_EINVAL, "paged_append: pointers must be 16-byte aligned");
    if (!em::device_present()) return fail(EM_ENODEV, "paged_append: no usable GPU");
    try {
        em::AppendArgs a{};
        a.p = em::paged_args(*s, *b, rows);
        a.q = q;
        a.k = k;
        a.v = v;
        a.freq = freq;
        a.q_out = q_out;
        a.kc = key_cache;
        a.vc = value_cache;
        a.q_stride = static_cast<long long>(q_stride);
        a.k_stride = static_cast<long long>(k_stride);
        a.v_stride = static_cast<long long>(v_stride);
        a.q_out_stride = static_cast<long long>(q_out_stride);
        a.rotary = rotary;
        a.halves = halves != 0;
        em::run_paged_append(a, s->type, static_cast<hipStream_t>(stream));
        em::hip_check(hipGetLastError(), "launch");
    } catch (const std::exception& e) {
        return fail(EM_EDEVICE, e.what());
    }
    return EM_OK;
}

}  // extern "C"
