// Attention of a batch's rows over a paged KV cache.
#include <cmath>

#include "paged.hpp"

namespace em {
namespace {

struct PagedAttnArgs {
    PagedArgs p;
    const float* q;
    const void *kc, *vc;
    float* out;
    long long q_stride, out_stride;
    float scale;
    int window;
};

template <class T>
__device__ __forceinline__ float value_of(T x) {
    return static_cast<float>(x);
}

// Row blockIdx.x, head blockIdx.y: 256 positions at a time, a score a thread,
// then a head dim a thread over their values. Positions the row does not see
// are never read.
template <class T>
__global__ __launch_bounds__(kThreads) void paged_row_kernel(PagedAttnArgs a) {
    const PagedArgs& p = a.p;
    __shared__ float q_s[256];
    __shared__ float w_s[kThreads];
    __shared__ long long off_s[kThreads];
    __shared__ float part[4];
    const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, D = p.head_size;
    const int seq = row_sequence(p, r);
    if (seq < 0) return;
    const long long pos = p.lengths[seq] - (static_cast<long long>(p.row_start[seq + 1]) - r);
    const long long limit = static_cast<long long>(p.max_pages) * p.page_size;
    const int end = static_cast<int>(max(0LL, min(pos + 1, limit)));
    const int first = a.window ? static_cast<int>(min(limit, max(0LL, pos + 1 - a.window))) : 0;
    const T* kc = static_cast<const T*>(a.kc) + (h / p.group) * p.head_stride;
    const T* vc = static_cast<const T*>(a.vc) + (h / p.group) * p.head_stride;
    if (tid < D) q_s[tid] = a.q[r * a.q_stride + h * D + tid];
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int t0 = first; t0 < end; t0 += kThreads) {
        const int t = t0 + tid;
        const long long off = t < end ? slot_offset(p, seq, t) : -1;
        __syncthreads();
        float s = -INFINITY;
        if (off >= 0) {
            float dot = 0.0f;
            for (int d = 0; d < D; ++d) dot = fmaf(q_s[d], value_of(kc[off + d]), dot);
            s = dot * a.scale;
        }
        const float mn = fmaxf(m, block_max(s, part));
        const float alpha = mn == -INFINITY ? 1.0f : expf(m - mn);
        const float w = off < 0 || s == -INFINITY ? 0.0f : expf(s - mn);
        off_s[tid] = off;
        w_s[tid] = w;
        l = l * alpha + block_sum(w, part);  // its barriers publish the weights
        m = mn;
        o *= alpha;
        if (tid < D) {
            const int n = min(kThreads, end - t0);
            for (int i = 0; i < n; ++i)
                if (off_s[i] >= 0) o = fmaf(w_s[i], value_of(vc[off_s[i] + tid]), o);
        }
    }
    if (tid < D) a.out[r * a.out_stride + h * D + tid] = l == 0.0f ? 0.0f : o / l;
}

void run_paged_attention(const PagedAttnArgs& a, int type, hipStream_t stream) {
    const dim3 grid(a.p.rows, a.p.n_heads), block(kThreads);
    if (type == EM_CACHE_F32)
        hipLaunchKernelGGL(paged_row_kernel<float>, grid, block, 0, stream, a);
    else if (type == EM_CACHE_F16)
        hipLaunchKernelGGL(paged_row_kernel<_Float16>, grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL(paged_row_kernel<__bf16>, grid, block, 0, stream, a);
}

std::size_t paged_attention_scratch(const em_paged_shape&, std::size_t, std::size_t) { return 0; }

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
    if (window < 0) return fail(EM_EINVAL, "paged_attention: negative window");
    if (!std::isfinite(scale)) return fail(EM_EINVAL, "paged_attention: scale is not finite");
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
    try {
        em::PagedAttnArgs a{};
        a.p = em::paged_args(*s, *b, rows);
        a.q = q;
        a.kc = key_cache;
        a.vc = value_cache;
        a.out = out;
        a.q_stride = static_cast<long long>(q_stride);
        a.out_stride = static_cast<long long>(out_stride);
        a.scale = scale != 0.0f ? scale
                                : static_cast<float>(1.0 / std::sqrt(static_cast<double>(s->head_size)));
        a.window = window;
        em::run_paged_attention(a, s->type, static_cast<hipStream_t>(stream));
        em::hip_check(hipGetLastError(), "launch");
    } catch (const std::exception& e) {
        return fail(EM_EDEVICE, e.what());
    }
    return EM_OK;
}

}  // extern "C"
