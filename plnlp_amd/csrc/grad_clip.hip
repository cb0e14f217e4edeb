// The global norm of a list of gradients, and the gradients clipped by it, without a word to the host.
//   N = (sum |g|^p)^(1/p) for p = 1, 2, or max |g|;   c = min(1, max_norm / (N + 1e-6));   dst = c * src
// Bound by bytes: every gradient is read for the norm and, where c < 1 or dst is another tensor, read again and written.
//   pass 1 (norm_kernel):  each workgroup reduces one chunk of one tensor in f64 and stores ONE partial.  f64 because a square
//     of an f32 above 1.8e19 (below 1e-23) leaves f32's range and a sum over 1e9 elements loses its small terms; the f64 pipe
//     has ten times the rate the bytes come at.
//     684 M bf16 elements in 73 tensors: 272 us, 5.0 TB/s.
//   pass 2 (clip_kernel):  each workgroup adds ALL partials in the same fixed order (a few KiB out of L2), so c needs no launch
//     of its own, no counter and no atomic: the same bits every run, and nothing that two streams or two graphs could share.
//     The same tensors into others of their type: 535 us, 5.1 TB/s read and written (a copy of 2 GiB: 4.9).
// The tensors travel in the kernel's arguments (CLIP_LAUNCH a launch), so a captured graph holds them by value.
#include "half.hip.h"

namespace plnlp {

constexpr int CLIP_LAUNCH = 128;          // 128 * 29 B of table: below the 4 KiB of arguments a launch may carry
constexpr int CLIP_THREADS = 256;
constexpr int64_t CLIP_BLOCKS = 2048;     // workgroups a pass aims at: 8 per CU, what 256 threads of < 64 registers fill
constexpr int64_t CLIP_MIN_CHUNK = 4096;  // elements: two 16-byte loads a thread
constexpr int64_t CLIP_PARTIALS = 4096;   // partials beyond which one workgroup adds them up once, for all

struct ClipTable {
    const void* src[CLIP_LAUNCH];
    void*       dst[CLIP_LAUNCH];
    int64_t     n[CLIP_LAUNCH];
    int32_t     first[CLIP_LAUNCH];       // first workgroup of the tensor
    uint8_t     types[CLIP_LAUNCH];       // src | dst << 4
    int32_t     count;
    int64_t     chunk;
};

__device__ __forceinline__ int clip_tensor(const ClipTable& t, int block) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= block) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int KIND> __device__ __forceinline__ double norm_join(double a, double b) {
    if (KIND != PLNLP_NORM_MAX) return a + b;
    return (b > a || b != b) ? b : a;             // NaN wins, as in a sum
}
template <int KIND> __device__ __forceinline__ double norm_term(double s, float x) {
    const double d = (double)x;
    if (KIND == PLNLP_NORM_L2) return fma(d, d, s);
    return norm_join<KIND>(s, fabs(d));
}

// the workgroup's value in thread 0 (fixed order)
template <int KIND> __device__ __forceinline__ double norm_block(double s) {
    __shared__ double part[CLIP_THREADS / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s = norm_join<KIND>(s, __shfl_xor(s, o, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < CLIP_THREADS / 64; ++w) s = norm_join<KIND>(s, part[w]);
    return s;
}

template <int KIND, typename T> __device__ double norm_chunk(const T* __restrict__ p, int64_t n) {
    constexpr int V = 16 / sizeof(T);
    const int tid = threadIdx.x;
    double s = 0.0;
    int64_t head = (int64_t)((16 - ((uintptr_t)p & 15)) & 15) / (int64_t)sizeof(T);
    if (head > n) head = n;
    if (tid < head) s = norm_term<KIND>(s, (float)p[tid]);
    p += head; n -= head;
    const int64_t nv = n / V;
    int64_t i = tid;
    for (; i + 3 * CLIP_THREADS < nv; i += 4 * CLIP_THREADS) {
        float x[4][V];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_f32<T, V>(p + (i + u * CLIP_THREADS) * V, x[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) s = norm_term<KIND>(s, x[u][j]);
    }
    for (; i < nv; i += CLIP_THREADS) {
        float x[V];
        load_f32<T, V>(p + i * V, x);
#pragma unroll
        for (int j = 0; j < V; ++j) s = norm_term<KIND>(s, x[j]);
    }
    if (tid < n - nv * V) s = norm_term<KIND>(s, (float)p[nv * V + tid]);
    return s;
}

template <int KIND> __global__ __launch_bounds__(CLIP_THREADS) void norm_kernel(ClipTable t, double* __restrict__ partial) {
    const int i = clip_tensor(t, blockIdx.x);
    const int64_t lo = (int64_t)(blockIdx.x - t.first[i]) * t.chunk;
    const int64_t n = min(t.chunk, t.n[i] - lo);
    const int d = t.types[i] & 15;
    double s;
    if (d == PLNLP_DTYPE_F32) s = norm_chunk<KIND>((const float*)t.src[i] + lo, n);
    else if (d == PLNLP_DTYPE_BF16) s = norm_chunk<KIND>((const __bf16*)t.src[i] + lo, n);
    else s = norm_chunk<KIND>((const _Float16*)t.src[i] + lo, n);
    s = norm_block<KIND>(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// thread 0: the joined partials
template <int KIND> __device__ __forceinline__ double join_partials(const double* __restrict__ partial, int64_t n) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += CLIP_THREADS) s = norm_join<KIND>(s, partial[i]);
    return norm_block<KIND>(s);
}

// partials -> one value, and / or the norm
template <int KIND> __global__ __launch_bounds__(CLIP_THREADS) void norm_finish_kernel(const double* __restrict__ partial, int64_t n,
                                                                                       double* __restrict__ sum, float* __restrict__ norm) {
    const double s = join_partials<KIND>(partial, n);
    if (threadIdx.x) return;
    if (sum) *sum = s;
    if (norm) *norm = (float)(KIND == PLNLP_NORM_L2 ? sqrt(s) : s);
}

template <typename S, typename D> __device__ void clip_chunk(const S* src, D* dst, int64_t n, float c) {
    constexpr int V = 8;
    const int tid = threadIdx.x;
    constexpr int SA = V * sizeof(S) > 16 ? 16 : V * sizeof(S), DA = V * sizeof(D) > 16 ? 16 : V * sizeof(D);
    // elements until both sides are aligned for V-element packs; none within V elements: one at a time throughout
    int64_t head = n;
    for (int h = 0; h < V; ++h)
        if (((uintptr_t)(src + h) % SA) == 0 && ((uintptr_t)(dst + h) % DA) == 0) { head = min((int64_t)h, n); break; }
    for (int64_t i = tid; i < head; i += CLIP_THREADS) dst[i] = (D)((float)src[i] * c);
    src += head; dst += head; n -= head;
    const int64_t nv = n / V;
    int64_t i = tid;
    for (; i + 3 * CLIP_THREADS < nv; i += 4 * CLIP_THREADS) {
        float x[4][V];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_f32<S, V>(src + (i + u * CLIP_THREADS) * V, x[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int j = 0; j < V; ++j) x[u][j] *= c;
            store_f32<D, V>(dst + (i + u * CLIP_THREADS) * V, x[u]);
        }
    }
    for (; i < nv; i += CLIP_THREADS) {
        float x[V];
        load_f32<S, V>(src + i * V, x);
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] *= c;
        store_f32<D, V>(dst + i * V, x);
    }
    if (tid < n - nv * V) dst[nv * V + tid] = (D)((float)src[nv * V + tid] * c);
}

template <typename S> __device__ void clip_chunk_to(const S* src, void* dst, int64_t lo, int type, int64_t n, float c) {
    if (type == PLNLP_DTYPE_F32) clip_chunk(src, (float*)dst + lo, n, c);
    else if (type == PLNLP_DTYPE_BF16) clip_chunk(src, (__bf16*)dst + lo, n, c);
    else clip_chunk(src, (_Float16*)dst + lo, n, c);
}

template <int KIND> __global__ __launch_bounds__(CLIP_THREADS) void clip_kernel(ClipTable t, const double* __restrict__ partial, int64_t n_partial,
                                                                                double max_norm, float* __restrict__ norm_out) {
    __shared__ float coef;
    const double s = join_partials<KIND>(partial, n_partial);
    if (threadIdx.x == 0) {
        const double norm = KIND == PLNLP_NORM_L2 ? sqrt(s) : s;
        if (norm_out && blockIdx.x == 0) *norm_out = (float)norm;
        const double c = max_norm / (norm + 1e-6);
        coef = c > 1.0 ? 1.f : (float)c;          // (a NaN norm stays NaN: the gradients become NaN, as the sums they are)
    }
    __syncthreads();
    const float c = coef;
    const int i = clip_tensor(t, blockIdx.x);
    if (c == 1.f && t.src[i] == t.dst[i]) return;  // in place (the types are equal then) and below the limit: nothing changes
    const int64_t lo = (int64_t)(blockIdx.x - t.first[i]) * t.chunk;
    const int64_t n = min(t.chunk, t.n[i] - lo);
    const int sd = t.types[i] & 15, dd = t.types[i] >> 4;
    if (sd == PLNLP_DTYPE_F32) clip_chunk_to((const float*)t.src[i] + lo, t.dst[i], lo, dd, n, c);
    else if (sd == PLNLP_DTYPE_BF16) clip_chunk_to((const __bf16*)t.src[i] + lo, t.dst[i], lo, dd, n, c);
    else clip_chunk_to((const _Float16*)t.src[i] + lo, t.dst[i], lo, dd, n, c);
}

// elements per workgroup: whole 4096s, about CLIP_BLOCKS workgroups over all tensors
static int64_t clip_chunk_elems(const plnlp_grad_tensor* t, int n_tensors) {
    int64_t total = 0;
    for (int i = 0; i < n_tensors; ++i) total += t[i].n;
    const int64_t c = (total + CLIP_BLOCKS - 1) / CLIP_BLOCKS;
    return (c + CLIP_MIN_CHUNK - 1) / CLIP_MIN_CHUNK * CLIP_MIN_CHUNK;
}

// f(table, workgroups before it) for every launch's worth of non-empty tensors
template <typename F> static void clip_launches(const plnlp_grad_tensor* t, int n_tensors, int64_t chunk, F&& f) {
    ClipTable tab;
    tab.chunk = chunk;
    tab.count = 0;
    int64_t done = 0, blocks = 0;
    for (int i = 0; i < n_tensors; ++i) {
        if (t[i].n == 0) continue;
        const int k = tab.count++;
        tab.src[k] = t[i].src; tab.dst[k] = t[i].dst; tab.n[k] = t[i].n;
        tab.first[k] = (int32_t)blocks;
        tab.types[k] = (uint8_t)(t[i].src_dtype | (t[i].dst_dtype << 4));
        blocks += (t[i].n + chunk - 1) / chunk;
        if (tab.count == CLIP_LAUNCH) { f(tab, done, blocks); done += blocks; blocks = 0; tab.count = 0; }
    }
    if (tab.count) f(tab, done, blocks);
}

static int clip_check(const plnlp_grad_tensor* t, int n_tensors, int kind, bool dst) {
    if (n_tensors < 0 || kind < PLNLP_NORM_L2 || kind > PLNLP_NORM_MAX) return PLNLP_E_SHAPE;
    if (n_tensors && !t) return PLNLP_E_NULL;
    for (int i = 0; i < n_tensors; ++i) {
        if (t[i].n < 0) return PLNLP_E_SHAPE;
        if (!is_dtype(t[i].src_dtype) || (dst && !is_dtype(t[i].dst_dtype))) return PLNLP_E_UNSUPPORTED;
        if (t[i].n && (!t[i].src || (dst && !t[i].dst))) return PLNLP_E_NULL;
        if (t[i].n && ((uintptr_t)t[i].src % dtype_size(t[i].src_dtype) || (dst && (uintptr_t)t[i].dst % dtype_size(t[i].dst_dtype))))
            return PLNLP_E_ALIGN;
        if (dst && t[i].n && t[i].src == t[i].dst && t[i].src_dtype != t[i].dst_dtype) return PLNLP_E_UNSUPPORTED;
    }
    return 0;
}

static int64_t clip_partials(const plnlp_grad_tensor* t, int n_tensors) {
    const int64_t chunk = clip_chunk_elems(t, n_tensors);
    int64_t p = 0;
    for (int i = 0; i < n_tensors; ++i) p += chunk ? (t[i].n + chunk - 1) / chunk : 0;
    return p;
}

template <int KIND> static int clip_run(const plnlp_grad_tensor* t, int n_tensors, bool apply, double max_norm, double* partial,
                                        int64_t n_partial, float* norm, hipStream_t s) {
    const int64_t chunk = clip_chunk_elems(t, n_tensors);
    int rc = 0;
    clip_launches(t, n_tensors, chunk, [&](const ClipTable& tab, int64_t before, int64_t blocks) {
        if (rc) return;
        hipLaunchKernelGGL((norm_kernel<KIND>), dim3((unsigned)blocks), dim3(CLIP_THREADS), 0, s, tab, partial + before);
        rc = launch_status();
    });
    if (rc) return rc;
    const bool finish = !apply || n_partial > CLIP_PARTIALS || n_partial == 0;
    double* total = partial + n_partial;
    if (finish) {
        hipLaunchKernelGGL((norm_finish_kernel<KIND>), dim3(1), dim3(CLIP_THREADS), 0, s, partial, n_partial, total, norm);
        if ((rc = launch_status())) return rc;
    }
    if (!apply) return 0;
    const double* from = finish ? total : partial;
    const int64_t n_from = finish ? 1 : n_partial;
    clip_launches(t, n_tensors, chunk, [&](const ClipTable& tab, int64_t before, int64_t blocks) {
        if (rc) return;
        hipLaunchKernelGGL((clip_kernel<KIND>), dim3((unsigned)blocks), dim3(CLIP_THREADS), 0, s, tab, from, n_from, max_norm,
                           (finish || before) ? nullptr : norm);
        rc = launch_status();
    });
    return rc;
}

static int clip_entry(const plnlp_grad_tensor* t, int n_tensors, int kind, bool apply, double max_norm, double* workspace,
                      int64_t workspace_doubles, float* norm, void* stream) {
    if (int rc = clip_check(t, n_tensors, kind, apply)) return rc;
    if (!workspace || !norm) return PLNLP_E_NULL;
    if ((uintptr_t)workspace % 8 || (uintptr_t)norm % 4) return PLNLP_E_ALIGN;
    if (apply && !(max_norm >= 0.0)) return PLNLP_E_SHAPE;
    const int64_t p = clip_partials(t, n_tensors);
    if (p >= ((int64_t)1 << 31)) return PLNLP_E_SHAPE;
    if (workspace_doubles < p + 1) return PLNLP_E_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    if (kind == PLNLP_NORM_L2) return clip_run<PLNLP_NORM_L2>(t, n_tensors, apply, max_norm, workspace, p, norm, s);
    if (kind == PLNLP_NORM_L1) return clip_run<PLNLP_NORM_L1>(t, n_tensors, apply, max_norm, workspace, p, norm, s);
    return clip_run<PLNLP_NORM_MAX>(t, n_tensors, apply, max_norm, workspace, p, norm, s);
}

}  // namespace plnlp

extern "C" int64_t plnlp_grad_norm_workspace_doubles(const plnlp_grad_tensor* tensors, int n_tensors) {
    if (n_tensors < 0 || (n_tensors && !tensors)) return 0;
    for (int i = 0; i < n_tensors; ++i) if (tensors[i].n < 0) return 0;
    return plnlp::clip_partials(tensors, n_tensors) + 1;
}

extern "C" int plnlp_grad_norm(const plnlp_grad_tensor* tensors, int n_tensors, int norm_kind, double* workspace,
                               int64_t workspace_doubles, float* norm, void* stream) {
    return plnlp::clip_entry(tensors, n_tensors, norm_kind, false, 0.0, workspace, workspace_doubles, norm, stream);
}

extern "C" int plnlp_grad_clip(const plnlp_grad_tensor* tensors, int n_tensors, int norm_kind, double max_norm, double* workspace,
                               int64_t workspace_doubles, float* norm, void* stream) {
    return plnlp::clip_entry(tensors, n_tensors, norm_kind, true, max_norm, workspace, workspace_doubles, norm, stream);
}
