// Rows of a table by id, and the gradient of the table.
//   y[t, :]  = scale * E[id_t, :]                       (a row of zeros where id_t lies outside [0, V))
//   dE[v, :] = scale * sum_{t : id_t = v} dy[t, :]      (every row of dE is written; 0 where no id, or the padding id, is v)
// Both are bound by bytes: the forward reads T ids and the touched rows and writes T rows, the backward reads T rows of dy and
// writes V rows.  Sums are f32, rounded once.
//
// The gradient takes no float atomics (their order would change its bits): the ids are SORTED -- (id, position) pairs, ties in
// the order of the positions -- and every row of dE has ONE owner that finds its run of the sorted list, adds those rows of dy in a
// fixed order and stores the row, so untouched rows need no clearing pass.
//   sort: up to SORT_SMALL ids in one workgroup's LDS (a bitonic network on unique 64-bit words: 1 launch); more in 1 .. 3
//     counting passes of at most 11 bits, each stable (histogram of 4096-id tiles / offsets along the tiles / scatter).
//   sum: a run longer than 2 * SEG (a frequent id) would make its owner's chain the launch's length, so every whole SEG-aligned
//     piece of the sorted list that holds one id is summed beforehand by a workgroup of its own; the owner adds those partials
//     and the two ragged ends.
#include "half.hip.h"

namespace plnlp {

constexpr int LOOKUP_THREADS = 256;
constexpr int SORT_SMALL = 4096;          // ids one workgroup sorts in LDS
constexpr int SORT_TILE = 4096;           // ids per workgroup and counting pass: 256 threads * 16
constexpr int SORT_BITS = 11;             // widest digit: 2048 counters a wave, 4 waves = 32 KiB of LDS
constexpr int SEG = 256;                  // sorted positions per partial sum of a long run

template <typename I> __device__ __forceinline__ int64_t read_id(const I* ids, int64_t i) { return (int64_t)ids[i]; }

// ---- forward ------------------------------------------------------------------------------------------
// TX lanes walk a row in V-element packs, 256 / TX rows at a time, U rows in flight per lane
template <typename T, typename O, typename I, int V, int U>
__global__ __launch_bounds__(LOOKUP_THREADS) void lookup_kernel(const T* __restrict__ table, int64_t ld, int64_t n_rows, int packs, int tx,
                                                                const I* __restrict__ ids, int64_t n_ids, float scale,
                                                                O* __restrict__ out, int64_t ldo) {
    const int ty = LOOKUP_THREADS / tx, x = threadIdx.x & (tx - 1), y = threadIdx.x / tx;
    const int64_t t0 = (int64_t)blockIdx.x * ty * U + y;
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t t = t0 + (int64_t)u * ty;
        row[u] = t < n_ids ? read_id(ids, t) : -1;
    }
    for (int c = x; c < packs; c += tx) {
        float v[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (row[u] >= 0 && row[u] < n_rows) load_f32<T, V>(table + row[u] * ld + (int64_t)c * V, v[u]);
            else
#pragma unroll
                for (int j = 0; j < V; ++j) v[u][j] = 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = t0 + (int64_t)u * ty;
            const bool in = row[u] >= 0 && row[u] < n_rows;
            if (t < n_ids) {
#pragma unroll
                for (int j = 0; j < V; ++j) v[u][j] = in ? v[u][j] * scale : 0.f;
                store_f32<O, V>(out + t * ldo + (int64_t)c * V, v[u]);
            }
        }
    }
}

// ---- sort ---------------------------------------------------------------------------------------------
// the sort key of position i: its id, or n_rows (behind every row) where the id gets no gradient
template <typename I> __device__ __forceinline__ uint32_t sort_key(const I* ids, int64_t i, int64_t n_rows, int64_t padding) {
    const int64_t id = read_id(ids, i);
    return (id < 0 || id >= n_rows || id == padding) ? (uint32_t)n_rows : (uint32_t)id;
}

template <typename I, int N>
__global__ __launch_bounds__(1024) void sort_small_kernel(const I* __restrict__ ids, int n, int64_t n_rows, int64_t padding,
                                                          uint32_t* __restrict__ keys, int32_t* __restrict__ pos) {
    __shared__ uint64_t k[N];
    for (int i = threadIdx.x; i < N; i += 1024)
        k[i] = i < n ? ((uint64_t)sort_key(ids, i, n_rows, padding) << 32) | (uint32_t)i : ~0ull;
    __syncthreads();
    for (int size = 2; size <= N; size <<= 1)
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            for (int i = threadIdx.x; i < N / 2; i += 1024) {
                const int a = 2 * i - (i & (stride - 1)), b = a + stride;
                const uint64_t ka = k[a], kb = k[b];
                if ((ka > kb) == ((a & size) == 0)) { k[a] = kb; k[b] = ka; }
            }
            __syncthreads();
        }
    for (int i = threadIdx.x; i < n; i += 1024) {
        keys[i] = (uint32_t)(k[i] >> 32);
        pos[i] = (int32_t)(uint32_t)k[i];
    }
}

// one counting pass sorts by digit (key >> shift) & (bins - 1); FIRST: the keys come from the ids, the positions are 0 .. n-1
template <typename I, bool FIRST>
__global__ __launch_bounds__(LOOKUP_THREADS) void sort_count_kernel(const I* __restrict__ ids, const uint32_t* __restrict__ keys, int64_t n,
                                                                    int64_t n_rows, int64_t padding, int shift, int bins, int tiles,
                                                                    uint32_t* __restrict__ hist) {
    extern __shared__ uint32_t cnt[];
    for (int d = threadIdx.x; d < bins; d += LOOKUP_THREADS) cnt[d] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * SORT_TILE;
#pragma unroll 4
    for (int u = 0; u < SORT_TILE / LOOKUP_THREADS; ++u) {
        const int64_t i = lo + u * LOOKUP_THREADS + threadIdx.x;
        if (i >= n) break;
        const uint32_t key = FIRST ? sort_key(ids, i, n_rows, padding) : keys[i];
        atomicAdd(&cnt[(key >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += LOOKUP_THREADS) hist[(int64_t)d * tiles + blockIdx.x] = cnt[d];
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {     // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t t = __shfl_up(v, o, 64);
        if ((int)(threadIdx.x & 63) >= o) v += t;
    }
    return v;
}

// exclusive offsets of one digit along the tiles, and the digit's total
__global__ __launch_bounds__(LOOKUP_THREADS) void sort_offsets_kernel(uint32_t* __restrict__ hist, int tiles, uint32_t* __restrict__ total) {
    __shared__ uint32_t part[LOOKUP_THREADS / 64];
    uint32_t* row = hist + (int64_t)blockIdx.x * tiles;
    uint32_t carry = 0;
    for (int lo = 0; lo < tiles; lo += LOOKUP_THREADS) {
        const int i = lo + threadIdx.x;
        const uint32_t v = i < tiles ? row[i] : 0;
        uint32_t s = wave_scan(v);
        if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = s;
        __syncthreads();
        uint32_t before = carry, all = 0;
        for (int w = 0; w < LOOKUP_THREADS / 64; ++w) {
            if (w < (int)(threadIdx.x >> 6)) before += part[w];
            all += part[w];
        }
        if (i < tiles) row[i] = before + s - v;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(LOOKUP_THREADS) void sort_scatter_kernel(const I* __restrict__ ids, const uint32_t* __restrict__ keys,
                                                                      const int32_t* __restrict__ pos, int64_t n, int64_t n_rows,
                                                                      int64_t padding, int shift, int bits, int tiles,
                                                                      const uint32_t* __restrict__ hist, const uint32_t* __restrict__ total,
                                                                      uint32_t* __restrict__ keys_out, int32_t* __restrict__ pos_out) {
    constexpr int WAVES = LOOKUP_THREADS / 64, ROUNDS = SORT_TILE / LOOKUP_THREADS;
    extern __shared__ uint32_t lds[];                  // cnt[WAVES][bins]
    __shared__ uint32_t part[WAVES];
    const int bins = 1 << bits, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int d = threadIdx.x; d < WAVES * bins; d += LOOKUP_THREADS) lds[d] = 0;
    __syncthreads();
    // ranks within the wave's own run of 1024 ids, in order: lanes of the same digit find each other by one ballot a bit
    uint32_t key[ROUNDS], rank[ROUNDS];
    int32_t p[ROUNDS];
    uint32_t* cnt = lds + wave * bins;
    const int64_t lo = (int64_t)blockIdx.x * SORT_TILE + wave * (SORT_TILE / WAVES);
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
        const int64_t i = lo + u * 64 + lane;
        key[u] = 0; p[u] = 0;
        if (i < n) {
            key[u] = FIRST ? sort_key(ids, i, n_rows, padding) : keys[i];
            p[u] = FIRST ? (int32_t)i : pos[i];
        }
    }
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
        const bool in = lo + u * 64 + lane < n;
        const uint32_t d = (key[u] >> shift) & (bins - 1);
        uint64_t same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const uint64_t m = __ballot((d >> b) & 1);
            same &= ((d >> b) & 1) ? m : ~m;
        }
        rank[u] = 0;
        if (in) {
            const int leader = __ffsll((unsigned long long)same) - 1;
            uint32_t before = 0;
            if (lane == leader) before = atomicAdd(&cnt[d], (uint32_t)__popcll(same));
            rank[u] = __shfl(before, leader, 64) + (uint32_t)__popcll(same & ((1ull << lane) - 1));
        }
    }
    __syncthreads();
    // digit starts: the totals' exclusive scan + the tile's offset + the earlier waves' counts
    uint32_t carry = 0;
    for (int b0 = 0; b0 < bins; b0 += LOOKUP_THREADS) {
        const int d = b0 + threadIdx.x;
        const uint32_t v = d < bins ? total[d] : 0;
        const uint32_t s = wave_scan(v);
        if (lane == 63) part[wave] = s;
        __syncthreads();
        uint32_t before = carry;
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) before += part[w];
            carry += part[w];
        }
        if (d < bins) {
            uint32_t start = before + s - v + hist[(int64_t)d * tiles + blockIdx.x];
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t c = lds[w * bins + d];
                lds[w * bins + d] = start;
                start += c;
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
        if (lo + u * 64 + lane >= n) continue;
        const uint32_t at = cnt[(key[u] >> shift) & (bins - 1)] + rank[u];
        keys_out[at] = key[u];
        pos_out[at] = p[u];
    }
}

// ---- gradient -----------------------------------------------------------------------------------------
// s[j] += rows pos[b .. e) step `step` of gy, columns of this lane's pack; four rows in flight
template <typename G, int V>
__device__ __forceinline__ void add_rows(const G* __restrict__ gy, int64_t ldg, int64_t col, const int32_t* __restrict__ pos, int64_t b,
                                         int64_t e, int64_t step, float (&s)[V]) {
    int64_t i = b;
    for (; i + 3 * step < e; i += 4 * step) {
        float x[4][V];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_f32<G, V>(gy + (int64_t)pos[i + u * step] * ldg + col, x[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] += x[u][j];
    }
    for (; i < e; i += step) {
        float x[V];
        load_f32<G, V>(gy + (int64_t)pos[i] * ldg + col, x);
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] += x[j];
    }
}

// joins the 256 / tx groups' sums in group order; group 0 holds the result
template <int V> __device__ __forceinline__ void join_groups(float (&s)[V], float* lds, int tx) {
    const int x = threadIdx.x & (tx - 1), y = threadIdx.x / tx, ty = LOOKUP_THREADS / tx;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) lds[(y * V + j) * tx + x] = s[j];
    __syncthreads();
    if (y == 0)
        for (int g = 1; g < ty; ++g)
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] += lds[(g * V + j) * tx + x];
}

// piece i of the sorted list, [i * SEG, (i + 1) * SEG), where it holds one id: partial[i, :] = its rows of gy, added
template <typename G, int V>
__global__ __launch_bounds__(LOOKUP_THREADS) void grad_pieces_kernel(const G* __restrict__ gy, int64_t ldg, const uint32_t* __restrict__ keys,
                                                                     const int32_t* __restrict__ pos, int64_t n_rows, int packs, int tx,
                                                                     float* __restrict__ partial) {
    __shared__ float lds[LOOKUP_THREADS * V];
    const int64_t b = (int64_t)blockIdx.x * SEG;
    const uint32_t key = keys[b];
    if (key != keys[b + SEG - 1] || key >= (uint32_t)n_rows) return;
    const int x = threadIdx.x & (tx - 1), y = threadIdx.x / tx, ty = LOOKUP_THREADS / tx;
    for (int c0 = 0; c0 < packs; c0 += tx) {
        const int c = c0 + x;
        float s[V] = {};
        if (c < packs) add_rows<G, V>(gy, ldg, (int64_t)c * V, pos, b + y, b + SEG, ty, s);
        join_groups<V>(s, lds, tx);
        if (y == 0 && c < packs) {
            float* o = partial + (int64_t)blockIdx.x * packs * V + (int64_t)c * V;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = s[j];
        }
    }
}

constexpr int GRAD_ROWS = 64;             // rows of dE per workgroup
constexpr int GRAD_POS = 1024;            // positions of those rows kept in LDS

template <typename G, typename E, int V>
__global__ __launch_bounds__(LOOKUP_THREADS) void grad_rows_kernel(const G* __restrict__ gy, int64_t ldg, const uint32_t* __restrict__ keys,
                                                                   const int32_t* __restrict__ pos, int64_t n, int64_t n_rows, int packs,
                                                                   int tx, const float* __restrict__ partial, float scale,
                                                                   E* __restrict__ grad, int64_t lde) {
    __shared__ int64_t beg[GRAD_ROWS + 1];
    __shared__ int32_t near_pos[GRAD_POS];
    __shared__ float lds[LOOKUP_THREADS * V];
    const int64_t row0 = (int64_t)blockIdx.x * GRAD_ROWS;
    if (threadIdx.x <= GRAD_ROWS) {                   // first sorted position whose id is >= row0 + thread
        const int64_t want = min(row0 + (int64_t)threadIdx.x, n_rows);
        int64_t lo = 0, hi = n;
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if ((int64_t)keys[mid] < want) lo = mid + 1; else hi = mid;
        }
        beg[threadIdx.x] = lo;
    }
    __syncthreads();
    const int64_t p0 = beg[0], held = min(beg[GRAD_ROWS] - p0, (int64_t)GRAD_POS);
    for (int i = threadIdx.x; i < held; i += LOOKUP_THREADS) near_pos[i] = pos[p0 + i];
    __syncthreads();
    const int x = threadIdx.x & (tx - 1), y = threadIdx.x / tx, ty = LOOKUP_THREADS / tx;
    const int rows = (int)min((int64_t)GRAD_ROWS, n_rows - row0);
    for (int r = y; r < rows; r += ty) {              // short runs: a group a row
        const int64_t b = beg[r], e = beg[r + 1];
        if (e - b > 2 * SEG) continue;
        for (int c = x; c < packs; c += tx) {
            float s[V] = {};
            if (e - p0 <= GRAD_POS) add_rows<G, V>(gy, ldg, (int64_t)c * V, near_pos, b - p0, e - p0, 1, s);
            else add_rows<G, V>(gy, ldg, (int64_t)c * V, pos, b, e, 1, s);
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] *= scale;
            store_f32<E, V>(grad + (row0 + r) * lde + (int64_t)c * V, s);
        }
    }
    for (int r = 0; r < rows; ++r) {                  // long runs: the workgroup a row
        const int64_t b = beg[r], e = beg[r + 1];
        if (e - b <= 2 * SEG) continue;
        const int64_t i0 = (b + SEG - 1) / SEG, i1 = e / SEG;       // whole pieces [i0, i1)
        for (int c0 = 0; c0 < packs; c0 += tx) {
            const int c = c0 + x;
            float s[V] = {};
            if (c < packs) {
                add_rows<G, V>(gy, ldg, (int64_t)c * V, pos, b + y, i0 * SEG, ty, s);
                for (int64_t i = i0 + y; i < i1; i += ty) {
                    const float* q = partial + i * packs * V + (int64_t)c * V;
#pragma unroll
                    for (int j = 0; j < V; ++j) s[j] += q[j];
                }
                add_rows<G, V>(gy, ldg, (int64_t)c * V, pos, i1 * SEG + y, e, ty, s);
            }
            join_groups<V>(s, lds, tx);
            if (y == 0 && c < packs) {
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] *= scale;
                store_f32<E, V>(grad + (row0 + r) * lde + (int64_t)c * V, s);
            }
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------
// widest pack both sides allow: V divides the width and both row strides, and V elements are aligned (to 16 bytes at most)
static bool pack_fits(int v, const void* p, int64_t ld, int size) {
    const int bytes = v * size > 16 ? 16 : v * size;
    return (uintptr_t)p % bytes == 0 && (ld * size) % bytes == 0;
}
static int pick_pack(int64_t width, const void* a, int64_t lda, int sa, const void* b, int64_t ldb, int sb) {
    for (int v = 8; v > 1; v >>= 1)
        if (width % v == 0 && pack_fits(v, a, lda, sa) && pack_fits(v, b, ldb, sb)) return v;
    return 1;
}
static int lanes_for(int64_t packs, int most) {
    int t = 1;
    while (t < most && t < packs) t <<= 1;
    return t;
}
template <typename F> static int with_pack(int v, F&& f) {
    if (v == 8) return f(std::integral_constant<int, 8>{});
    if (v == 4) return f(std::integral_constant<int, 4>{});
    if (v == 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}
template <typename F> static int with_id(int bytes, F&& f) { return bytes == 8 ? f(int64_t{}) : f(int32_t{}); }

constexpr int64_t LOOKUP_MAX = ((int64_t)1 << 31) - 2;

static int lookup_check(int64_t n_rows, int64_t width, int id_bytes, int64_t n_ids, int d0, int d1) {
    if (n_rows < 0 || width < 0 || n_ids < 0 || n_rows > LOOKUP_MAX || n_ids > LOOKUP_MAX || width > ((int64_t)1 << 30)) return PLNLP_E_SHAPE;
    if ((id_bytes != 4 && id_bytes != 8) || !is_dtype(d0) || !is_dtype(d1)) return PLNLP_E_UNSUPPORTED;
    return 0;
}

struct GradWorkspace { int64_t keys[2], pos[2], hist, total, partial, bytes; };
static GradWorkspace grad_workspace(int64_t n, int64_t width) {
    GradWorkspace w{};
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t a = at; at += (bytes + 255) / 256 * 256; return a; };
    const bool small = n <= SORT_SMALL;
    for (int i = 0; i < (small ? 1 : 2); ++i) { w.keys[i] = take(4 * n); w.pos[i] = take(4 * n); }
    const int64_t tiles = (n + SORT_TILE - 1) / SORT_TILE;
    w.hist = take(small ? 0 : 4 * tiles << SORT_BITS);
    w.total = take(small ? 0 : 4 << SORT_BITS);
    w.partial = take(n / SEG * width * 4);
    w.bytes = at;
    return w;
}

}  // namespace plnlp

extern "C" int plnlp_embedding_lookup(const void* table, int64_t ld, int table_dtype, int64_t n_rows, int64_t width, const void* ids,
                                      int id_bytes, int64_t n_ids, float scale, void* out, int64_t ldo, int out_dtype, void* stream) {
    using namespace plnlp;
    if (int rc = lookup_check(n_rows, width, id_bytes, n_ids, table_dtype, out_dtype)) return rc;
    if (n_ids == 0 || width == 0) return 0;
    if ((!table && n_rows) || !ids || !out) return PLNLP_E_NULL;
    if (ld < width || ldo < width) return PLNLP_E_SHAPE;
    if ((uintptr_t)table % dtype_size(table_dtype) || (uintptr_t)out % dtype_size(out_dtype) || (uintptr_t)ids % id_bytes) return PLNLP_E_ALIGN;
    const int v = pick_pack(width, table, ld, dtype_size(table_dtype), out, ldo, dtype_size(out_dtype));
    const int64_t packs = width / v;
    const int tx = lanes_for(packs, LOOKUP_THREADS), ty = LOOKUP_THREADS / tx;
    const bool four = n_ids >= (int64_t)4 * ty * 1024;       // enough rows to fill the chip with four per lane in flight
    const int64_t blocks = (n_ids + ty * (four ? 4 : 1) - 1) / (ty * (four ? 4 : 1));
    return with_dtype(table_dtype, [&](auto tt) { return with_dtype(out_dtype, [&](auto ot) { return with_id(id_bytes, [&](auto it) {
        return with_pack(v, [&](auto vc) {
            using T = decltype(tt); using O = decltype(ot); using I = decltype(it);
            constexpr int V = decltype(vc)::value;
            auto run = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(LOOKUP_THREADS), 0, (hipStream_t)stream, (const T*)table, ld, n_rows,
                                   (int)packs, tx, (const I*)ids, n_ids, scale, (O*)out, ldo);
                return launch_status();
            };
            return four ? run(lookup_kernel<T, O, I, V, 4>) : run(lookup_kernel<T, O, I, V, 1>);
        }); }); }); });
}

extern "C" int64_t plnlp_embedding_grad_workspace_bytes(int64_t n_ids, int64_t width) {
    return (n_ids <= 0 || width < 0 || n_ids > plnlp::LOOKUP_MAX) ? 0 : plnlp::grad_workspace(n_ids, width).bytes;
}

extern "C" int plnlp_embedding_grad(const void* gy, int64_t ldg, int gy_dtype, const void* ids, int id_bytes, int64_t n_ids,
                                    int64_t padding_id, float scale, void* grad, int64_t lde, int grad_dtype, int64_t n_rows,
                                    int64_t width, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace plnlp;
    if (int rc = lookup_check(n_rows, width, id_bytes, n_ids, gy_dtype, grad_dtype)) return rc;
    if (n_rows == 0 || width == 0) return 0;
    if (!grad || (n_ids && (!gy || !ids))) return PLNLP_E_NULL;
    if (lde < width || (n_ids && ldg < width)) return PLNLP_E_SHAPE;
    if ((uintptr_t)gy % dtype_size(gy_dtype) || (uintptr_t)grad % dtype_size(grad_dtype) || (n_ids && (uintptr_t)ids % id_bytes)) return PLNLP_E_ALIGN;
    const GradWorkspace w = grad_workspace(n_ids, width);
    if (n_ids && (!workspace || workspace_bytes < w.bytes)) return PLNLP_E_WORKSPACE;
    if ((uintptr_t)workspace % 16) return PLNLP_E_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    uint32_t* keys[2] = {(uint32_t*)(ws + w.keys[0]), (uint32_t*)(ws + w.keys[1])};
    int32_t* pos[2] = {(int32_t*)(ws + w.pos[0]), (int32_t*)(ws + w.pos[1])};
    float* partial = (float*)(ws + w.partial);
    int cur = 0, rc = 0;
    if (n_ids && n_ids <= SORT_SMALL) {
        rc = with_id(id_bytes, [&](auto it) {
            using I = decltype(it);
            auto run = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(1), dim3(1024), 0, s, (const I*)ids, (int)n_ids, n_rows, padding_id, keys[0], pos[0]);
                return launch_status();
            };
            return n_ids <= 256 ? run(sort_small_kernel<I, 256>) : n_ids <= 1024 ? run(sort_small_kernel<I, 1024>) : run(sort_small_kernel<I, SORT_SMALL>);
        });
    } else if (n_ids) {
        int bits = 1;
        while (((int64_t)1 << bits) <= n_rows) ++bits;               // keys are 0 .. n_rows
        const int passes = (bits + SORT_BITS - 1) / SORT_BITS, digit = (bits + passes - 1) / passes;
        const int tiles = (int)((n_ids + SORT_TILE - 1) / SORT_TILE), bins = 1 << digit;
        uint32_t* hist = (uint32_t*)(ws + w.hist);
        uint32_t* total = (uint32_t*)(ws + w.total);
        for (int p = 0; p < passes && !rc; ++p) {
            const int shift = p * digit;
            rc = with_id(id_bytes, [&](auto it) {
                using I = decltype(it);
                auto pass = [&](auto first) {
                    constexpr bool F = decltype(first)::value;
                    hipLaunchKernelGGL((sort_count_kernel<I, F>), dim3(tiles), dim3(LOOKUP_THREADS), 4 * bins, s, (const I*)ids, keys[cur],
                                       n_ids, n_rows, padding_id, shift, bins, tiles, hist);
                    hipLaunchKernelGGL(sort_offsets_kernel, dim3(bins), dim3(LOOKUP_THREADS), 0, s, hist, tiles, total);
                    hipLaunchKernelGGL((sort_scatter_kernel<I, F>), dim3(tiles), dim3(LOOKUP_THREADS), 4 * bins * (LOOKUP_THREADS / 64), s,
                                       (const I*)ids, keys[cur], pos[cur], n_ids, n_rows, padding_id, shift, digit, tiles, hist, total,
                                       keys[cur ^ 1], pos[cur ^ 1]);
                    return launch_status();
                };
                return p == 0 ? pass(std::true_type{}) : pass(std::false_type{});
            });
            cur ^= 1;
        }
    }
    if (rc) return rc;
    const int gs = dtype_size(gy_dtype), es = dtype_size(grad_dtype);
    const int v = n_ids ? pick_pack(width, gy, ldg, gs, grad, lde, es) : pick_pack(width, grad, lde, es, grad, lde, es);
    const int64_t packs = width / v;
    const int tx = lanes_for(packs, 64);
    return with_dtype(gy_dtype, [&](auto gt) { return with_dtype(grad_dtype, [&](auto et) { return with_pack(v, [&](auto vc) {
        using G = decltype(gt); using E = decltype(et);
        constexpr int V = decltype(vc)::value;
        if (n_ids > 2 * SEG) {
            hipLaunchKernelGGL((grad_pieces_kernel<G, V>), dim3((unsigned)(n_ids / SEG)), dim3(LOOKUP_THREADS), 0, s, (const G*)gy, ldg,
                               keys[cur], pos[cur], n_rows, (int)packs, tx, partial);
            if (int e = launch_status()) return e;
        }
        hipLaunchKernelGGL((grad_rows_kernel<G, E, V>), dim3((unsigned)((n_rows + GRAD_ROWS - 1) / GRAD_ROWS)), dim3(LOOKUP_THREADS), 0, s,
                           (const G*)gy, ldg, keys[cur], pos[cur], n_ids, n_rows, (int)packs, tx, partial, scale, (E*)grad, lde);
        return launch_status();
    }); }); });
}
