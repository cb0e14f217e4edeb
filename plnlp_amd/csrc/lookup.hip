// Rows of a table by id, and the gradient of the table.
//   y[t, :]  = scale * E[id_t, :]                       (a row of zeros where id_t lies outside [0, V))
//   dE[v, :] = scale * sum_{t : id_t = v} dy[t, :]      (every row of dE is written; 0 where no id, or the padding id, is v)
// Both are bound by bytes: the forward reads T ids and the touched rows and writes T rows, the backward reads T rows of dy and
// writes V rows.  Sums are f32, rounded once.
//
// The gradient takes no float atomics (their order would change its bits): the ids are SORTED -- (id, position) pairs, ties in
// the order of the positions -- and the sorted list is cut into ranges of equal length, whatever the ids are.
//   sort: up to SORT_SMALL ids in one launch, each placed by counting the pairs before it (sort_small_kernel); more in 1 .. 3
//     counting passes of at most 11 bits, each stable (histogram of the tiles / offsets along the tiles / scatter).  262 144 ids of
//     a table of 235 868 rows, two passes: 34 us, six launches of 4 .. 9 us that wait for memory more than they move.
//   runs: a group of lanes walks one range with eight rows of dy in flight, adds the rows of a run of equal ids and stores the row
//     of dE when the run ends.  A run that crosses the ends of its range leaves an f32 partial there instead; the range in which
//     it begins adds those up in order (grad_joins_kernel).  So a frequent id costs what its rows cost, spread over the chip.
//     Further workgroups of the same launch look up which rows of dE have no id and clear them: every row is written once.
#include "half.hip.h"

namespace plnlp {

constexpr int LOOKUP_THREADS = 256;
constexpr int SORT_SMALL = 8192;          // ids that are placed by counting, in one launch
constexpr int OFFSET_DIGITS = 32;         // digits a workgroup of sort_offsets_kernel
constexpr int SORT_BITS = 11;             // widest digit: 2048 counters a wave, 4 waves = 32 KiB of LDS

template <typename I> __device__ __forceinline__ int64_t read_id(const I* ids, int64_t i) { return (int64_t)ids[i]; }

// ---- forward ------------------------------------------------------------------------------------------
// TX lanes walk a row in V-element packs, 256 / TX rows at a time, U rows in flight per lane (four: eight were 10 % slower).
// STREAM: the result is written past the caches (524 288 rows of 2 KiB: 310 -> 279 us, and the table stays where it is read from)
template <typename T, typename O, typename I, int V, int U, bool STREAM>
__global__ __launch_bounds__(LOOKUP_THREADS) void lookup_kernel(const T* __restrict__ table, int64_t ld, int64_t n_rows, int packs, int tx,
                                                                const I* __restrict__ ids, int64_t n_ids, float scale,
                                                                O* __restrict__ out, int64_t ldo) {
    const int ty = LOOKUP_THREADS / tx, x = threadIdx.x & (tx - 1), y = threadIdx.x / tx;
    const int64_t t0 = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ty * U + y;      // (past the last rows nothing is read or written)
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
                if (STREAM) stream_f32<O, V>(out + t * ldo + (int64_t)c * V, v[u]);
                else store_f32<O, V>(out + t * ldo + (int64_t)c * V, v[u]);
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

// The sort's launches wait for memory more than they move: further workgroups of them clear dE meanwhile (clear_first).  Bytes; a piece is
// a row, or 8 KiB where the rows lie side by side.
constexpr int CLEAR_PIECE = 8192;
struct Clear {
    char* at;
    int64_t ld, width, total;          // of the pieces; the last one ends at `total`
    int64_t pieces;
    int unit, tx;                      // bytes a store, lanes a piece
    int first, launch, launches;       // this launch's workgroups of the sort; its share of the pieces
};
__device__ void clear_share(const Clear& c) {
    const int x = threadIdx.x & (c.tx - 1), y = threadIdx.x / c.tx, ty = blockDim.x / c.tx;
    const int64_t per = (c.pieces + c.launches - 1) / c.launches, lo = per * c.launch, hi = min(lo + per, c.pieces);
    for (int64_t p = lo + (int64_t)(blockIdx.x - c.first) * ty + y; p < hi; p += (int64_t)(gridDim.x - c.first) * ty) {
        char* row = c.at + p * c.ld;
        const int64_t n = min(c.width, c.total - p * c.ld);
        for (int64_t b = (int64_t)x * c.unit; b < n; b += (int64_t)c.tx * c.unit) {
            if (b + c.unit > n)                                        // (elements are two bytes at least)
                for (int64_t e = b; e < n; e += 2) *reinterpret_cast<uint16_t*>(row + e) = 0;
            else if (c.unit == 16) *reinterpret_cast<u32x4*>(row + b) = u32x4{0, 0, 0, 0};
            else if (c.unit == 8) *reinterpret_cast<uint64_t*>(row + b) = 0;
            else if (c.unit == 4) *reinterpret_cast<uint32_t*>(row + b) = 0;
            else *reinterpret_cast<uint16_t*>(row + b) = 0;
        }
    }
}

// Up to SORT_SMALL ids: an id's place is the number of pairs that come before its own, counted.  A workgroup places 64 ids, one a lane;
// its 16 waves share the keys, read from LDS by all lanes at once: before the ids' own positions equal keys count, behind them not.
template <typename I>
__global__ __launch_bounds__(1024) void sort_small_kernel(const I* __restrict__ ids, int n, int64_t n_rows, int64_t padding,
                                                          uint2* __restrict__ sorted, Clear clear) {
    if ((int)blockIdx.x >= clear.first) { clear_share(clear); return; }
    __shared__ u32x4 keys[SORT_SMALL / 4];
    __shared__ uint32_t part[16][64];
    const uint32_t* k = reinterpret_cast<const uint32_t*>(keys);
    const int quads = (n + 3) / 4;
    for (int i = threadIdx.x; i < quads * 4; i += 1024)
        reinterpret_cast<uint32_t*>(keys)[i] = i < n ? sort_key(ids, i, n_rows, padding) : ~0u;
    __syncthreads();
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i0 = blockIdx.x * 64, i = i0 + lane;
    const uint32_t key = i < n ? k[i] : 0;
    const int per = (quads + 15) / 16, hi = min((wave + 1) * per, quads), own = min(i0 / 4, hi), behind = min(i0 / 4 + 16, hi);
    uint32_t before = 0;
    int q = wave * per;
#pragma unroll 4
    for (; q < own; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) before += keys[q][j] <= key;
    for (; q < behind; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) before += keys[q][j] < key + (4 * q + j < i);
#pragma unroll 4
    for (; q < hi; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) before += keys[q][j] < key;
    part[wave][lane] = before;
    __syncthreads();
    if (wave || i >= n) return;
    for (int w = 1; w < 16; ++w) before += part[w][lane];
    sorted[before] = make_uint2(key, (uint32_t)i);
}

// One counting pass sorts by the digit (key >> shift) & (bins - 1).  A tile is 256 * ROUNDS ids; hist[tile][digit].
// FIRST: the keys come from the ids, the positions are 0 .. n-1.
template <typename I, bool FIRST, int ROUNDS>
__global__ __launch_bounds__(LOOKUP_THREADS) void sort_count_kernel(const I* __restrict__ ids, const uint2* __restrict__ in, int64_t n,
                                                                    int64_t n_rows, int64_t padding, int shift, int bins,
                                                                    uint32_t* __restrict__ hist, Clear clear) {
    if ((int)blockIdx.x >= clear.first) { clear_share(clear); return; }
    extern __shared__ uint32_t cnt[];
    const int64_t lo = (int64_t)blockIdx.x * ROUNDS * LOOKUP_THREADS + threadIdx.x;
    uint32_t key[ROUNDS];
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
        const int64_t i = lo + u * LOOKUP_THREADS;
        key[u] = i >= n ? 0 : FIRST ? sort_key(ids, i, n_rows, padding) : in[i].x;
    }
    for (int d = threadIdx.x; d < bins; d += LOOKUP_THREADS) cnt[d] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u)
        if (lo + u * LOOKUP_THREADS < n) atomicAdd(&cnt[(key[u] >> shift) & (bins - 1)], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += LOOKUP_THREADS) hist[(int64_t)blockIdx.x * bins + d] = cnt[d];
}

// counts -> exclusive offsets along the tiles, and the digits' totals: 32 digits a workgroup, 32 groups of its threads share the tiles
// (16 groups of 64: 1 000 000 ids of 200-byte rows 204 us instead of 197; 64 of 16: no faster, and 3 us lost on few tiles)
__global__ __launch_bounds__(1024) void sort_offsets_kernel(uint32_t* __restrict__ hist, int tiles, int bins, uint32_t* __restrict__ total,
                                                            Clear clear) {
    if ((int)blockIdx.x >= clear.first) { clear_share(clear); return; }
    constexpr int GROUPS = 1024 / OFFSET_DIGITS;
    __shared__ uint32_t part[GROUPS][OFFSET_DIGITS];
    const int group = threadIdx.x / OFFSET_DIGITS, x = threadIdx.x % OFFSET_DIGITS, d = blockIdx.x * OFFSET_DIGITS + x;
    const int per = (tiles + GROUPS - 1) / GROUPS, lo = min(group * per, tiles), hi = min(lo + per, tiles);
    const bool in = d < bins;
    uint32_t s = 0;
#pragma unroll 8
    for (int t = lo; t < hi; ++t) s += in ? hist[(int64_t)t * bins + d] : 0;
    part[group][x] = s;
    __syncthreads();
    uint32_t run = 0;
#pragma unroll 8
    for (int w = 0; w < GROUPS; ++w) run += w < group ? part[w][x] : 0;
    if (!in) return;
    if (group == GROUPS - 1) total[d] = run + s;
#pragma unroll 8
    for (int t = lo; t < hi; ++t) {
        const uint32_t c = hist[(int64_t)t * bins + d];
        hist[(int64_t)t * bins + d] = run;
        run += c;
    }
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {     // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t t = __shfl_up(v, o, 64);
        if ((int)(threadIdx.x & 63) >= o) v += t;
    }
    return v;
}

template <typename I, bool FIRST, int ROUNDS>
__global__ __launch_bounds__(LOOKUP_THREADS) void sort_scatter_kernel(const I* __restrict__ ids, const uint2* __restrict__ in, int64_t n,
                                                                      int64_t n_rows, int64_t padding, int shift, int bits,
                                                                      const uint32_t* __restrict__ hist, const uint32_t* __restrict__ total,
                                                                      uint2* __restrict__ out, Clear clear) {
    if ((int)blockIdx.x >= clear.first) { clear_share(clear); return; }
    constexpr int WAVES = LOOKUP_THREADS / 64;
    extern __shared__ uint32_t lds[];                  // cnt[WAVES][bins]
    __shared__ uint32_t part[WAVES];
    const int bins = 1 << bits, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // ranks within the wave's own run of 64 * ROUNDS ids, in order: lanes of the same digit find each other by one ballot a bit
    uint2 pair[ROUNDS];
    uint32_t rank[ROUNDS];
    uint32_t* cnt = lds + wave * bins;
    const int64_t lo = ((int64_t)blockIdx.x * WAVES + wave) * 64 * ROUNDS + lane;
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
        const int64_t i = lo + u * 64;
        pair[u] = i >= n ? make_uint2(0, 0) : FIRST ? make_uint2(sort_key(ids, i, n_rows, padding), (uint32_t)i) : in[i];
    }
    // (the digits' totals and offsets are asked for before the ranking: one wait instead of one per 256 digits: 10.3 -> 8.6 us)
    constexpr int MOST = (1 << SORT_BITS) / LOOKUP_THREADS;
    uint32_t sum[MOST], off[MOST];
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        const int d = i * LOOKUP_THREADS + threadIdx.x;
        sum[i] = d < bins ? total[d] : 0;
        off[i] = d < bins ? hist[(int64_t)blockIdx.x * bins + d] : 0;
    }
    for (int d = threadIdx.x; d < WAVES * bins; d += LOOKUP_THREADS) lds[d] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
        const bool real = lo + u * 64 < n;
        const uint32_t d = (pair[u].x >> shift) & (bins - 1);
        uint64_t same = __ballot(real);
        for (int b = 0; b < bits; ++b) {
            const uint64_t m = __ballot((d >> b) & 1);
            same &= ((d >> b) & 1) ? m : ~m;
        }
        rank[u] = 0;
        if (real) {
            const int leader = __ffsll((unsigned long long)same) - 1;
            uint32_t before = 0;
            if (lane == leader) before = atomicAdd(&cnt[d], (uint32_t)__popcll(same));
            rank[u] = __shfl(before, leader, 64) + (uint32_t)__popcll(same & ((1ull << lane) - 1));
        }
    }
    __syncthreads();
    // digit starts: the totals' exclusive scan + the tile's offset + the earlier waves' counts
    uint32_t carry = 0;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        if (i * LOOKUP_THREADS >= bins) break;
        const int d = i * LOOKUP_THREADS + threadIdx.x;
        const uint32_t v = sum[i], s = wave_scan(v);
        if (lane == 63) part[wave] = s;
        __syncthreads();
        uint32_t before = carry;
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) before += part[w];
            carry += part[w];
        }
        if (d < bins) {
            uint32_t start = before + s - v + off[i];
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
        if (lo + u * 64 >= n) continue;
        out[cnt[(pair[u].x >> shift) & (bins - 1)] + rank[u]] = pair[u];
    }
}

// ---- gradient -----------------------------------------------------------------------------------------
constexpr int CLEAR_ROWS = LOOKUP_THREADS;      // rows of dE a clearing workgroup looks up, one a thread

// the first sorted position in [lo, hi) whose key is >= want, hi if there is none
__device__ __forceinline__ int64_t lower_bound(const uint2* __restrict__ sorted, int64_t lo, int64_t hi, uint32_t want) {
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (sorted[mid].x < want) lo = mid + 1; else hi = mid;
    }
    return lo;
}

template <typename G, typename E, int V> struct GradArgs {
    const G* gy; int64_t ldg;
    const uint2* sorted;              // (key, position), by key and then by position
    int64_t n, n_rows;
    int packs, tx, slabs;             // a row is `packs` packs of V; a group of tx lanes takes one slab of tx packs
    int range;                        // sorted positions per group
    int64_t n_ranges, run_blocks;     // workgroups before run_blocks walk ranges, the others clear rows
    float* head; float* tail;         // [n_ranges, packs * V]: sums of the runs that enter / leave a range
    float scale;
    E* grad; int64_t lde;
};

template <typename G, typename E, int V> __global__ __launch_bounds__(LOOKUP_THREADS) void grad_runs_kernel(GradArgs<G, E, V> a) {
    const int x = threadIdx.x & (a.tx - 1), y = threadIdx.x / a.tx, ty = LOOKUP_THREADS / a.tx;
    if (blockIdx.x >= a.run_blocks) {
        __shared__ uint8_t none[CLEAR_ROWS];
        const int64_t row0 = ((int64_t)blockIdx.x - a.run_blocks) * CLEAR_ROWS, row = row0 + threadIdx.x;
        bool empty = row < a.n_rows;
        if (empty && a.n > 0) {
            const int64_t at = lower_bound(a.sorted, 0, a.n, (uint32_t)row);
            empty = at == a.n || a.sorted[at].x != (uint32_t)row;
        }
        none[threadIdx.x] = empty;
        __syncthreads();
        const float zero[V] = {};
        for (int r = y; r < CLEAR_ROWS; r += ty)
            if (none[r])
                for (int c = x; c < a.packs; c += a.tx) store_f32<E, V>(a.grad + (row0 + r) * a.lde + (int64_t)c * V, zero);
        return;
    }
    const int64_t unit = (int64_t)blockIdx.x * ty + y, range = unit / a.slabs;
    const int c = (int)(unit % a.slabs) * a.tx + x;
    if (range >= a.n_ranges || c >= a.packs) return;
    const int64_t b = range * a.range, e = min(b + a.range, a.n), col = (int64_t)c * V;
    const uint32_t end = (uint32_t)a.n_rows;
    uint32_t cur = a.sorted[b].x;
    bool entered = b > 0 && a.sorted[b - 1].x == cur;          // the current run began in an earlier range
    float s[V] = {};
    auto put = [&](bool leaves) {
        if (cur >= end) return;
        if (entered || leaves) {
            float* o = (entered ? a.head : a.tail) + range * a.packs * V + col;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = s[j];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] *= a.scale;
            store_f32<E, V>(a.grad + (int64_t)cur * a.lde + col, s);
        }
    };
    constexpr int U = 8;
    uint2 next[U];
    auto ask = [&](int64_t i) {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = a.sorted[min(i + u, e - 1)];
    };
    ask(b);
    for (int64_t i = b; i < e; i += U) {
        if (next[0].x >= end) { if (cur < end) put(false); cur = end; break; }      // only ids without a gradient follow
        Pack<G, V> row[U];
        uint32_t key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            key[u] = next[u].x;
            row[u] = stream_pack<G, V>(a.gy + (int64_t)next[u].y * a.ldg + col);      // (524 288 rows of 2 KiB: 242 -> 225 us)
        }
        if (i + U < e) ask(i + U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= e) break;
            if (key[u] != cur) {
                put(false);
                cur = key[u];
                entered = false;
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] += (float)row[u].v[j];
        }
    }
    put(e < a.n && a.sorted[e].x == cur);
}

// the range in which a run begins that leaves it: its tail + the heads of the ranges the run enters, in order of the groups of lanes
// that share them
template <typename G, typename E, int V> __global__ __launch_bounds__(LOOKUP_THREADS) void grad_joins_kernel(GradArgs<G, E, V> a) {
    __shared__ float lds[LOOKUP_THREADS * V];
    const int64_t range = blockIdx.x, b = range * a.range, e = b + a.range;      // (not the last range: e < n)
    const uint32_t key = a.sorted[e - 1].x;
    if (key >= (uint32_t)a.n_rows || a.sorted[e].x != key || (b > 0 && a.sorted[b - 1].x == key)) return;
    // the range the run ends in: mostly the next one
    const int64_t next_end = min(e + a.range, a.n);
    const int64_t last = (next_end == a.n || a.sorted[next_end].x != key) ? range + 1
                                                                           : (lower_bound(a.sorted, next_end, a.n, key + 1) - 1) / a.range;
    const int x = threadIdx.x & (a.tx - 1), y = threadIdx.x / a.tx, ty = LOOKUP_THREADS / a.tx;
    const int c = blockIdx.y * a.tx + x;
    const int64_t width = (int64_t)a.packs * V, col = (int64_t)c * V;
    float s[V] = {};
    if (c < a.packs) {
        if (y == 0)
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = a.tail[range * width + col + j];
        int64_t i = range + 1 + y;
        for (; i + 3 * ty <= last; i += 4 * ty) {
            float h[4][V];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < V; ++j) h[u][j] = a.head[(i + u * ty) * width + col + j];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] += h[u][j];
        }
        for (; i <= last; i += ty)
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] += a.head[i * width + col + j];
    }
    if (last - range > 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) lds[(y * V + j) * a.tx + x] = s[j];
        __syncthreads();
        if (y == 0)
            for (int g = 1; g < ty; ++g)
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] += lds[(g * V + j) * a.tx + x];
    }
    if (y == 0 && c < a.packs) {
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] *= a.scale;
        store_f32<E, V>(a.grad + (int64_t)key * a.lde + col, s);
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

constexpr int64_t CLEAR_TWICE = (int64_t)192 << 20;
constexpr int64_t LOOKUP_MAX = ((int64_t)1 << 31) - 2, LOOKUP_MAX_WIDTH = (int64_t)1 << 21;

static int lookup_check(int64_t n_rows, int64_t width, int id_bytes, int64_t n_ids, int d0, int d1) {
    if (n_rows < 0 || width < 0 || n_ids < 0 || n_rows > LOOKUP_MAX || n_ids > LOOKUP_MAX || width > LOOKUP_MAX_WIDTH) return PLNLP_E_SHAPE;
    if ((id_bytes != 4 && id_bytes != 8) || !is_dtype(d0) || !is_dtype(d1)) return PLNLP_E_UNSUPPORTED;
    return 0;
}

// ids per counting tile: small tiles until there are four workgroups a CU
static int sort_rounds(int64_t n) { return n <= ((int64_t)1 << 20) ? 4 : 16; }
// sorted positions per group of lanes: about 2048 waves of 512 columns, 16 .. 256 positions each (twice as many waves walk no faster
// and leave twice as many runs to join)
static int grad_range(int64_t n, int64_t width) {
    int r = 16;
    while (r < 256 && (double)n * width > (double)r * 2048 * 512) r *= 2;
    return r;
}

// Is all of dE cleared in the sort's launches, instead of the rows without an id after it?  Rows with an id are then written twice: not
// where most rows have one, or where there are more bytes of them than the sort hides.  (us, in the sort's launches / after them: 131 071
// ids of 1 000 003 rows of 200 B 81 / 100, 4096 of 47 / 81; 180 000 of 235 868 rows of 1 KiB 127 / 132, but of 2 KiB 238 / 228; 131 072 of
// 65 536 rows of 1 KiB 76 / 69)
static bool clear_first(int64_t n_ids, int64_t n_rows, int64_t row_bytes) {
    return 4 * n_ids <= 3 * n_rows && n_ids * row_bytes <= CLEAR_TWICE;
}
static Clear make_clear(void* grad, int64_t ld, int64_t width, int64_t n_rows) {
    Clear c{};
    c.at = (char*)grad;
    c.total = (n_rows - 1) * ld + width;
    const bool flat = ld == width;
    c.ld = flat ? CLEAR_PIECE : ld;
    c.width = flat ? CLEAR_PIECE : width;
    c.pieces = flat ? (c.total + CLEAR_PIECE - 1) / CLEAR_PIECE : n_rows;
    c.unit = 16;
    while (((uintptr_t)grad | (uintptr_t)c.ld) & (c.unit - 1)) c.unit >>= 1;
    c.tx = lanes_for((c.width + c.unit - 1) / c.unit, LOOKUP_THREADS);
    return c;
}
static int clear_blocks(const Clear& c, int threads) {
    const int64_t per = (c.pieces + c.launches - 1) / c.launches, rows = threads / c.tx;
    return (int)std::min<int64_t>((per + rows - 1) / rows, 262144 / threads);
}

struct GradWorkspace { int64_t sorted[2], hist, total, head, tail, bytes; };
static GradWorkspace grad_workspace(int64_t n, int64_t width) {
    GradWorkspace w{};
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t a = at; at += (bytes + 255) / 256 * 256; return a; };
    const bool small = n <= SORT_SMALL;
    for (int i = 0; i < (small ? 1 : 2); ++i) w.sorted[i] = take(8 * n);
    const int64_t tile = sort_rounds(n) * LOOKUP_THREADS, tiles = (n + tile - 1) / tile;
    w.hist = take(small ? 0 : 4 * tiles << SORT_BITS);
    w.total = take(small ? 0 : 4 << SORT_BITS);
    const int64_t range = grad_range(n, width), ranges = (n + range - 1) / range;
    w.head = take(ranges * width * 4);
    w.tail = take(ranges * width * 4);
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
    // (one dimension of a grid holds less than 2^32 threads)
    const int64_t most = (int64_t)1 << 23;
    const dim3 grid((unsigned)std::min(blocks, most), (unsigned)((blocks + most - 1) / most));
    return with_dtype(table_dtype, [&](auto tt) { return with_dtype(out_dtype, [&](auto ot) { return with_id(id_bytes, [&](auto it) {
        return with_pack(v, [&](auto vc) {
            using T = decltype(tt); using O = decltype(ot); using I = decltype(it);
            constexpr int V = decltype(vc)::value;
            auto run = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, grid, dim3(LOOKUP_THREADS), 0, (hipStream_t)stream, (const T*)table, ld, n_rows,
                                   (int)packs, tx, (const I*)ids, n_ids, scale, (O*)out, ldo);
                return launch_status();
            };
            const bool stream_out = n_ids * width * (int64_t)sizeof(O) >= STREAM_BYTES;
            return !four ? run(lookup_kernel<T, O, I, V, 1, false>)
                 : stream_out ? run(lookup_kernel<T, O, I, V, 4, true>) : run(lookup_kernel<T, O, I, V, 4, false>);
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
    uint2* sorted[2] = {(uint2*)(ws + w.sorted[0]), (uint2*)(ws + w.sorted[1])};
    int cur = 0, rc = 0;
    const int es = dtype_size(grad_dtype);
    Clear clear = make_clear(grad, lde * es, width * es, n_rows);
    const bool cleared = n_ids > 0 && clear_first(n_ids, n_rows, width * es);
    // workgroups of a launch with `own` of its sort
    auto with_clear = [&](int own, int threads) {
        clear.first = own;
        return dim3((unsigned)(own + (cleared ? clear_blocks(clear, threads) : 0)));
    };
    if (n_ids && n_ids <= SORT_SMALL) {
        clear.launches = 1;
        const dim3 grid = with_clear((int)((n_ids + 63) / 64), 1024);
        rc = with_id(id_bytes, [&](auto it) {
            using I = decltype(it);
            hipLaunchKernelGGL((sort_small_kernel<I>), grid, dim3(1024), 0, s, (const I*)ids, (int)n_ids, n_rows, padding_id, sorted[0], clear);
            return launch_status();
        });
    } else if (n_ids) {
        int bits = 1;
        while (((int64_t)1 << bits) <= n_rows) ++bits;               // keys are 0 .. n_rows
        const int passes = (bits + SORT_BITS - 1) / SORT_BITS, digit = (bits + passes - 1) / passes;
        const int rounds = sort_rounds(n_ids), tile = rounds * LOOKUP_THREADS, bins = 1 << digit;
        const int tiles = (int)((n_ids + tile - 1) / tile);
        uint32_t* hist = (uint32_t*)(ws + w.hist);
        uint32_t* total = (uint32_t*)(ws + w.total);
        clear.launches = 3 * passes;
        for (int p = 0; p < passes && !rc; ++p) {
            const int shift = p * digit;
            rc = with_id(id_bytes, [&](auto it) {
                using I = decltype(it);
                auto pass = [&](auto first, auto count) {
                    constexpr bool F = decltype(first)::value;
                    constexpr int R = decltype(count)::value;
                    dim3 grid = with_clear(tiles, LOOKUP_THREADS);
                    clear.launch = 3 * p;
                    hipLaunchKernelGGL((sort_count_kernel<I, F, R>), grid, dim3(LOOKUP_THREADS), 4 * bins, s, (const I*)ids,
                                       sorted[cur], n_ids, n_rows, padding_id, shift, bins, hist, clear);
                    grid = with_clear((bins + OFFSET_DIGITS - 1) / OFFSET_DIGITS, 1024);
                    clear.launch = 3 * p + 1;
                    hipLaunchKernelGGL(sort_offsets_kernel, grid, dim3(1024), 0, s, hist, tiles, bins, total, clear);
                    grid = with_clear(tiles, LOOKUP_THREADS);
                    clear.launch = 3 * p + 2;
                    hipLaunchKernelGGL((sort_scatter_kernel<I, F, R>), grid, dim3(LOOKUP_THREADS), 4 * bins * (LOOKUP_THREADS / 64), s,
                                       (const I*)ids, sorted[cur], n_ids, n_rows, padding_id, shift, digit, hist, total, sorted[cur ^ 1], clear);
                    return launch_status();
                };
                auto sized = [&](auto first) {
                    return rounds == 4 ? pass(first, std::integral_constant<int, 4>{}) : pass(first, std::integral_constant<int, 16>{});
                };
                return p == 0 ? sized(std::true_type{}) : sized(std::false_type{});
            });
            cur ^= 1;
        }
    }
    if (rc) return rc;
    const int gs = dtype_size(gy_dtype);
    const int v = n_ids ? pick_pack(width, gy, ldg, gs, grad, lde, es) : pick_pack(width, grad, lde, es, grad, lde, es);
    const int64_t packs = width / v;
    const int tx = lanes_for(packs, 64);
    return with_dtype(gy_dtype, [&](auto gt) { return with_dtype(grad_dtype, [&](auto et) { return with_pack(v, [&](auto vc) {
        using G = decltype(gt); using E = decltype(et);
        constexpr int V = decltype(vc)::value;
        const int slabs = (int)((packs + tx - 1) / tx), range = grad_range(n_ids, width), ty = LOOKUP_THREADS / tx;
        const int64_t ranges = (n_ids + range - 1) / range, run_blocks = (ranges * slabs + ty - 1) / ty;
        const GradArgs<G, E, V> a{(const G*)gy, ldg, sorted[cur], n_ids, n_rows, (int)packs, tx, slabs, range, ranges, run_blocks,
                                  (float*)(ws + w.head), (float*)(ws + w.tail), scale, (E*)grad, lde};
        const int64_t clearing = cleared ? 0 : (n_rows + CLEAR_ROWS - 1) / CLEAR_ROWS;
        hipLaunchKernelGGL((grad_runs_kernel<G, E, V>), dim3((unsigned)(run_blocks + clearing)), dim3(LOOKUP_THREADS), 0, s, a);
        if (int e = launch_status()) return e;
        if (ranges > 1) {
            hipLaunchKernelGGL((grad_joins_kernel<G, E, V>), dim3((unsigned)(ranges - 1), slabs), dim3(LOOKUP_THREADS), 0, s, a);
            return launch_status();
        }
        return 0;
    }); }); });
}
