// y = act(x W^T + bias) + residual for 16-bit x, W, bias, residual (bf16 or fp16), and its gradients:
//   z = x W^T + bias;  y = act(z) + residual;   dz = dy * act'(z);  dx = dz W;  dW = dz^T x;  db = sum_rows dz;  d residual = dy
// Products on the matrix cores with f32 accumulation; bias, activation and residual on the f32 accumulators, ONE rounding to the
// stored type.  What is rounded besides:
//   act'(z), kept for the backward pass in the 16 bits z itself would take, so that it evaluates no exponential: FIXED point in steps of
//     2^-14 (|act'| <= 1.13), an absolute 2^-15, around |z| = 1 a sixth of what rounding z to fp16 (a fiftieth of what rounding it to
//     bf16) would do to dz; and where a unit is saturated (-2^-5 < act' < 0: z below -2.6 for gelu, -4.8 for silu) ten bits of
//     significand, a relative 2^-10 down to 2^-59, so that the gradients of a layer whose units all are keep their digits;
//   dz, which the two gradient products read as 16-bit operands: an error of the size of the result's own rounding, averaged over
//     the sums, and infinite past the type's range (fp16: |dy| above 57 900 where act' > 1).  A small dz (see TWO_TERMS) is kept as the
//     sum of two 16-bit terms instead: its few roundings would not average.
//
// One tile kernel serves the three products, written as C[m, n] = sum_k P(m, k) Q(n, k):
//   forward  P = x   (k contiguous)            Q = W (k contiguous)
//   dx       P = dz  (k contiguous)            Q = W read with k along its ROWS
//   dW       P = dz, Q = x, both with k along their rows
// A tile of P and of Q is staged global -> registers -> LDS as rows of 64 consecutive k (128 bytes); an operand with k along its
// rows is transposed on the way, in registers (8 k x 8 columns a thread, 32 v_perm_b32), so the product itself reads one layout.
// The 16-byte units of a row are XOR-swizzled (swz) so that the stores of both kinds and the reads hit all LDS banks.
// Q is the MFMA's first operand and its rows are dealt so that a lane ends up with groups of 8 CONSECUTIVE columns of one row of C: bias,
// residual and result move as 16-byte accesses straight from the accumulators, with no pass through LDS.
#include "half.hip.h"

namespace plnlp {

constexpr int BK = 64;

template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x4 go(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma<_Float16> {
    typedef f16x8 frag;
    static __device__ __forceinline__ f32x4 go(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// ---- activations ------------------------------------------------------------------------------------------
// (these run on every element of a result whose product may take less time than they do: an instruction counts)
__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.f + exp2_f(-LOG2E * z)); }

// the normal distribution function, g = exp(-z^2/2):  Phi(-|z|) = g * P(t), t = 1 / (1 + 0.45 |z| / sqrt 2), P a polynomial fitted to
// exp(u^2) erfc(u) / 2 on [0, 30] in RELATIVE error (1.2e-5, a fortieth of half an fp16 step), so the far negative tail keeps its digits
__device__ __forceinline__ float normal_cdf(float z, float g) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.45f * 0.70710678f, fabsf(z), 1.f));
    float p = 0.5f * -0.13489297032356262f;
    p = fmaf(p, t, 0.5f * 0.28983235359191895f);
    p = fmaf(p, t, 0.5f * 0.09164738655090332f);
    p = fmaf(p, t, 0.5f * 0.24759894609451294f);
    p = fmaf(p, t, 0.5f * 0.2518513798713684f);
    p = fmaf(p, t, 0.5f * 0.2539602816104889f);
    const float q = p * t * g;
    return z > 0.f ? 1.f - q : q;
}
constexpr float TANH_C = 1.5957691216057308f;                   // 2 sqrt(2 / pi)
constexpr float TANH_A = 0.044715f;

// act(z); SLOPE: and act'(z)
template <int ACT, bool SLOPE> __device__ __forceinline__ float act_of(float z, float& slope) {
    if (ACT == PLNLP_ACT_RELU) {
        if (SLOPE) slope = z > 0.f ? 1.f : (z == z ? 0.f : z);
        return z < 0.f ? 0.f : z;                                // (a NaN stays)
    }
    if (ACT == PLNLP_ACT_SILU) {
        const float s = sigmoid_f(z);
        if (SLOPE) slope = s * fmaf(z, 1.f - s, 1.f);
        return z * s;
    }
    if (ACT == PLNLP_ACT_GELU) {
        const float g = exp2_f((-0.5f * LOG2E * z) * z), c = normal_cdf(z, g);
        if (SLOPE) slope = fmaf(z * 0.3989422804014327f, g, c);
        return z * c;
    }
    if (ACT == PLNLP_ACT_GELU_TANH) {
        const float z2 = z * z, s = __builtin_amdgcn_rcpf(1.f + exp2_f(z * fmaf(-LOG2E * TANH_C * TANH_A, z2, -LOG2E * TANH_C)));
        const float y = z * s;
        // (z2 may be infinite where 1 - s is 0)
        if (SLOPE) slope = fmaf(fmaf(-y, s, y), fmaf(3.f * TANH_C * TANH_A, fminf(z2, 1e30f), TANH_C), s);
        return y;
    }
    return z;
}
// The slope in 16 bits.  Mostly in steps of 2^-14: adding 1.5 * 2^23 rounds to a whole number and leaves it in the low bits; a NaN becomes
// SLOPE_NAN, which no slope reaches (the smaller of a NaN and a number is the number).  -2^-5 <= slope < 0 is the f32's own sign, exponent
// and first nine bits, rounded: its upper 18 bits less those of -2^-59, counted up from -32768.  They end at -5120; the steps of the other
// negative slopes (gelu's reach -0.13) begin at -2121.  What lies between -2^-59 and 0 is 0, in steps.  (us, with the
// relative form / without: 131 072 x 256 x 256 with gelu forward 76 / 73, backward 131 / 128; 8192 x 4096 x 4096 309 / 308, 544 / 544)
constexpr float SLOPE_STEP = 1.f / 16384.f;
constexpr int SLOPE_NAN = 20000;
constexpr uint32_t SLOPE_TAIL = 0xa2000000u + ((uint32_t)32768 << 14);     // bits of -2^-59, less the shifted -32768 they are kept as
constexpr int SLOPE_TAIL_LO = -32767, SLOPE_TAIL_HI = -5120;
__device__ __forceinline__ int16_t pack_slope(float s) {
    const int tail = (int)(__float_as_uint(s) - SLOPE_TAIL + (1u << 13)) >> 14;
    const int steps = (int)__float_as_uint(fminf(fmaf(s, 16384.f, 12582912.f), 12582912.f + SLOPE_NAN));
    return (int16_t)((uint32_t)(tail - SLOPE_TAIL_LO) <= (uint32_t)(SLOPE_TAIL_HI - SLOPE_TAIL_LO) ? tail : steps);
}
__device__ __forceinline__ float unpack_slope(int16_t q) {
    const float tail = __uint_as_float(((uint32_t)(int)q << 14) + SLOPE_TAIL);
    return q <= SLOPE_TAIL_HI ? tail : q == SLOPE_NAN ? __builtin_nanf("") : (float)q * SLOPE_STEP;
}
// f(std::integral_constant<int, ACT>{}) of a run-time activation
template <typename F> __host__ __device__ __forceinline__ int with_act(int act, F&& f) {
    switch (act) {
        case PLNLP_ACT_RELU: return f(std::integral_constant<int, PLNLP_ACT_RELU>{});
        case PLNLP_ACT_SILU: return f(std::integral_constant<int, PLNLP_ACT_SILU>{});
        case PLNLP_ACT_GELU: return f(std::integral_constant<int, PLNLP_ACT_GELU>{});
        case PLNLP_ACT_GELU_TANH: return f(std::integral_constant<int, PLNLP_ACT_GELU_TANH>{});
        default: return f(std::integral_constant<int, PLNLP_ACT_NONE>{});
    }
}

// ---- what happens to a finished sum ---------------------------------------------------------------------------
template <typename T> struct Finish {
    const T* bias;          // nullable [n]
    const T* res;           // nullable [m, ldr]
    int16_t* slope;         // nullable [m, ldp]: act'(z), for the backward pass
    T*       out;           // [m, ldo]
    int64_t  ldr, ldp, ldo;
    int      vec;           // 8-column groups may move as 16 bytes
};
constexpr int PARTIAL = -1; // in the place of an activation: the sum is one K slice's, stored as it is

// V consecutive columns of row m from column n on (all inside the matrix); b = the bias there, res = the residual there (if f.res).
// LOOSE: at any alignment
template <int ACT, bool LOOSE, typename T, int V>
__device__ __forceinline__ void finish_with(const Finish<T>& f, float (&v)[V], const float (&b)[V], const typename PackOf<T, V, LOOSE>::type& res,
                                            int64_t m, int64_t n) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += b[j];
    float s[V];
    if (ACT != PLNLP_ACT_NONE && f.slope) {
        typedef typename PackOf<int16_t, V, LOOSE>::type P;
        P q;
#pragma unroll
        for (int j = 0; j < V; ++j) { v[j] = act_of<ACT, true>(v[j], s[j]); q.v[j] = pack_slope(s[j]); }
        *reinterpret_cast<P*>(f.slope + m * f.ldp + n) = q;
    } else
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = act_of<ACT, false>(v[j], s[j]);
    typedef typename PackOf<T, V, LOOSE>::type P;
    P o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = (T)(f.res ? v[j] + (float)res.v[j] : v[j]);
    *reinterpret_cast<P*>(f.out + m * f.ldo + n) = o;
}
template <int ACT, bool LOOSE, typename T, int V>
__device__ __forceinline__ void finish_cols(const Finish<T>& f, float (&v)[V], const float (&b)[V], int64_t m, int64_t n) {
    typedef typename PackOf<T, V, LOOSE>::type P;
    P res;
    if (f.res) res = *reinterpret_cast<const P*>(f.res + m * f.ldr + n);
    finish_with<ACT, LOOSE, T, V>(f, v, b, res, m, n);
}

// ---- the tile kernel --------------------------------------------------------------------------------------------
template <typename T> struct TileArgs {
    const T* p; const T* q;
    int64_t  ldp, ldq;
    int64_t  m, n, k;
    int64_t  plane;                                // P's second term lies this many elements behind its first
    int      terms;                                // 1, or 2: C = (P + P2) Q^T as one sum over twice as many steps
    int      tiles_m, tiles_n, slices, steps;      // steps: BK-steps per slice
    float*   sums;                                 // nullable [slices, m]: sum_k P(m, k) of each slice (PT, tiles of 128 x 128)
    float*   partial;                              // slices > 1: [slices, m, n]
    Finish<T> fin;
};

// Unit u of LDS row r sits at u ^ swz(r).  A 16-byte read serves 16 lanes a clock from 64 banks, two rows of 128 bytes: of the rows
// 0..15 of a fragment, or of the dealt Q rows (q_row), those of one parity sit in eight different units; so do the rows 8 apart that a
// transposed block's store touches at once (of one parity all: two clocks).
__device__ __forceinline__ int swz(int r) {
    return ((r >> 1) & 1) ^ (((r >> 3) & 1) << 1) ^ (((r >> 2) & 1) << 2) ^ (((r >> 4) & 1) * 5) ^ ((r >> 5) & 1);
}

// Q row (column of C) behind row r of the MFMA's tile t: lane group g = r >> 2 gets columns 32 (t / 2) + 8 g + 4 (t & 1) + 0..3, so its
// tiles 2h and 2h + 1 are eight consecutive columns, and the four groups' stores 64 consecutive bytes
__device__ __forceinline__ int q_row(int t, int r) { return 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3); }

// column j of a block of 8 k by 4 or 8 columns, held as eight rows of W words: its eight k
template <int W> __device__ __forceinline__ u32x4 block_column(const uint32_t* d, int j) {
    u32x4 o;
#pragma unroll
    for (int h = 0; h < 4; ++h)
        o[h] = __builtin_amdgcn_perm(d[(2 * h + 1) * W + (j >> 1)], d[(2 * h) * W + (j >> 1)], (j & 1) ? 0x07060302u : 0x05040100u);
    return o;
}

// How an operand's tile is read: element by element (any matrix), 16 bytes at any alignment (k >= BK), or 16 bytes at a time through a
// buffer descriptor (16-byte aligned rows of whole units)
enum { BY_ELEMENT = 0, LOOSELY = 1, ALIGNED = 2 };

// One operand's tile of R rows x BK on its way to LDS, staged by R threads, 8 loads of 16 bytes each: the first half of a workgroup's
// waves stages P, the other Q.  (With both staged by all, an operand with k along its rows came in blocks of 8 k x 4 columns, 8 bytes a
// lane, and a wave's load takes the address unit as long for 8 bytes a lane as for 16: dW of 4096 x 4096 over 8192 rows took 351 us
// against 234.)
// Every step issues the same loads, whatever the matrix's edges: rows past the last repeat it (their results are not stored); the last
// step of a k that is no multiple of BK begins early, and what it reads twice is cleared on the way to LDS.
// COLS: k lies along the operand's rows: blocks of 8 k x 8 columns.
template <typename T, int R, int MODE> struct Operand {
    static constexpr int N = 8;
    u32x4 reg[N];
    uint32_t off[2];                       // ALIGNED: bytes from the (uniform) first element of a load -- rows of a tile come R / 8 a load;
                                           // off[1]: in the last load that holds rows of the matrix, which the loads past it repeat
    int skip[2], valid[2];                 // of the step in each half of reg: k in [skip, valid) are real and not read before

    static __device__ __forceinline__ int tid() { return threadIdx.x & (R - 1); }
    static __device__ __forceinline__ int row_of(int i) { return (tid() + i * R) >> 3; }
    static __device__ __forceinline__ int unit() { return tid() & 7; }
    static __device__ __forceinline__ int col() { return tid() % (R / 8) * 8; }
    static __device__ __forceinline__ int group() { return tid() / (R / 8); }

    // rows: of the tile inside the matrix; k: the matrix's depth (COLS: at least BK unless BY_ELEMENT)
    template <bool COLS> __device__ __forceinline__ void begin(int64_t ld, int rows, int64_t k) {
        if (MODE != ALIGNED) return;
        if (COLS) off[0] = (uint32_t)((int64_t)(group() * 8) * ld + min(col(), rows - 8)) * 2;        // (whole groups of eight columns)
        else
#pragma unroll
            for (int l = 0; l < 2; ++l)
                off[l] = (uint32_t)((l ? min(tid() >> 3, (rows - 1) % (R / 8)) : tid() >> 3) * ld + min((int64_t)unit() * 8, k - 8)) * 2;
    }
    // loads LO .. HI - 1 of the eight (half of them or all); `base`: the tile's element at depth k0
    template <bool COLS, int LO, int HI> __device__ __forceinline__ void fetch(const T* base, int64_t ld, int rows, int64_t k0, int64_t k) {
        const int left = (int)min(k - k0, (int64_t)BK), back = MODE != BY_ELEMENT && k >= BK ? BK - left : 0;
        for (int h = LO / 4; h < HI / 4; ++h) { skip[h] = back; valid[h] = left + back; }
        base -= COLS ? back * ld : back;
        // (a buffer descriptor of the step's first element: the loads then take one 32-bit register of addresses each)
        const auto at = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, -1, 0x00027000);
        const int last = (rows - 1) / (R / 8);
#pragma unroll
        for (int i = LO; i < HI; ++i) {
            const int kk = group() * 8 + i;
            const T* p = COLS ? base + kk * ld + min(col(), rows - 8) : base + min(row_of(i), rows - 1) * ld + unit() * 8;
            if (MODE == ALIGNED)
                reg[i] = __builtin_bit_cast(u32x4, COLS ? __builtin_amdgcn_raw_buffer_load_b128(at, off[0], (int)(i * ld * 2), 0)
                                                        : __builtin_amdgcn_raw_buffer_load_b128(at, i < last ? off[0] : off[1], (int)(min(i, last) * (R / 8) * ld * 2), 0));
            else if (MODE == LOOSELY) reg[i] = __builtin_bit_cast(u32x4, *reinterpret_cast<const LoosePack<T, 8>*>(p));
            else {
                union { T t[8]; u32x4 u; } x;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (COLS) x.t[j] = (kk < left && col() + j < rows) ? base[kk * ld + col() + j] : (T)0.f;
                    else x.t[j] = unit() * 8 + j < left ? p[j] : (T)0.f;
                reg[i] = x.u;
            }
        }
    }
    // the same part of them into LDS rows of 128 bytes (COLS: all)
    template <bool COLS, int LO, int HI> __device__ __forceinline__ void store(char* lds, int rows) {
        static_assert(!COLS || HI - LO == N, "a block is transposed as a whole");
        const int skip = this->skip[LO / 4], valid = this->valid[LO / 4];
        const bool part = MODE != BY_ELEMENT && (skip > 0 || valid < BK);
        if (COLS) {
            if (part)
#pragma unroll
                for (int i = 0; i < N; ++i) if (group() * 8 + i < skip || group() * 8 + i >= valid) reg[i] = u32x4{0, 0, 0, 0};
            if (MODE == LOOSELY && (rows & 7)) {          // the last block of columns was read up to seven columns early
                const int early = min(max(col() - (rows - 8), 0), 7);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    uint64_t lo = ((uint64_t)reg[i][1] << 32) | reg[i][0], hi = ((uint64_t)reg[i][3] << 32) | reg[i][2];
                    if (early >= 4) { lo = hi; hi = 0; }
                    const int by = (early & 3) * 16;
                    if (by) { lo = (lo >> by) | (hi << (64 - by)); hi >>= by; }
                    reg[i] = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                *reinterpret_cast<u32x4*>(lds + (col() + j) * 128 + ((group() ^ swz(col() + j)) << 4)) =
                    block_column<4>(reinterpret_cast<const uint32_t*>(reg), j);
        } else {
            if (part) {
                const int lo = skip - unit() * 8, hi = valid - unit() * 8;      // elements [lo, hi) of the unit stay
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const uint32_t keep = (2 * h >= lo && 2 * h < hi ? 0xffffu : 0u) | (2 * h + 1 >= lo && 2 * h + 1 < hi ? 0xffff0000u : 0u);
#pragma unroll
                    for (int i = LO; i < HI; ++i) reg[i][h] &= keep;
                }
            }
#pragma unroll
            for (int i = LO; i < HI; ++i)
                *reinterpret_cast<u32x4*>(lds + row_of(i) * 128 + ((unit() ^ swz(row_of(i))) << 4)) = reg[i];
        }
    }
};

template <typename T, int BM, int BN, int WM, int WN, bool PT, bool QT, int MODE, int ACT>
__global__ __launch_bounds__(WM * WN * 64, 2) void tile_kernel(TileArgs<T> a) {
    constexpr int THREADS = WM * WN * 64, TM = BM / WM / 16;         // 16-row pieces of a wave's part; it is 64 columns wide
    static_assert(BN / WN == 64, "a wave covers 64 columns");
    typedef typename Mfma<T>::frag frag;
    extern __shared__ __attribute__((aligned(16))) char lds[];       // two buffers of P rows, then Q rows
    constexpr int BUF = (BM + BN) * 128;

    // Workgroups are dealt to the eight XCDs in turn: each XCD gets a contiguous run of tiles, so that its L2 holds the panels they share
    const int tiles = a.tiles_m * a.tiles_n, total = tiles * a.slices;
    const int per = total >> 3, extra = total & 7, xcd = blockIdx.x & 7, nth = blockIdx.x >> 3;
    const int id = xcd * per + min(xcd, extra) + nth;
    const int slice = id / tiles, tile = id % tiles;
    // and walks groups of 8 row panels column by column
    constexpr int GROUP = 8;
    const int group = tile / (GROUP * a.tiles_n), in_group = tile % (GROUP * a.tiles_n);
    const int g_rows = min(GROUP, a.tiles_m - group * GROUP);
    const int64_t m0 = (int64_t)(group * GROUP + in_group % g_rows) * BM, n0 = (int64_t)(in_group / g_rows) * BN;

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * 64;
    const int term_steps = (int)((a.k + BK - 1) / BK), first = slice * a.steps;
    const int steps = min(a.steps, term_steps * a.terms - first);
    const int rows_p = (int)min((int64_t)BM, a.m - m0), rows_q = (int)min((int64_t)BN, a.n - n0);

    f32x4 acc[TM][4];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    // sums over k of P, the bias gradient where P is dz: one more product, with a Q of ones, in the waves of the first column tile
    constexpr bool SUMS = PT && BM == 128;      // (large_tiles)
    const bool sum_p = SUMS && a.sums && n0 == 0 && wn == 0;
    f32x4 psum[SUMS ? TM : 1];
    frag ones;
#pragma unroll
    for (int i = 0; i < (SUMS ? TM : 1); ++i) psum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j] = (T)1.f;

    static_assert(BM == BN && THREADS == 2 * BM, "half of the threads stage P, half Q");
    const bool later = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= WM * WN / 2;     // the half that stages Q
    Operand<T, BM, MODE> mine;
    if (steps > 0) { if (later) mine.template begin<QT>(a.ldq, rows_q, a.k); else mine.template begin<PT>(a.ldp, rows_p, a.k); }
    // (a step past the last fetches the last again: the loads in flight at any point are the same in every step)
    typedef std::integral_constant<int, 0> Zero;
    typedef std::integral_constant<int, 4> Half;
    typedef std::integral_constant<int, 8> All;
    auto fetch = [&](int step, auto lo, auto hi) {
        constexpr int LO = decltype(lo)::value, HI = decltype(hi)::value;
        const int at = first + min(step, steps - 1), term = at >= term_steps;
        const int64_t k = (int64_t)(at - (term ? term_steps : 0)) * BK;
        if (later) mine.template fetch<QT, LO, HI>(QT ? a.q + k * a.ldq + n0 : a.q + n0 * a.ldq + k, a.ldq, rows_q, k, a.k);
        else {
            const T* p = a.p + (term ? a.plane : 0);
            mine.template fetch<PT, LO, HI>(PT ? p + k * a.ldp + m0 : p + m0 * a.ldp + k, a.ldp, rows_p, k, a.k);
        }
    };
    auto stage_all = [&](int buf) {
        char* b = lds + buf * BUF;
        if (later) mine.template store<QT, 0, 8>(b + BM * 128, rows_q); else mine.template store<PT, 0, 8>(b, rows_p);
    };
    // half of what a thread stages, where that operand's k is contiguous
    auto move_half = [&](int step, auto lo, auto hi) {
        constexpr int LO = decltype(lo)::value, HI = decltype(hi)::value;
        char* b = lds + (step & 1) * BUF;
        if constexpr (!QT) if (later) mine.template store<false, LO, HI>(b + BM * 128, rows_q);
        if constexpr (!PT) if (!later) mine.template store<false, LO, HI>(b, rows_p);
        fetch(step + 1, lo, hi);
    };
    auto q_frag = [&](const char* b, int ks, int t) {
        const int row = wn + q_row(t, r);
        return *reinterpret_cast<const frag*>(b + (BM + row) * 128 + (((ks * 4 + g) ^ swz(row)) << 4));
    };
    auto p_frag = [&](const char* b, int ks, int i) {
        const int row = wm + i * 16 + r;
        return *reinterpret_cast<const frag*>(b + row * 128 + (((ks * 4 + g) ^ swz(row)) << 4));
    };
    if (steps > 0) {
        fetch(0, Zero{}, All{});
        stage_all(0);
        fetch(1, Zero{}, All{});
        __syncthreads();
    }
    if constexpr (BM == 256) {
        // Two waves a SIMD, half a step apart: while waves 0..3 multiply (32 MFMAs, 512 clocks), waves 4..7 read their next fragments and
        // move the next tile, and the other way round; a barrier ends each half.  With both in step all of them waited for LDS at
        // the same time (8192 x 4096 x 4096: 334 us against 258).  A step's buffer is read in halves 4 s (waves 0..3) to 4 s + 3 (waves 4..7), the
        // other one written in the same halves.  Every wave passes 4 barriers a step and one more, the later half before,
        // the earlier half after.
        if (later) __syncthreads();
        for (int step = 0; step < steps; ++step) {
            const char* b = lds + (step & 1) * BUF;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const bool blocks = later ? QT : PT;
                if (ks == 1 && blocks) {         // (before the fragments are read: their registers are not there to spare)
                    stage_all((step + 1) & 1);
                    fetch(step + 2, Zero{}, All{});
                    __builtin_amdgcn_sched_barrier(0);
                }
                frag p[TM], q[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) q[t] = q_frag(b, ks, t);
#pragma unroll
                for (int i = 0; i < TM; ++i) p[i] = p_frag(b, ks, i);
                if (!blocks) { if (ks == 0) move_half(step + 1, Zero{}, Half{}); else move_half(step + 1, Half{}, All{}); }
                __syncthreads();
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int t = 0; t < 4; ++t) acc[i][t] = Mfma<T>::go(q[t], p[i], acc[i][t]);
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                __syncthreads();
            }
        }
        if (!later) __syncthreads();
    } else {
        for (int step = 0; step < steps; ++step) {
            const char* b = lds + (step & 1) * BUF;
            // (the other buffer was read before the barrier that ended the last step; what is fetched has a whole step to arrive in)
            stage_all((step + 1) & 1);
            fetch(step + 2, Zero{}, All{});
#pragma unroll
            for (int ks = 0; ks < BK / 32; ++ks) {
                frag q[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) q[t] = q_frag(b, ks, t);
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const frag p = p_frag(b, ks, i);
#pragma unroll
                    for (int t = 0; t < 4; ++t) acc[i][t] = Mfma<T>::go(q[t], p, acc[i][t]);
                    if (SUMS) if (sum_p) psum[SUMS ? i : 0] = Mfma<T>::go(ones, p, psum[SUMS ? i : 0]);
                }
            }
            __syncthreads();
        }
    }

    if (SUMS && sum_p && g == 0) {
#pragma unroll
        for (int i = 0; i < (SUMS ? TM : 1); ++i) {
            const int64_t m = m0 + wm + i * 16 + r;
            if (m < a.m) a.sums[(int64_t)slice * a.m + m] = psum[i][0];
        }
    }
    // lane (r, g) holds columns n + 32 h + 0..7 (h = 0, 1) of rows wm + 16 i + r
    const int64_t n = n0 + wn + 8 * g;
    int cols[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) cols[h] = (int)max(min((int64_t)8, a.n - n - 32 * h), (int64_t)0);
    float bias[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) bias[h][j] = (ACT != PARTIAL && a.fin.bias && j < cols[h]) ? (float)a.fin.bias[n + 32 * h + j] : 0.f;
    // (the residual two rows ahead: a load waited for next to its use would wait for the last row's stores as well)
    constexpr bool AHEAD = MODE == ALIGNED && ACT != PARTIAL;
    Pack<T, 8> res[AHEAD ? 3 : 1][2];
    auto ask = [&](int i) {
        const int64_t m = m0 + wm + i * 16 + r;
        if (!a.fin.res || i >= TM || m >= a.m) return;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (cols[h] > 0) res[i % 3][h] = *reinterpret_cast<const Pack<T, 8>*>(a.fin.res + m * a.fin.ldr + n + 32 * h);
    };
    if constexpr (AHEAD) { ask(0); ask(1); }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t m = m0 + wm + i * 16 + r;
        if (m >= a.m) continue;
        if constexpr (AHEAD) ask(i + 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t col = n + 32 * h;
            if (cols[h] <= 0) continue;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = acc[i][2 * h + (j >> 2)][j & 3];
            if constexpr (ACT == PARTIAL) {
                float* o = a.partial + ((int64_t)slice * a.m + m) * a.n + col;
                if (MODE == ALIGNED) store_f32<float, 8>(o, v);      // (n is whole groups of eight)
                else if (cols[h] == 8) {
                    LoosePack<float, 8> q;
#pragma unroll
                    for (int j = 0; j < 8; ++j) q.v[j] = v[j];
                    *reinterpret_cast<LoosePack<float, 8>*>(o) = q;
                } else
#pragma unroll
                    for (int j = 0; j < 8; ++j) if (j < cols[h]) o[j] = v[j];
            } else if constexpr (AHEAD) finish_with<ACT, false, T, 8>(a.fin, v, bias[h], res[i % 3][h], m, col);
            else if (cols[h] == 8) finish_cols<ACT, true, T, 8>(a.fin, v, bias[h], m, col);
            else
                for (int j = 0; j < cols[h]; ++j) {
                    float x[1] = {v[0]}, y[1] = {bias[h][0]};
#pragma unroll
                    for (int c = 1; c < 8; ++c) if (c == j) { x[0] = v[c]; y[0] = bias[h][c]; }
                    finish_cols<ACT, true, T, 1>(a.fin, x, y, m, col + j);
                }
        }
    }
}

// the slices' sums, then the finish: 64 lanes of V columns a workgroup, its four waves share the slices (wave w: w, w + 4, ...; joined in
// wave order), so that a small result over many slices still has loads enough in flight
template <typename T, int V, int ACT>
__global__ __launch_bounds__(256) void slices_kernel(const float* __restrict__ partial, int slices, int64_t m, int64_t n, Finish<T> fin) {
    __shared__ float lds[4][V][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t groups = n / V, i = (int64_t)blockIdx.x * 64 + lane, row = i / groups, col = (i - row * groups) * V;
    const bool in = row < m;
    float v[V] = {}, b[V] = {};
    if (in) {
        const float* p = partial + row * n + col;
#pragma unroll 8
        for (int s = wave; s < slices; s += 4) {
            float x[V];
            load_f32<float, V>(p + (int64_t)s * m * n, x);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] += x[j];
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) lds[wave][j][lane] = v[j];
    __syncthreads();
    if (wave || !in) return;
#pragma unroll
    for (int j = 0; j < V; ++j)
        for (int w = 1; w < 4; ++w) v[j] += lds[w][j][lane];
    if (fin.bias)
#pragma unroll
        for (int j = 0; j < V; ++j) b[j] = (float)fin.bias[col + j];
    finish_cols<ACT, V == 1, T, V>(fin, v, b, row, col);
}

// ---- many rows, a Q that fits LDS: Q stays there, P streams through registers -----------------------------------------
// A layer of a few hundred columns on 10^4 .. 10^6 rows is bound by its rows' bytes, and a tile of a few K steps (load, wait, multiply,
// finish) spends most of its time waiting for them.  Here one workgroup a CU stages all
// of Q in LDS once; after that its waves never meet again: each takes 16 rows, holds them as MFMA fragments (loaded straight from
// memory, 64 consecutive bytes a row and load) and walks Q's columns 64 at a time, finishing each group before the next -- so a
// wave needs 16 accumulators whatever n is -- and the next 16 rows, and the next columns' residual, load meanwhile.
// What it measured, and against what: at rows_fit.
// SLOPED: P = dy * slope, formed in the registers (the backward pass: dz = dy * act'(z), dx = dz W), and kept in dz for the
// weights' gradient; its column sums are taken here, before it is rounded.
template <typename T> struct RowsArgs {
    const T* p; int64_t ldp;
    const int16_t* slope; int64_t lds;      // SLOPED
    T* dz; int64_t ldz;
    float* sums;                            // SLOPED, nullable: [workgroups, k] column sums of dz
    const T* q; int64_t ldq;
    int64_t m; int n, k;
    Finish<T> fin;
};

// rows of KS * 64 bytes begin at the same bank (KS >= 4): the dealt Q rows of a fragment sit in sixteen different units instead
template <int KS> __device__ __forceinline__ int rows_swz(int r) { return KS < 4 ? swz(r) : (r & 3) ^ (((r >> 3) & 3) << 2); }

// the sum over the 16 lanes of a row of the wave, in each of them
__device__ __forceinline__ float row_sum(float v) {
    auto turned = [](float x, auto by) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + decltype(by)::value, 0xf, 0xf, true));
    };
    v += turned(v, std::integral_constant<int, 8>{});
    v += turned(v, std::integral_constant<int, 4>{});
    v += turned(v, std::integral_constant<int, 2>{});
    v += turned(v, std::integral_constant<int, 1>{});
    return v;
}

template <typename T, int KS, bool QT, bool SLOPED, int ACT>
__global__ __launch_bounds__(512) void rows_kernel(RowsArgs<T> a) {
    typedef typename Mfma<T>::frag frag;
    constexpr int THREADS = 512, WAVES = THREADS / 64, UNITS = KS * 4, ROW = KS * 64;
    constexpr bool EARLY = KS <= 8;          // registers for the next rows from the beginning of a tile; else from its last columns
    extern __shared__ __attribute__((aligned(16))) char lds[];       // [n rounded up to 64][KS * 32] of Q, [n rounded up to 64] of the bias
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int64_t tiles = (a.m + 15) / 16, stride = (int64_t)gridDim.x * WAVES;
    int64_t t = (int64_t)blockIdx.x * WAVES + wave;

    frag next[KS];                           // P as it lies in memory
    Pack<int16_t, 8> sl[SLOPED ? KS : 1];
    auto fetch = [&](int64_t tile) {
        const int64_t row = min(tile * 16 + r, a.m - 1);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int k = ks * 32 + g * 8;
            const frag zero = {};
            next[ks] = k < a.k ? *reinterpret_cast<const frag*>(a.p + row * a.ldp + k) : zero;
            if (SLOPED && k < a.k) sl[SLOPED ? ks : 0] = *reinterpret_cast<const Pack<int16_t, 8>*>(a.slope + row * a.lds + k);
        }
    };
    Pack<T, 8> res[2];                       // the residual of the columns that come next
    auto ask = [&](int64_t tile, int n0) {
        const int64_t m = tile * 16 + r;
        if (!a.fin.res || m >= a.m) return;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (n0 + 8 * g + 32 * h < a.n) res[h] = *reinterpret_cast<const Pack<T, 8>*>(a.fin.res + m * a.fin.ldr + n0 + 8 * g + 32 * h);
    };
    if (t < tiles) { fetch(t); ask(t, 0); }

    // (loads and stores of a wave complete in order: the bias lies in LDS because a load of it among the columns would wait for the
    // next rows and the last columns' stores; several loads of a thread in flight: one after the other they took longer than the rows)
    const int n64 = (a.n + 63) / 64 * 64;
    float* bias = reinterpret_cast<float*>(lds + n64 * ROW);
    for (int i = threadIdx.x; i < n64; i += THREADS) bias[i] = (a.fin.bias && i < a.n) ? (float)a.fin.bias[i] : 0.f;
    if (!QT) {
        constexpr int AHEAD = 8;
        for (int u0 = threadIdx.x; u0 < n64 * UNITS; u0 += THREADS * AHEAD) {
            u32x4 v[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int u = u0 + i * THREADS, row = u / UNITS, unit = u % UNITS;
                v[i] = u32x4{0, 0, 0, 0};
                if (row < a.n && unit * 8 < a.k) v[i] = *reinterpret_cast<const u32x4*>(a.q + (int64_t)row * a.ldq + unit * 8);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int u = u0 + i * THREADS, row = u / UNITS, unit = u % UNITS;
                if (row < n64) *reinterpret_cast<u32x4*>(lds + row * ROW + ((unit ^ rows_swz<KS>(row)) << 4)) = v[i];
            }
        }
    } else {
        constexpr int AHEAD = 3;
        const int quads = n64 / 4;
        for (int u0 = threadIdx.x; u0 < quads * UNITS; u0 += THREADS * AHEAD) {
            uint64_t d[AHEAD][8];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int u = u0 + i * THREADS, c = u % quads * 4, k0 = u / quads * 8;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int k = k0 + j;
                    d[i][j] = (c < a.n && k < a.k) ? *reinterpret_cast<const uint64_t*>(a.q + (int64_t)k * a.ldq + c) : 0;
                }
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int u = u0 + i * THREADS, c = u % quads * 4, unit = u / quads;
                if (unit >= UNITS) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *reinterpret_cast<u32x4*>(lds + (c + j) * ROW + ((unit ^ rows_swz<KS>(c + j)) << 4)) = block_column<2>(reinterpret_cast<const uint32_t*>(d[i]), j);
            }
        }
    }
    __syncthreads();

    float sums[SLOPED ? KS / 2 : 1] = {};          // of the tiles' 16 rows: lane r keeps every 16th of its group's 8 KS columns
    while (t < tiles) {
        const int64_t m = t * 16 + r;
        const bool in = m < a.m;
        frag p[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int k = ks * 32 + g * 8;
            p[ks] = next[ks];
            if (SLOPED) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = (float)next[ks][j] * unpack_slope(sl[SLOPED ? ks : 0].v[j]);
                    p[ks][j] = (T)d;
                    if (a.sums) {
                        const float all = row_sum(in && k < a.k ? d : 0.f);
                        sums[SLOPED ? ks / 2 : 0] += r == (ks & 1) * 8 + j ? all : 0.f;
                    }
                }
                if (k >= a.k) p[ks] = frag{};
                else if (in) *reinterpret_cast<frag*>(a.dz + m * a.ldz + k) = p[ks];
            }
        }
        const int64_t here = t;
        t += stride;
        for (int n0 = 0; n0 < a.n; n0 += 64) {
            const int n = n0 + 8 * g;
            const bool last = n0 + 64 >= a.n;
            const Pack<T, 8> mine[2] = {res[0], res[1]};
            if (!last) ask(here, n0 + 64);
            else if (t < tiles) ask(t, 0);
            if (EARLY && n0 == 0 && t < tiles) fetch(t);
            f32x4 acc[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = n0 + q_row(i, r);
                    acc[i] = Mfma<T>::go(*reinterpret_cast<const frag*>(lds + row * ROW + (((ks * 4 + g) ^ rows_swz<KS>(row)) << 4)), p[ks], acc[i]);
                }
            if (!EARLY && last && t < tiles) fetch(t);
            if (!in) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (n + 32 * h >= a.n) continue;
                float v[8], b[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = acc[2 * h + (j >> 2)][j & 3];
                    b[j] = bias[n + 32 * h + j];
                }
                finish_with<ACT, false, T, 8>(a.fin, v, b, mine[h], m, n + 32 * h);
            }
        }
    }
    if constexpr (SLOPED) {
        if (!a.sums) return;
        __syncthreads();                           // (Q is done with)
        float* part = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int i = 0; i < KS / 2; ++i) part[wave * KS * 32 + (2 * i + (r >> 3)) * 32 + g * 8 + (r & 7)] = sums[i];
        __syncthreads();
        for (int c = threadIdx.x; c < a.k; c += THREADS) {
            float v = 0.f;
            for (int w = 0; w < WAVES; ++w) v += part[w * KS * 32 + c];
            a.sums[(int64_t)blockIdx.x * a.k + c] = v;
        }
    }
}

// ---- few rows: the weights stream from memory once, straight into the MFMA's registers ---------------------------
// eight consecutive k of a row of which `left` remain
template <typename T, bool LOOSE> __device__ __forceinline__ typename Mfma<T>::frag few_unit(const T* p, int64_t left) {
    typedef typename Mfma<T>::frag frag;
    frag v = {};
    if (!LOOSE) {
        if (left > 0) v = *reinterpret_cast<const frag*>(p);
    } else if (left >= 8) v = __builtin_bit_cast(frag, *reinterpret_cast<const LoosePack<T, 8>*>(p));
    else if (left > 0)
#pragma unroll
        for (int j = 0; j < 7; ++j) if (j < left) v[j] = p[j];
    return v;
}

// A workgroup owns 16 columns of y and all (<= 16 * TM) rows; its waves share K, 64 at a time.  A lane reads 32 consecutive bytes of
// a weight row (the four lanes of a row 128): which k a lane holds is free as long as x is read the same way.  The waves'
// sums meet in LDS and are added in wave order.
template <typename T, int TM, int WAVES, bool LOOSE, int ACT>
__global__ __launch_bounds__(WAVES * 64) void few_rows_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, int m,
                                                              int64_t n, int64_t k, Finish<T> fin) {
    typedef typename Mfma<T>::frag frag;
    constexpr int AHEAD = TM == 1 ? 4 : 2;                 // 64-k units in flight a wave
    __shared__ float part[WAVES][TM][16][17];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const T* wr = w + min(n0 + r, n - 1) * ldw + g * 16;
    const T* xr[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) xr[i] = x + (int64_t)min(i * 16 + r, m - 1) * ldx + g * 16;
    f32x4 acc[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t units = (k + 63) / 64;
    for (int64_t u0 = wave; u0 < units; u0 += WAVES * AHEAD) {
        frag a[AHEAD][2], b[AHEAD][TM][2];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int64_t at = (u0 + j * WAVES) * 64;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t left = k - (at + g * 16 + h * 8);           // (whole groups of eight unless LOOSE)
                a[j][h] = few_unit<T, LOOSE>(wr + at + h * 8, left);
#pragma unroll
                for (int i = 0; i < TM; ++i) b[j][i][h] = few_unit<T, LOOSE>(xr[i] + at + h * 8, left);
            }
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < TM; ++i) acc[i] = Mfma<T>::go(a[j][h], b[j][i][h], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[wave][i][r][4 * g + j] = acc[i][j];      // [row of x][column]
    __syncthreads();
    for (int e = threadIdx.x; e < TM * 256; e += WAVES * 64) {
        const int i = e >> 8, row = (e >> 4) & 15, c = e & 15;
        const int64_t mm = i * 16 + row, nn = n0 + c;
        float v[1] = {0.f}, b[1] = {0.f};
#pragma unroll
        for (int s = 0; s < WAVES; ++s) v[0] += part[s][i][row][c];
        if (mm >= m || nn >= n) continue;
        if (fin.bias) b[0] = (float)fin.bias[nn];
        finish_cols<ACT, true, T, 1>(fin, v, b, mm, nn);
    }
}

// ---- dz = dy * act'(z), and the column sums of dz ---------------------------------------------------------------------
// 256 / tx rows of tx lanes, V columns a lane; a workgroup takes `rows` consecutive rows and leaves their column sums (of dz before it
// is rounded) in partial[block, :].  plane > 0: what rounding leaves of dz goes `plane` elements behind it.  SLOPE false: dz = dy, sums only.
template <typename T, int V, bool SLOPE>
__global__ __launch_bounds__(256) void act_back_kernel(const T* __restrict__ gy, int64_t ldg, const int16_t* __restrict__ slope, int64_t lds_,
                                                       T* __restrict__ dz, int64_t ldz, int64_t plane, int64_t m, int packs, int tx, int64_t rows,
                                                       float* __restrict__ partial) {
    __shared__ float lds[256 * V];
    const int x = threadIdx.x & (tx - 1), y = threadIdx.x / tx, ty = 256 / tx;
    const int64_t lo = (int64_t)blockIdx.x * rows, hi = min(lo + rows, m);
    for (int c0 = blockIdx.y * tx; c0 < packs; c0 += gridDim.y * tx) {
        const int c = c0 + x;
        float s[V] = {};
        if (c < packs) {
            const int64_t col = (int64_t)c * V;
            int64_t i = lo + y;
            auto go = [&](auto count) {
                constexpr int U = decltype(count)::value;
                Pack<T, V> d[U];
                Pack<int16_t, V> q[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    d[u] = *reinterpret_cast<const Pack<T, V>*>(gy + (i + u * ty) * ldg + col);
                    if (SLOPE) q[u] = *reinterpret_cast<const Pack<int16_t, V>*>(slope + (i + u * ty) * lds_ + col);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float z[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        z[j] = (float)d[u].v[j] * (SLOPE ? unpack_slope(q[u].v[j]) : 1.f);
                        s[j] += z[j];
                    }
                    if (SLOPE) {
                        T* o = dz + (i + u * ty) * ldz + col;
                        if (plane) {
                            // (past the type's range: its largest number and the rest; infinities and NaN have none)
                            constexpr float MOST = std::is_same<T, _Float16>::value ? 65504.f : 3.38953139e38f;
                            float rest[V];
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                const float all = z[j];
                                const bool finite = fabsf(all) < __builtin_inff();
                                if (finite) z[j] = fminf(fmaxf(all, -MOST), MOST);
                                rest[j] = finite ? all - (float)(T)z[j] : 0.f;
                            }
                            store_f32<T, V>(o + plane, rest);
                        }
                        store_f32<T, V>(o, z);
                    }
                }
            };
            for (; i + 3 * ty < hi; i += 4 * ty) go(std::integral_constant<int, 4>{});
            for (; i < hi; i += ty) go(std::integral_constant<int, 1>{});
        }
        if (!partial) continue;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) lds[(y * V + j) * tx + x] = s[j];
        __syncthreads();
        if (y == 0 && c < packs) {
            for (int t = 1; t < ty; ++t)
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] += lds[(t * V + j) * tx + x];
#pragma unroll
            for (int j = 0; j < V; ++j) partial[(int64_t)blockIdx.x * packs * V + (int64_t)c * V + j] = s[j];
        }
    }
}

// the blocks' column sums, added: 16 columns a workgroup, 64 threads a column with up to 16 loads in flight each
template <typename T>
__global__ __launch_bounds__(1024) void col_join_kernel(const float* __restrict__ partial, int blocks, int64_t n, T* __restrict__ out) {
    __shared__ float lds[16][16];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const int64_t col = (int64_t)blockIdx.x * 16 + x;
    float s = 0.f;
    if (col < n)
#pragma unroll 16
        for (int b = y; b < blocks; b += 64) s += partial[(int64_t)b * n + col];
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    if ((threadIdx.x & 63) < 16) lds[threadIdx.x >> 6][x] = s;
    __syncthreads();
    if (threadIdx.x < 16 && col < n) {
        for (int w = 1; w < 16; ++w) s += lds[w][x];
        out[col] = (T)s;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
// Up to 16 rows the weights' bytes are all there is, whatever their number (1 x 4096 x 4096: 8.5 us against 13.9 on the tile kernel; 1 x
// 16384 x 4096 25, 5.3 TB/s).  Up to 64 rows every workgroup reads x again for its 16 columns: only small and not too deep weights
// (us: 64 x 1024 x 1024 7.0 / 9.8, 40 x 2048 x 2048 9.8 / 10.6; but 32 x 1024 x 4096 12.7 / 10.8, 64 x 8192 x 4096 43 / 25).
static bool few_rows(int64_t m, int64_t n, int64_t k) { return m <= 16 || (m <= 64 && k <= 2048 && n * k <= ((int64_t)1 << 22)); }
constexpr int64_t LINEAR_MAX = (int64_t)1 << 31, LINEAR_MAX_N = (int64_t)1 << 26;   // rows and depth; columns

static bool units_ok(const void* p, int64_t ld, int64_t along) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && along % 8 == 0; }

// Tile shape and K slices of a product.  256 x 256 tiles read LDS and the caches half as often an MFMA as 128 x 128 ones, but one
// workgroup of them fills a CU: they are taken where they leave less than an eighth of their area empty and make at least three
// quarters of the chip's 256 workgroups, alone or with K cut into slices of at least 24 steps.  Else 128 x 128: alone
// where they make three quarters of a workgroup a CU (4096 x 1024 x 1024: 20 us, in two slices 32), else with K cut: a step takes a lone
// workgroup about 0.7 us and 2^18 sums of a slice, written and read again, about 0.4, which s = sqrt(1.75 steps / (m n / 2^18)) slices
// balance -- two steps a slice at least, two workgroups a CU at most.  (us, so / with four steps a slice: 300 x 300 x 300 9.7 / 12.1,
// 1024 x 1024 x 1024 16.5 / 19.9, 2048 x 512 x 512 12.3 / 14.6, 1000 x 256 x 2048 14.1 / 14.2; / with twice as many: 9.7, 20.0, 14.7,
// 15.2)  (us: 8192 x 4096 x 4096 258 against 345; dW of 4096 x 4000 over 8192
// rows 230 against 372; of 2048 x 1024 over 16384 rows, eight slices, 83 against 107)
struct Plan { bool big; int tiles_m, tiles_n, slices, steps; };
static Plan plan_product(int64_t m, int64_t n, int64_t k, int terms = 1) {
    Plan p{};
    const int64_t steps = (k + BK - 1) / BK * terms;
    auto tiles = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const int64_t t256 = tiles(m, 256) * tiles(n, 256), cut = t256 ? std::max<int64_t>(1, 256 / t256) : 1;
    p.big = m > 0 && n > 0 && (double)t256 * 65536 * 0.875 <= (double)m * n && t256 * cut >= 192 && steps / cut >= (cut > 1 ? 24 : 8);
    const int b = p.big ? 256 : 128;
    p.tiles_m = (int)tiles(m, b);
    p.tiles_n = (int)tiles(n, b);
    const int64_t t = (int64_t)p.tiles_m * p.tiles_n;
    int64_t s = p.big ? cut : t == 0 || t >= 192 ? 1 : 512 / t;
    const int64_t balanced = (int64_t)std::sqrt(1.75 * (double)steps * 262144.0 / std::max(1.0, (double)m * (double)n));
    s = std::max<int64_t>(1, std::min(s, p.big ? steps / 4 : std::min(steps / 2, balanced)));
    p.steps = (int)((steps + s - 1) / s);
    p.slices = p.steps ? (int)((steps + p.steps - 1) / p.steps) : 1;
    if (p.slices < 1) p.slices = 1;
    return p;
}
static int64_t plan_bytes(const Plan& p, int64_t m, int64_t n) { return p.slices > 1 ? (int64_t)p.slices * m * n * 4 : 0; }

template <typename T, int BM, int BN, int WM, int WN, bool PT, bool QT, int MODE, int ACT>
static int launch_tile(const TileArgs<T>& a, hipStream_t s) {
    auto kernel = tile_kernel<T, BM, BN, WM, WN, PT, QT, MODE, ACT>;
    constexpr int LDS = 2 * (BM + BN) * 128;
    if (LDS > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.tiles_m * a.tiles_n * a.slices)), dim3(WM * WN * 64), LDS, s, a);
    return launch_status();
}

// Q in LDS for the rows kernel: 32-k pieces a row (0: it does not take the product).  Every workgroup reads all of Q once, so there
// have to be rows enough for each: 128 a column of the result (256 workgroups times n k of Q against m k of P, twice).
//   us, with gelu, slope and residual, here / on the tile kernel, forward: 131 072 x 256 x 256 74 / 77 (3.6 TB/s), 32 768 x 256 x 256 20.5 /
//   20.5 but 16 384 x 256 x 256 18.2 / 15.1; 262 144 x 64 x 256 42 / 66, 16 384 x 64 x 64 6.8 / 10.8, 8192 x 64 x 64 6.7 / 10.6;
//   backward: 124 / 130, 50.5 / 49.4, 43.6 / 37.7, 110 / 121, 20 / 26, 19 / 24
constexpr int64_t ROWS_MIN = 8192, ROWS_PER_COLUMN = 128, ROWS_LDS = 155648;
static int rows_fit(int64_t m, int64_t n, int64_t k, int64_t most_k = 512) {
    if (m < ROWS_MIN || m < ROWS_PER_COLUMN * n || n == 0 || k == 0 || k > most_k) return 0;
    for (int ks : {2, 4, 8, 12, 16})
        if (ks * 32 >= k) return (n + 63) / 64 * 64 * (ks * 64 + 4) <= ROWS_LDS ? ks : 0;
    return 0;
}

static int64_t rows_blocks(int64_t m) { return std::min<int64_t>((m + 127) / 128, 256); }      // eight waves of 16 rows, one workgroup a CU

template <typename T, int KS, bool QT, bool SLOPED, int ACT> static int launch_rows(const RowsArgs<T>& a, hipStream_t s) {
    auto kernel = rows_kernel<T, KS, QT, SLOPED, ACT>;
    constexpr int THREADS = 512;
    const int lds = (a.n + 63) / 64 * 64 * (KS * 64 + 4);
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows_blocks(a.m)), dim3(THREADS), lds, s, a);
    return launch_status();
}
template <typename T, bool QT, bool SLOPED, int ACT> static int run_rows(int ks, const RowsArgs<T>& a, hipStream_t s) {
    if (ks == 2) return launch_rows<T, 2, QT, SLOPED, ACT>(a, s);
    if (ks == 4) return launch_rows<T, 4, QT, SLOPED, ACT>(a, s);
    if constexpr (!SLOPED) {                 // (deeper with the slopes would not fit the registers: rows_fit's most_k)
        if (ks == 12) return launch_rows<T, 12, QT, SLOPED, ACT>(a, s);
        if (ks == 16) return launch_rows<T, 16, QT, SLOPED, ACT>(a, s);
    }
    return launch_rows<T, 8, QT, SLOPED, ACT>(a, s);
}

// how the tile kernel reads a product's operands (32-bit offsets inside a tile; an operand with k along its rows needs a whole step of them)
static int product_mode(bool vec, bool pt, const void* p, int64_t ldp, bool qt, const void* q, int64_t ldq, int64_t m, int64_t n, int64_t k) {
    if (vec && ldp < ((int64_t)1 << 22) && ldq < ((int64_t)1 << 22) && (k >= BK || !(pt || qt)) && k > 0 &&
        units_ok(p, ldp, pt ? m : k) && units_ok(q, ldq, qt ? n : k)) return ALIGNED;
    return k >= BK && (!pt || m >= 8) && (!qt || n >= 8) ? LOOSELY : BY_ELEMENT;
}
// does it run on 256 x 256 tiles?  (Those take no TileArgs::sums: who wants them asks here first.)
static bool large_tiles(const Plan& pl, int mode) { return pl.big && mode == ALIGNED; }

// C = P Q^T on the tile kernel, with its finish (ACT: the activation of the finish)
template <typename T, bool PT, bool QT, int ACT>
static int product(const T* p, int64_t ldp, int64_t plane, const T* q, int64_t ldq, int64_t m, int64_t n, int64_t k, const Finish<T>& fin,
                   float* partial, hipStream_t s, float* sums = nullptr) {
    const int terms = plane ? 2 : 1;
    const Plan pl = plan_product(m, n, k, terms);
    TileArgs<T> a{p, q, ldp, ldq, m, n, k, plane, terms, pl.tiles_m, pl.tiles_n, pl.slices, pl.steps, sums, partial, fin};
    const int mode = product_mode(fin.vec, PT, p, ldp, QT, q, ldq, m, n, k);
    auto run = [&](auto act) {
        constexpr int A = decltype(act)::value;
        if (large_tiles(pl, mode)) return launch_tile<T, 256, 256, 2, 4, PT, QT, ALIGNED, A>(a, s);
        if (pl.big) { a.tiles_m = (int)((m + 127) / 128); a.tiles_n = (int)((n + 127) / 128); }
        return mode == ALIGNED ? launch_tile<T, 128, 128, 2, 2, PT, QT, ALIGNED, A>(a, s)
             : mode == LOOSELY ? launch_tile<T, 128, 128, 2, 2, PT, QT, LOOSELY, A>(a, s)
                               : launch_tile<T, 128, 128, 2, 2, PT, QT, BY_ELEMENT, A>(a, s);
    };
    if (pl.slices == 1) return run(std::integral_constant<int, ACT>{});
    if (int rc = run(std::integral_constant<int, PARTIAL>{})) return rc;
    const int v = fin.vec ? 4 : 1;
    const dim3 blocks((unsigned)((m * (n / v) + 63) / 64));
    if (v == 4) hipLaunchKernelGGL((slices_kernel<T, 4, ACT>), blocks, dim3(256), 0, s, partial, pl.slices, m, n, fin);
    else hipLaunchKernelGGL((slices_kernel<T, 1, ACT>), blocks, dim3(256), 0, s, partial, pl.slices, m, n, fin);
    return launch_status();
}

template <typename T> static Finish<T> make_finish(const void* bias, const void* res, int64_t ldr, int16_t* slope, int64_t ldp, void* out, int64_t ldo,
                                                   int64_t n) {
    Finish<T> f{(const T*)bias, (const T*)res, slope, (T*)out, ldr, ldp, ldo, 0};
    f.vec = units_ok(out, ldo, n) && (!res || units_ok(res, ldr, n)) && (!slope || units_ok(slope, ldp, n));
    return f;
}

template <typename F> static int with_half(int d, F&& f) { return d == PLNLP_DTYPE_BF16 ? f(__bf16{}) : f(_Float16{}); }

static int linear_check(int64_t m, int64_t n, int64_t k, int act, int dtype) {
    if (m < 0 || n < 0 || k < 0 || m >= LINEAR_MAX || n >= LINEAR_MAX_N || k >= LINEAR_MAX) return PLNLP_E_SHAPE;
    // (a launch holds less than 2^32 threads: 256 for a tile of each of the three products, 64 for a column where columns are joined)
    const int64_t tm = (m + 127) / 128, tn = (n + 127) / 128, tk = (k + 127) / 128, most = (int64_t)1 << 24;
    if (tm * tn >= most || tm * tk >= most || tn * tk >= most) return PLNLP_E_SHAPE;
    if (act < PLNLP_ACT_NONE || act > PLNLP_ACT_SILU) return PLNLP_E_UNSUPPORTED;
    if (dtype != PLNLP_DTYPE_BF16 && dtype != PLNLP_DTYPE_F16) return PLNLP_E_UNSUPPORTED;
    return 0;
}
static int matrix_check(const void* p, int64_t ld, int64_t rows, int64_t cols) {
    if (!rows || !cols) return 0;
    if (!p) return PLNLP_E_NULL;
    if ((uintptr_t)p % 2) return PLNLP_E_ALIGN;
    return ld < cols ? PLNLP_E_SHAPE : 0;
}

// a dz of at most this many elements is kept as two 16-bit terms: its products are latency-bound and the second term costs nothing to
// speak of, while with few elements the rounding of a single one shows in the result
constexpr int64_t TWO_TERMS = 16384;

struct BackPlan { int64_t dz, plane, ldz, sums, partial, bytes, rows, blocks, slices; };
static int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }
static BackPlan back_plan(int64_t m, int64_t n, int64_t k, int act) {
    BackPlan b{};
    // rows per workgroup of act_back_kernel: about 1024 workgroups, 64 rows at least
    b.rows = std::max<int64_t>(64, (m + 1023) / 1024);
    b.blocks = (m + b.rows - 1) / b.rows;
    b.ldz = (n + 7) / 8 * 8;
    const bool two = act != PLNLP_ACT_NONE && m * n <= TWO_TERMS;
    b.plane = two ? m * b.ldz : 0;
    int64_t at = 0;
    b.dz = at; at += act == PLNLP_ACT_NONE ? 0 : round256(m * b.ldz * 2 * (two ? 2 : 1));
    b.slices = plan_product(n, k, m, two ? 2 : 1).slices;        // of the weights' gradient, which may bring the column sums of dy
    b.sums = at; at += round256(std::max(std::max(b.blocks, b.slices), rows_blocks(m)) * n * 4);
    b.partial = at;
    const int terms = two ? 2 : 1;
    at += round256(std::max(plan_bytes(plan_product(m, k, n, terms), m, k), plan_bytes(plan_product(n, k, m, terms), n, k)));
    b.bytes = at;
    return b;
}

}  // namespace plnlp

extern "C" int64_t plnlp_linear_act_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (m <= 0 || n <= 0 || k < 0 || plnlp::few_rows(m, n, k)) return 0;
    return plnlp::plan_bytes(plnlp::plan_product(m, n, k), m, n);
}

extern "C" int plnlp_linear_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual, int64_t ldr,
                                int act, int64_t m, int64_t n, int64_t k, int16_t* slope, int64_t lds, void* out, int64_t ldo, int dtype,
                                void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace plnlp;
    if (int rc = linear_check(m, n, k, act, dtype)) return rc;
    if (m == 0 || n == 0) return 0;
    int rc = matrix_check(x, ldx, m, k);
    if (!rc) rc = matrix_check(w, ldw, n, k);
    if (!rc) rc = matrix_check(out, ldo, m, n);
    if (!rc && residual) rc = matrix_check(residual, ldr, m, n);
    if (!rc && slope) rc = matrix_check(slope, lds, m, n);
    if (!rc && bias && (uintptr_t)bias % 2) rc = PLNLP_E_ALIGN;
    if (rc) return rc;
    const int64_t need = plnlp_linear_act_workspace_bytes(m, n, k);
    hipStream_t s = (hipStream_t)stream;
    return with_half(dtype, [&](auto tt) { return with_act(act, [&](auto at) {
        using T = decltype(tt);
        constexpr int A = decltype(at)::value;
        const Finish<T> fin = make_finish<T>(bias, residual, ldr, slope, lds, out, ldo, n);
        if (few_rows(m, n, k)) {
            const bool aligned = units_ok(x, ldx, k) && units_ok(w, ldw, k);
            const unsigned blocks = (unsigned)((n + 15) / 16);
            auto run = [&](auto kernel, int waves) {
                hipLaunchKernelGGL(kernel, dim3(blocks), dim3(waves * 64), 0, s, (const T*)x, ldx, (const T*)w, ldw, (int)m, n, k, fin);
                return launch_status();
            };
            auto sized = [&](auto loose) {
                constexpr bool L = decltype(loose)::value;
                if (m <= 16) return k >= 1024 ? run(few_rows_kernel<T, 1, 8, L, A>, 8) : run(few_rows_kernel<T, 1, 4, L, A>, 4);
                return m <= 32 ? run(few_rows_kernel<T, 2, 8, L, A>, 8) : run(few_rows_kernel<T, 4, 8, L, A>, 8);
            };
            return aligned ? sized(std::false_type{}) : sized(std::true_type{});
        }
        const int ks = rows_fit(m, n, k);
        if (ks && fin.vec && units_ok(x, ldx, k) && units_ok(w, ldw, k)) {
            const RowsArgs<T> a{(const T*)x, ldx, nullptr, 0, nullptr, 0, nullptr, (const T*)w, ldw, m, (int)n, (int)k, fin};
            return run_rows<T, false, false, A>(ks, a, s);
        }
        if (need && (!workspace || workspace_bytes < need)) return PLNLP_E_WORKSPACE;
        if ((uintptr_t)workspace % 16) return PLNLP_E_ALIGN;
        return product<T, false, false, A>((const T*)x, ldx, 0, (const T*)w, ldw, m, n, k, fin, (float*)workspace, s);
    }); });
}

extern "C" int64_t plnlp_linear_act_backward_workspace_bytes(int64_t m, int64_t n, int64_t k, int act) {
    if (m <= 0 || n <= 0 || k < 0) return 0;
    return plnlp::back_plan(m, n, k, act).bytes;
}

extern "C" int plnlp_linear_act_backward(const void* gy, int64_t ldg, const int16_t* slope, int64_t lds, int act, const void* x, int64_t ldx,
                                         const void* w, int64_t ldw, int64_t m, int64_t n, int64_t k, void* dx, int64_t lddx, void* dw,
                                         int64_t lddw, void* db, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace plnlp;
    if (int rc = linear_check(m, n, k, act, dtype)) return rc;
    int rc = matrix_check(gy, ldg, m, n);
    if (!rc && act != PLNLP_ACT_NONE) rc = matrix_check(slope, lds, m, n);
    if (!rc && dw) rc = matrix_check(x, ldx, m, k);
    if (!rc && dx) rc = matrix_check(w, ldw, n, k);
    if (!rc && dx) rc = matrix_check(dx, lddx, m, k);
    if (!rc && dw) rc = matrix_check(dw, lddw, n, k);
    if (!rc && db && (uintptr_t)db % 2) rc = PLNLP_E_ALIGN;
    if (rc) return rc;
    const int64_t need = plnlp_linear_act_backward_workspace_bytes(m, n, k, act);
    if (need && (!workspace || workspace_bytes < need)) return PLNLP_E_WORKSPACE;
    if ((uintptr_t)workspace % 16) return PLNLP_E_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    return with_half(dtype, [&](auto tt) {
        using T = decltype(tt);
        const BackPlan b = back_plan(m, n, k, act);
        char* ws = (char*)workspace;
        const bool has_act = act != PLNLP_ACT_NONE;
        const T* dz = has_act ? (const T*)(ws + b.dz) : (const T*)gy;
        const int64_t ldz = has_act ? b.ldz : ldg, plane = b.plane;
        float* sums = (float*)(ws + b.sums);
        float* partial = (float*)(ws + b.partial);
        const bool want_dx = dx && m > 0 && k > 0, want_dw = dw && n > 0 && k > 0;
        const bool vec = units_ok(gy, ldg, n) && (!has_act || units_ok(slope, lds, n));
        // many rows and weights that fit LDS: dz and its column sums are formed on the way to dx; without an activation dz is dy and
        // its sums come with dw, unless so many rows sum up to few results that dw takes the large tiles (393 216 rows of 256 x 256)
        const Finish<T> fin_x = make_finish<T>(nullptr, nullptr, 0, nullptr, 0, dx, lddx, k);
        const Finish<T> fin_w = make_finish<T>(nullptr, nullptr, 0, nullptr, 0, dw, lddw, k);
        const int ks = want_dx && vec && !plane && fin_x.vec && (uintptr_t)w % 8 == 0 && ldw % 4 == 0 ? rows_fit(m, k, n, has_act ? 256 : 512) : 0;
        const bool sums_in_dx = ks && has_act;
        const bool sums_in_dw = ks && !has_act && want_dw &&
                                !large_tiles(plan_product(n, k, m), product_mode(fin_w.vec, true, dz, ldz, true, x, ldx, n, k, m));
        int64_t sum_blocks = m > 0 ? b.blocks : 0;
        if (m > 0 && n > 0 && ((has_act && !ks) || (db && !sums_in_dx && !sums_in_dw))) {
            const int64_t packs = vec ? n / 8 : n;
            int tx = 1;
            while (tx < 64 && tx < packs) tx <<= 1;
            auto run = [&](auto kernel) {
                const unsigned slabs = (unsigned)std::min<int64_t>((packs + tx - 1) / tx, 64);
                hipLaunchKernelGGL(kernel, dim3((unsigned)b.blocks, slabs), dim3(256), 0, s, (const T*)gy, ldg, slope, lds, (T*)(ws + b.dz), ldz, plane, m,
                                   (int)packs, tx, b.rows, db ? sums : nullptr);
                return launch_status();
            };
            const int e = has_act ? (vec ? run(act_back_kernel<T, 8, true>) : run(act_back_kernel<T, 1, true>))
                                  : (vec ? run(act_back_kernel<T, 8, false>) : run(act_back_kernel<T, 1, false>));
            if (e) return e;
        }
        if (ks) {
            const RowsArgs<T> a{(const T*)gy, ldg, slope, lds, (T*)(ws + b.dz), ldz, db ? sums : nullptr, (const T*)w, ldw, m, (int)k, (int)n, fin_x};
            if (sums_in_dx) sum_blocks = rows_blocks(m);
            if (int e = has_act ? run_rows<T, true, true, PLNLP_ACT_NONE>(ks, a, s) : run_rows<T, true, false, PLNLP_ACT_NONE>(ks, a, s)) return e;
        } else if (want_dx) {
            if (int e = product<T, false, true, PLNLP_ACT_NONE>(dz, ldz, plane, (const T*)w, ldw, m, k, n, fin_x, partial, s)) return e;
        }
        if (want_dw) {
            if (sums_in_dw) sum_blocks = b.slices;
            if (int e = product<T, true, true, PLNLP_ACT_NONE>(dz, ldz, plane, (const T*)x, ldx, n, k, m, fin_w, partial, s,
                                                               sums_in_dw && db ? sums : nullptr)) return e;
        }
        if (db && n > 0) {
            hipLaunchKernelGGL((col_join_kernel<T>), dim3((unsigned)((n + 15) / 16)), dim3(1024), 0, s, (const float*)sums, (int)sum_blocks, n, (T*)db);
            if (int e = launch_status()) return e;
        }
        return 0;
    });
}
