// Operators on rows of scores: log probabilities of given tokens with entropy and top
// alternatives, the routing of rows to experts, and the gradients of both.
#include <type_traits>

#include "common.h"

#define SC_WG 256
#define SC_WAVES (SC_WG / 64)
#define SC_LOG2E 1.44269504088896340736f
#define SC_LN2 0.69314718055994530942f

// ---- elements ------------------------------------------------------------------------------

typedef uint32_t sc_u4 __attribute__((ext_vector_type(4)));

// A type of the scores: V of them are 16 bytes, which is what a lane loads or stores at a time.  Rows start
// wherever their stride puts them, so these accesses are aligned to the element only (the hardware takes
// 16-byte accesses at any address).
struct F32 {
    typedef float E;
    enum { V = 4 };
    static __device__ __forceinline__ float get(const E* p) { return *p; }
    static __device__ __forceinline__ void put(E* p, float v) { *p = v; }
    static __device__ __forceinline__ void unpack(sc_u4 w, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ sc_u4 pack(const float* x) {
        sc_u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i]);
        return w;
    }
};
struct BF16 {
    typedef uint16_t E;
    enum { V = 8 };
    static __device__ __forceinline__ float get(const E* p) { return __uint_as_float((uint32_t)*p << 16); }
    // to nearest, ties to even; a NaN stays one
    static __device__ __forceinline__ E bits(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
    static __device__ __forceinline__ void put(E* p, float v) { *p = bits(v); }
    static __device__ __forceinline__ void unpack(sc_u4 w, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ sc_u4 pack(const float* x) {
        sc_u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bits(x[2 * i]) | (uint32_t)bits(x[2 * i + 1]) << 16;
        return w;
    }
};
struct F16 {
    typedef _Float16 E;
    enum { V = 8 };
    static __device__ __forceinline__ float get(const E* p) { return (float)*p; }
    static __device__ __forceinline__ void put(E* p, float v) { *p = (_Float16)v; }
    static __device__ __forceinline__ void unpack(sc_u4 w, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
            x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
        }
    }
    static __device__ __forceinline__ sc_u4 pack(const float* x) {
        sc_u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]) << 16;
        return w;
    }
};

template <typename E>
struct __attribute__((packed, aligned(sizeof(E)))) ScVec {
    sc_u4 v;
};

template <typename X>
__device__ __forceinline__ sc_u4 sc_load(const typename X::E* p) {
    return ((const ScVec<typename X::E>*)p)->v;
}
template <typename X>
__device__ __forceinline__ void sc_store(typename X::E* p, sc_u4 w) {
    ((ScVec<typename X::E>*)p)->v = w;
}
// The same for what is read or written once and is larger than the caches, or not worth their room: 8192 x 32768 bfloat16
// gradient 193 -> 181 us, of a routing of 65536 x 128 9.9 -> 7.4 us.  (Rows of a few hundred columns lose by it, 55 -> 61 us.)
template <typename X>
__device__ __forceinline__ sc_u4 sc_load_once(const typename X::E* p) {
    return __builtin_nontemporal_load(&((const ScVec<typename X::E>*)p)->v);
}
template <typename X>
__device__ __forceinline__ void sc_store_once(typename X::E* p, sc_u4 w) {
    __builtin_nontemporal_store(w, &((ScVec<typename X::E>*)p)->v);
}

// Columns at .. at + V - 1 of a row that ends before column n; what lies behind is not read and becomes -inf.
template <typename X>
__device__ __forceinline__ void sc_read(const typename X::E* x, int at, int n, float* f) {
    if (at + X::V <= n) {
        X::unpack(sc_load<X>(x + at), f);
    } else {
#pragma unroll
        for (int e = 0; e < X::V; ++e) f[e] = at + e < n ? X::get(x + at + e) : -INFINITY;
    }
}

// One whole number per (score, place): larger for the larger score, then for the lower place.  No key is 0.
__device__ __forceinline__ uint32_t sc_order(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 counts as 0
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sc_unorder(uint32_t o) { return __uint_as_float((o >> 31) ? (o & 0x7fffffffu) : ~o); }
__device__ __forceinline__ uint64_t sc_key(float x, uint32_t at) { return ((uint64_t)sc_order(x) << 32) | (uint32_t)~at; }
__device__ __forceinline__ float sc_key_score(uint64_t k) { return sc_unorder((uint32_t)(k >> 32)); }
__device__ __forceinline__ uint32_t sc_key_place(uint64_t k) { return ~(uint32_t)k; }

// ---- reductions ----------------------------------------------------------------------------

struct SumOp { template <typename T> __device__ T operator()(T a, T b) const { return a + b; } };
struct MaxOp { template <typename T> __device__ T operator()(T a, T b) const { return a > b ? a : b; } };
struct DMaxOp { __device__ double operator()(double a, double b) const { return fmax(a, b); } };
struct FMaxOp { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct MinOp { template <typename T> __device__ T operator()(T a, T b) const { return a < b ? a : b; } };

template <int CTRL>
__device__ __forceinline__ uint32_t sc_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}

// One step of a butterfly: p and q are v of the two neighbouring groups of STEP lanes.  Below 16 lanes p is a lane's own, so that
// the two groups have them in opposite orders and what is made of them must not depend on it; from 16 on the order is the same.
// Within a group of STEP lanes v is the same already, so that any lane of the other group will do: the row mirrors stand
// in for the exchanges at 4 and 8, and the row swaps of v with itself give both sides at 16 and 32.  (An exchange through
// LDS, as __shfl_xor, issues at a third of their rate.)
template <int STEP>
__device__ __forceinline__ void sc_pair(uint32_t v, uint32_t& p, uint32_t& q) {
    if constexpr (STEP >= 16) {
        const auto both = STEP == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false)
                                     : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        p = both[0];
        q = both[1];
    } else {
        p = v;
        q = STEP == 1 ? sc_dpp<0xB1>(v)     // quad_perm 1 0 3 2
            : STEP == 2 ? sc_dpp<0x4E>(v)   // quad_perm 2 3 0 1
            : STEP == 4 ? sc_dpp<0x141>(v)  // row_half_mirror
                        : sc_dpp<0x140>(v); // row_mirror
    }
}
template <int STEP>
__device__ __forceinline__ void sc_pair(float v, float& p, float& q) {
    uint32_t a, b;
    sc_pair<STEP>(__float_as_uint(v), a, b);
    p = __uint_as_float(a);
    q = __uint_as_float(b);
}
template <int STEP>
__device__ __forceinline__ void sc_pair(int v, int& p, int& q) {
    uint32_t a, b;
    sc_pair<STEP>((uint32_t)v, a, b);
    p = (int)a;
    q = (int)b;
}
template <int STEP>
__device__ __forceinline__ void sc_pair(uint64_t v, uint64_t& p, uint64_t& q) {
    uint32_t a, b, c, d;
    sc_pair<STEP>((uint32_t)v, a, b);
    sc_pair<STEP>((uint32_t)(v >> 32), c, d);
    p = (uint64_t)c << 32 | a;
    q = (uint64_t)d << 32 | b;
}
template <int STEP>
__device__ __forceinline__ void sc_pair(double v, double& p, double& q) {
    uint64_t a, b;
    sc_pair<STEP>((uint64_t)__double_as_longlong(v), a, b);
    p = __longlong_as_double(a);
    q = __longlong_as_double(b);
}
template <int STEP, typename T, typename F>
__device__ __forceinline__ T sc_step(T v, F f) {
    T p, q;
    sc_pair<STEP>(v, p, q);
    return f(p, q);
}

// Over the first `lanes` (a power of two) lanes and each further group of as many, every lane of the wavefront taking
// part; all of a group get its result.
template <typename T, typename F>
__device__ __forceinline__ T sc_lanes(T v, int lanes, F f) {
    if (lanes > 1) v = sc_step<1>(v, f);
    if (lanes > 2) v = sc_step<2>(v, f);
    if (lanes > 4) v = sc_step<4>(v, f);
    if (lanes > 8) v = sc_step<8>(v, f);
    if (lanes > 16) v = sc_step<16>(v, f);
    if (lanes > 32) v = sc_step<32>(v, f);
    return v;
}
template <typename T, typename F>
__device__ __forceinline__ T sc_wave(T v, F f) {
    return sc_lanes(v, 64, f);
}

template <int WG, typename T, typename F>
__device__ T sc_block(T v, F f, T* lds) {  // lds: WG / 64 values
    v = sc_wave(v, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < WG / 64; ++i) v = f(v, lds[i]);
    return v;
}

// How many of the n keys (in LDS, n <= the room there) are larger.
__device__ __forceinline__ int sc_rank(const uint64_t* keys, int n, uint64_t key) {
    int rank = 0, j = 0;
    for (; j + 8 <= n; j += 8) {  // eight reads in flight
#pragma unroll
        for (int i = 0; i < 8; ++i) rank += keys[j + i] > key;
    }
    for (; j < n; ++j) rank += keys[j] > key;
    return rank;
}

// ---- log probabilities ---------------------------------------------------------------------
//
// One pass over the row.  A lane keeps the largest score m it has seen, S = sum 2^t and W = sum 2^t t with
// t = (x - m) log2 e, and takes a chunk of scores at a time: the chunk's maximum first, then S and W are carried
// to it (S' = 2^d S, W' = 2^d (W + S d), d the step of m in the same units), then the chunk is added.  Lanes,
// wavefronts and slices of a row are joined by the same rule.  log S and the entropy log S - ln 2 W / S follow,
// both sums of terms of one sign.  The statistics are float32; a lane adds n / 64 (a wavefront to the row) or
// n / 256 terms one by one.
//
// The alternatives need no second look at the row either: the K-th largest of the lanes' maxima, tau, is a lower
// bound of the K-th largest score, so that only the few segments (a lane's part of a chunk) whose maximum reaches
// tau are read again, and only their scores that reach it are put into order.

struct Stat {
    float m, s, w;
};

// 2^-256 is 0 in float32: below that t only has to stay finite, 0 * -inf being no number.
__device__ __forceinline__ float sc_floor_t(float t) { return fmaxf(t, -256.0f); }

// st carried to the maximum `to` >= st.m.
__device__ __forceinline__ void sc_carry(Stat& st, float to) {
    const float base = to == -INFINITY ? 0.0f : to;
    const float d = sc_floor_t((st.m - base) * SC_LOG2E), f = __builtin_amdgcn_exp2f(d);
    st.w = f * fmaf(st.s, d, st.w);
    st.s *= f;
    st.m = to;
}

template <int N>
__device__ __forceinline__ float sc_max(const float* x, float m) {
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
    return m;
}

template <int N>
__device__ __forceinline__ void sc_add(Stat& st, const float* x) {
    const float base = st.m == -INFINITY ? 0.0f : st.m;
    float s[2] = {0, 0}, w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = (x[i] - base) * SC_LOG2E, e = __builtin_amdgcn_exp2f(t);
        s[i & 1] += e;  // a NaN, or +inf, shows up here
        w[i & 1] = fmaf(e, sc_floor_t(t), w[i & 1]);
        // (keeps W's sum here: left alone the compiler forms it behind S's, with every t and e in a register)
        if (i % 8 == 7) asm volatile("" : "+v"(s[0]), "+v"(s[1]), "+v"(w[0]), "+v"(w[1]));
    }
    st.s += s[0] + s[1];
    st.w += w[0] + w[1];
}

__device__ __forceinline__ void sc_join_wave(Stat& st) {
    sc_carry(st, sc_wave(st.m, FMaxOp()));
    st.s = sc_wave(st.s, SumOp());
    st.w = sc_wave(st.w, SumOp());
}

// The same over a workgroup; every thread gets it.  The caller synchronises before wave_stat is used again.
template <int WG>
__device__ __forceinline__ void sc_join_block(Stat& st, Stat* wave_stat) {
    constexpr int WAVES = WG / 64;
    sc_join_wave(st);
    if ((threadIdx.x & 63) == 0) wave_stat[threadIdx.x >> 6] = st;
    __syncthreads();
    st = wave_stat[threadIdx.x & (WAVES - 1)];
    sc_carry(st, sc_lanes(st.m, WAVES, FMaxOp()));
    st.s = sc_lanes(st.s, WAVES, SumOp());
    st.w = sc_lanes(st.w, WAVES, SumOp());
}

struct RowStat {
    float base, log_sum, entropy;  // base: the largest score, 0 for an empty row
    bool empty, bad;               // nothing above -inf; a NaN or +inf among the scores
};

__device__ __forceinline__ RowStat sc_row_stat(const Stat& st) {
    RowStat q;
    q.empty = st.s == 0;
    q.bad = st.s != st.s;
    q.base = st.m == -INFINITY ? 0.0f : st.m;
    q.log_sum = q.empty ? 0.0f : logf(st.s);
    q.entropy = q.empty ? 0.0f : q.log_sum - SC_LN2 * st.w / st.s;
    return q;
}

struct LogprobArgs {
    const void* x;
    int64_t rows, stride;
    int cols;
    const int32_t* widths;
    const int64_t* tokens;
    int n_tok, top;
    float *logp, *entropy, *stats, *top_logp;
    int32_t* top_index;
    int lanes;               // to a short row
    int slices, slice_cols;  // a long row in parts, one workgroup each (slice_cols a multiple of its chunk)
    Stat* part;              // [rows][slices]
    uint64_t* part_keys;     // [rows][slices][top], 0: none
};

__device__ __forceinline__ int sc_width(const int32_t* widths, int64_t r, int cols) {
    return widths ? pd_clampi(widths[r], 0, cols) : cols;
}

// Thread i's token of row r (n_tok <= 64) and its score, asked for before the row is read.
struct RowToken {
    bool have, given;
    float x;
};

template <typename X>
__device__ __forceinline__ RowToken sc_row_token(const LogprobArgs& a, int64_t r, const typename X::E* x, int n, int i) {
    RowToken q = {i < a.n_tok, false, -INFINITY};
    if (q.have) {
        const int64_t tok = a.tokens[r * a.n_tok + i];
        q.given = tok >= 0;
        if (q.given && tok < n) q.x = X::get(x + tok);
    }
    return q;
}

// Statistics and token log probabilities of row r.
__device__ __forceinline__ void sc_put_row(const LogprobArgs& a, int64_t r, const Stat& st, const RowStat& q, const RowToken& tok, int i) {
    if (i == 0) {
        if (a.stats) {
            a.stats[3 * r] = st.m;
            a.stats[3 * r + 1] = q.log_sum;
            a.stats[3 * r + 2] = q.entropy;
        }
        if (a.entropy) a.entropy[r] = q.entropy;
    }
    if (tok.have) a.logp[r * a.n_tok + i] = !tok.given ? 0.0f : q.empty ? -INFINITY : (tok.x - q.base) - q.log_sum;
}

// Alternative k of row r; key 0: the row has no more scores, what lies behind it counts as -inf.
__device__ __forceinline__ void sc_put_top(const LogprobArgs& a, int64_t r, int k, uint64_t key, const RowStat& q) {
    const int64_t at = r * a.top + k;
    a.top_index[at] = q.bad ? -1 : key ? (int)sc_key_place(key) : k;
    a.top_logp[at] = q.bad ? NAN : q.empty || !key ? -INFINITY : (sc_key_score(key) - q.base) - q.log_sum;
}

// The K-th largest of the orders o[0 .. N-1] of a wavefront's lanes.  For a few, one maximum after the other; for more, by
// its bits from the first in which they differ: as soon as exactly K values lie above the bits so far it is the least of
// them.
template <int N>
__device__ __forceinline__ uint32_t sc_kth(const uint32_t* o, int K) {
    if (N == 1 && K <= 6) {
        uint32_t left = o[0], top = sc_wave(left, MaxOp());
        for (int k = 1; k < K; ++k) {
            const uint64_t equal = __ballot(left == top);
            if ((threadIdx.x & 63) == (uint32_t)__ffsll((unsigned long long)equal) - 1) left = 0;
            top = sc_wave(left, MaxOp());
        }
        return top;
    }
    uint32_t hi = o[0], lo = o[0];
#pragma unroll
    for (int i = 1; i < N; ++i) hi = MaxOp()(hi, o[i]), lo = MinOp()(lo, o[i]);
    hi = __builtin_amdgcn_readfirstlane(sc_wave(hi, MaxOp()));
    lo = __builtin_amdgcn_readfirstlane(sc_wave(lo, MinOp()));
    if (hi == lo) return hi;
    const int bits = 32 - __clz(hi ^ lo);
    uint32_t t = bits == 32 ? 0 : hi >> bits << bits;
    for (int bit = bits - 1; bit >= 0; --bit) {
        const uint32_t trial = t | 1u << bit;
        int count = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) count += __popcll(__ballot(o[i] >= trial));
        if (count >= K) t = trial;
        if (count == K) {
            uint32_t least = ~0u;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (o[i] >= trial && o[i] < least) least = o[i];
            return sc_wave(least, MinOp());
        }
    }
    return t;
}

// A number that exactly K of a row's scores f reach, one wavefront to the row, or the K-th largest itself where there are
// equals; lo, hi: orders of which at least K scores reach the first, and none exceeds the second.
template <int N>
__device__ __forceinline__ float sc_kth_all(const float* f, int K, uint32_t lo, uint32_t hi) {
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    if (lo == hi) return sc_unorder(hi);
    const int bits = 32 - __clz(hi ^ lo);
    uint32_t t = bits == 32 ? 0 : hi >> bits << bits;
    for (int bit = bits - 1; bit >= 0; --bit) {
        const uint32_t trial = t | 1u << bit;
        if (trial > hi) continue;
        const float at = sc_unorder(trial);
        int count = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) count += __popcll(__ballot(f[i] >= at));
        if (count >= K) t = trial;
        if (count == K) break;
    }
    return sc_unorder(t > lo ? t : lo);
}

// ---- 16, 32 or 64 lanes to the row: up to 2048 columns, all of them in registers ----------------
//
// Some ten instructions a score, and a few hundred for the reductions, the alternatives and the results, which the rows of a
// wavefront share; so rows are packed as tightly as their number allows, nothing is exchanged through LDS but the handful of
// candidates, and wavefronts do not wait for each other.  Bound by latency first, with few wavefronts to cover it: 16-bit rows
// of 24 scores a lane take 107 registers, of 32 scores 125, which leaves four wavefronts to a SIMD, 4096 on the chip.  Issue is
// 38 of 63 to 74 us at 65536 x 1000 bfloat16 (floor 26) and 4.5 of 14.5 at 9216 ragged rows of up to 656, whose 4608
// wavefronts do not all start at once: 8192 rows take 10.8 us, 8448 13.8.

#define SC_WAVE_CAND 128  // candidates of a wavefront's rows

template <typename X, int NV>
__global__ __launch_bounds__(SC_WG) void k_token_logprobs_rows(LogprobArgs a) {
    constexpr int V = X::V, N = NV * V;
    __shared__ uint64_t cand[SC_WAVES][SC_WAVE_CAND];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int L = a.lanes, l = lane & (L - 1), first = lane & ~(L - 1), per_wave = 64 / L;
    const uint64_t row_lanes = (L == 64 ? ~0ull : (1ull << L) - 1) << first, before = row_lanes & ((1ull << lane) - 1);
    const int room = SC_WAVE_CAND / per_wave;
    uint64_t* mine = cand[wave] + first / L * room;
    const int64_t tiles = (a.rows + per_wave - 1) / per_wave;
    for (int64_t tile = (int64_t)blockIdx.x * SC_WAVES + wave; tile < tiles; tile += (int64_t)gridDim.x * SC_WAVES) {
        const int64_t r = tile * per_wave + lane / L;
        const bool on = r < a.rows;
        const typename X::E* x = (const typename X::E*)a.x + (on ? r : a.rows - 1) * a.stride;
        const int n = on ? sc_width(a.widths, r, a.cols) : 0;
        RowToken tok = {};
        if (on && a.n_tok <= L) tok = sc_row_token<X>(a, r, x, n, l);
        float f[N];
#pragma unroll
        for (int u = 0; u < NV; ++u) sc_read<X>(x, (u * L + l) * V, n, f + u * V);
        const float m = sc_max<N>(f, -INFINITY);
        Stat st = {sc_lanes(m, L, FMaxOp()), 0, 0};
        sc_add<N>(st, f);
        st.s = sc_lanes(st.s, L, SumOp());
        st.w = sc_lanes(st.w, L, SumOp());
        const RowStat q = sc_row_stat(st);
        if (on) {
            sc_put_row(a, r, st, q, tok, l);
            if (a.n_tok > L)
                for (int i = l; i < a.n_tok; i += L) sc_put_row(a, r, st, q, sc_row_token<X>(a, r, x, n, i), i);
        }
        if (!a.top) continue;
        const bool plain = on && !q.bad && !q.empty;
        float tau;
        if (L == 64 && a.top > 6) {
            const uint32_t o = sc_order(m);
            tau = sc_unorder(sc_kth<1>(&o, a.top));
        } else {  // a few: one maximum after the other
            float left = m;
            tau = sc_lanes(left, L, FMaxOp());
            for (int k = 1; k < a.top; ++k) {
                const uint64_t equal = __ballot(left == tau) & row_lanes;
                if (lane == __ffsll((unsigned long long)equal) - 1) left = -INFINITY;
                tau = sc_lanes(left, L, FMaxOp());
            }
        }
        // What reaches tau is marked without a branch, and the few are read again: N branches with a key each would take
        // 80 registers more.
        uint32_t take;
        int count;
        for (bool once = L == 64;; once = false) {
            take = 0;
#pragma unroll
            for (int i = N - 1; i >= 0; --i) take = take + take + (f[i] >= tau);
            if (__any(tau == -INFINITY)) {  // then what lies behind the row does, too
                uint32_t valid = 0;
                for (int u = 0; u < NV; ++u) valid |= ((1u << pd_clampi(n - (u * L + l) * V, 0, V)) - 1) << (u * V);
                take &= valid;
            }
            if (!plain) take = 0;
            count = sc_lanes(__popc(take), L, SumOp());
            if (!once || count <= room) break;
            // With many alternatives, or more than there are lanes in use, too many scores reach the lanes' bound (at 64 some
            // 250 of 2048): it is taken on from there among all of them.  (Rows that share a wavefront are then done one
            // alternative after the other, as below, which takes as long: 8000 x 100 with sixteen, a wavefront each, and 8192,
            // two to one, 26 us both.)
            tau = sc_kth_all<N>(f, a.top, sc_order(tau), sc_order(st.m));
        }
        if (__any(count > room)) {
            // Too many scores equal to tau (a masked row, a constant one): of those the first that make up the number.
            uint32_t above = 0;
#pragma unroll
            for (int i = N - 1; i >= 0; --i) above = above + above + (f[i] > tau);
            if (!plain) above = 0;
            const uint32_t equal = take & ~above;
            const bool cut = count > room;
            int have = sc_lanes(__popc(above), L, SumOp());
            if (cut) take = above;
            for (int u = 0; u < NV; ++u) {
                uint32_t bits = equal >> (u * V) & ((1u << V) - 1);
                const int c = __popc(bits);
                int upto = c;  // an inclusive scan over the row's lanes
                for (int d = 1; d < L; d <<= 1) {
                    const int o = __shfl_up(upto, d, L);
                    if (l >= d) upto += o;
                }
                for (int drop = c - pd_clampi(a.top - have - (upto - c), 0, c); drop > 0; --drop) bits &= ~(1u << (31 - __clz((int)bits)));
                if (cut) take |= bits << (u * V);
                have += __shfl(upto, first + L - 1);
            }
            count = sc_lanes(__popc(take), L, SumOp());
        }
        const bool fits = !__any(count > room);
        int from = 0;
        while (fits && __any(take != 0)) {
            const int i = __ffs((int)take) - 1, at = i / V * L * V + (i & (V - 1)) + l * V;
            const bool in = take != 0;
            take &= take - 1;
            const uint64_t mask = __ballot(in);
            if (in) mine[from + __popcll(mask & before)] = sc_key(X::get(x + at), at);
            from += __popcll(mask & row_lanes);
        }
        pd_wave_sync();
        if (fits) {
            for (int i = l; i < count; i += L) {
                const uint64_t key = mine[i];
                const int rank = sc_rank(mine, count, key);
                if (rank < a.top) sc_put_top(a, r, rank, key, q);
            }
            if (on && l < a.top && (!plain || l >= count)) sc_put_top(a, r, l, q.empty ? sc_key(-INFINITY, l) : 0, q);
        } else {
            uint64_t prev = ~0ull;  // many large scores in few lanes: one after the other
            for (int k = 0; k < a.top; ++k) {
                uint64_t best = 0;
                for (int at = l; at < n; at += L) {
                    const uint64_t key = sc_key(X::get(x + at), at);
                    if (key < prev && key > best) best = key;
                }
                prev = sc_lanes(best, L, MaxOp());
                if (on && l == 0) sc_put_top(a, r, k, prev, q);
            }
        }
        pd_wave_sync();  // the next rows' candidates go to the same place
    }
}

// ---- a workgroup to the row, or to a slice of it ------------------------------------------------
//
// Chunks of WG * 32 columns, 32 to a thread in 16-byte loads.  With many rows: 64 or 256 threads, and workgroups enough on
// a CU to keep the loads coming while others reduce; bound by the memory (4096 x 131072 bfloat16 with five alternatives:
// 196 us, 5.5 TB/s).  With 64 the LDS holds sixteen on a CU, 4096 on the chip: 4096 x 4096 takes 13 us, 4352 x 4096 15.6 and
// 8192 x 4096 22 (floor 13).  With 256 a row of 16384 columns takes 1.6 us of its CU, and 5.6 to start and to end: 1400 of
// them 15.5 us (floor 9), as long as 1536.  With few long rows: 1024 threads that load a chunk while they add the one before; bound by
// instruction issue on the one CU (131072 columns 9 us) and by the latency of the steps behind the last load.  Still fewer
// long rows are cut into slices, joined by k_token_logprobs_join.

#define SC_PER_THREAD 32
#define SC_MAX_CHUNKS(WG) ((WG) == 1024 ? 8 : 16)
#define SC_SEGS 128   // segments that are read again
#define SC_CAND 512   // candidates that are put into order

template <int WG>
struct TopShared {
    uint32_t seg_max[SC_MAX_CHUNKS(WG)][WG];
    uint32_t part_max[256];
    uint64_t cand[SC_CAND];
    uint64_t wave_best[WG / 64];
    uint16_t segs[SC_SEGS];
    uint32_t tau;
    int n_seg, n_cand, scanned[WG / 64];
};

// Reads the segments whose maximum is at least `from` again and collects their scores from there on (orders).
// False: there are more of either than there is room for.
template <typename X, int WG>
__device__ bool sc_collect(TopShared<WG>& sh, const typename X::E* x, int begin, int end, uint32_t from) {
    constexpr int V = X::V, NV = SC_PER_THREAD / V, CHUNK = WG * SC_PER_THREAD;
    const int t = threadIdx.x;
    __syncthreads();
    if (t == 0) sh.n_seg = sh.n_cand = 0;
    __syncthreads();
    const int chunks = (end - begin + CHUNK - 1) / CHUNK;
    for (int c = 0; c < chunks; ++c)
        if (sh.seg_max[c][t] >= from) {
            const int to = atomicAdd(&sh.n_seg, 1);
            if (to < SC_SEGS) sh.segs[to] = (uint16_t)(c * WG + t);
        }
    __syncthreads();
    if (sh.n_seg > SC_SEGS) return false;
    for (int i = t; i < sh.n_seg * NV; i += WG) {
        const int seg = sh.segs[i / NV];
        const int at = begin + (seg / WG) * CHUNK + ((i % NV) * WG + seg % WG) * V;
        if (at >= end) continue;
        float f[V];
        sc_read<X>(x, at, end, f);
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (sc_order(f[e]) >= from && at + e < end) {
                const int to = atomicAdd(&sh.n_cand, 1);
                if (to < SC_CAND) sh.cand[to] = sc_key(f[e], at + e);
            }
    }
    __syncthreads();
    return sh.n_cand <= SC_CAND;
}

// The `top` largest of columns begin .. end - 1 as keys, put(k, key) called once for each k, with 0 where there
// are no more columns.  lane_max: the largest of this thread's columns.  The segments' maxima are in sh.
template <typename X, int WG, typename Put>
__device__ void sc_top_block(TopShared<WG>& sh, const typename X::E* x, int begin, int end, int top, float lane_max, Put put) {
    constexpr int V = X::V;
    const int t = threadIdx.x;
    // The columns in 256 parts, or 64: the top-th largest of the parts' maxima is a bound.  Of 64 it is quicker found, and
    // some top + top^2 / 128 scores reach it; at top = 64 it would be the least of them all.
    // (A workgroup of 64 has 64, and is not given more than 32 alternatives to find.)
    const bool fine = WG > 64 && top > 32;
    const int part = fine ? WG / 256 : WG / 64;  // threads to a part
    lane_max = sc_lanes(lane_max, part, FMaxOp());
    if ((t & (part - 1)) == 0) sh.part_max[t / part] = sc_order(lane_max);
    __syncthreads();
    if (t < 64) {
        uint32_t o[4], tau;
        o[0] = sh.part_max[t];
        if (fine) {
#pragma unroll
            for (int i = 1; i < 4; ++i) o[i] = sh.part_max[t + 64 * i];
            tau = sc_kth<4>(o, top);
        } else {
            tau = sc_kth<1>(o, top);
        }
        if (t == 0) sh.tau = tau;
    }
    __syncthreads();
    const uint32_t tau = sh.tau;
    bool fits = sc_collect<X, WG>(sh, x, begin, end, tau);
    if (!fits && sc_collect<X, WG>(sh, x, begin, end, tau + 1)) {
        // too many scores equal to tau (a masked row, a constant one): what is larger has been collected, and the
        // first of the equal ones make up the number, found from the front
        fits = true;
        for (int at0 = begin; at0 < end && sh.n_cand < top; at0 += WG * V) {
            const int at = at0 + t * V;
            float f[V];
            sc_read<X>(x, at, end, f);
            int mine = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) mine += at + e < end && sc_order(f[e]) == tau;
            int before = mine;  // an inclusive scan over the wavefront
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(before, d);
                if ((t & 63) >= d) before += o;
            }
            if ((t & 63) == 63) sh.scanned[t >> 6] = before;
            const int have = sh.n_cand;
            __syncthreads();
            int total = 0;
            before += have - mine;
#pragma unroll
            for (int i = 0; i < WG / 64; ++i) {
                if (i < t >> 6) before += sh.scanned[i];
                total += sh.scanned[i];
            }
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (at + e < end && sc_order(f[e]) == tau) {
                    if (before < top) sh.cand[before] = sc_key(f[e], at + e);
                    ++before;
                }
            if (t == 0) sh.n_cand = have + total < top ? have + total : top;
            __syncthreads();
        }
    }
    if (fits) {
        const int n = sh.n_cand;
        for (int i = t; i < n; i += WG) {
            const uint64_t key = sh.cand[i];
            const int rank = sc_rank(sh.cand, n, key);
            if (rank < top) put(rank, key);
        }
        if (t >= n && t < top) put(t, 0);
    } else {
        uint64_t prev = ~0ull;  // many large scores in few lanes: one after the other
        for (int k = 0; k < top; ++k) {
            uint64_t best = 0;
            for (int at = begin + t * V; at < end; at += WG * V) {
                float f[V];
                sc_read<X>(x, at, end, f);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const uint64_t key = sc_key(f[e], at + e);
                    if (at + e < end && key < prev && key > best) best = key;
                }
            }
            prev = sc_block<WG>(best, MaxOp(), sh.wave_best);
            if (t == 0) put(k, prev);
        }
    }
    __syncthreads();
}

// Thread t's 32 scores of a whole chunk that starts at x.
template <typename X, int WG>
__device__ __forceinline__ void sc_load_chunk(const typename X::E* x, int t, sc_u4* w) {
#pragma unroll
    for (int u = 0; u < SC_PER_THREAD / X::V; ++u) w[u] = sc_load<X>(x + (u * WG + t) * X::V);
}

struct Nothing {};

template <typename X, int WG, bool TOP>
__global__ __launch_bounds__(WG) void k_token_logprobs_block(LogprobArgs a) {
    constexpr int V = X::V, NV = SC_PER_THREAD / V, CHUNK = WG * SC_PER_THREAD, WAVES = WG / 64;
    // few workgroups: nobody else to fill the time between a load and its use (float32: with alternatives six registers too
    // many; without them there is room, which is not taken)
    constexpr bool AHEAD = WG == 1024 && V == 8;
    __shared__ Stat wave_stat[WAVES];
    __shared__ typename std::conditional<TOP, TopShared<WG>, Nothing>::type sh;
    const int t = threadIdx.x;
    for (int64_t b = blockIdx.x; b < a.rows * a.slices; b += gridDim.x) {
        const int64_t r = b / a.slices;
        const int slice = (int)(b - r * a.slices);
        const typename X::E* x = (const typename X::E*)a.x + r * a.stride;
        const int n = sc_width(a.widths, r, a.cols);
        const int begin = slice * a.slice_cols < n ? slice * a.slice_cols : n;
        const int end = n - begin < a.slice_cols ? n : begin + a.slice_cols;
        RowToken tok = {};
        if (a.slices == 1) tok = sc_row_token<X>(a, r, x, n, t);
        Stat st = {-INFINITY, 0, 0};
        sc_u4 w[NV];
        if (AHEAD && begin + CHUNK <= end) sc_load_chunk<X, WG>(x + begin, t, w);
        for (int c = 0, at0 = begin; at0 < end; at0 += CHUNK, ++c) {
            float f[SC_PER_THREAD];
            if (at0 + CHUNK <= end) {
                if (!AHEAD) sc_load_chunk<X, WG>(x + at0, t, w);
#pragma unroll
                for (int u = 0; u < NV; ++u) X::unpack(w[u], f + u * V);
                if (AHEAD && at0 + 2 * CHUNK <= end) sc_load_chunk<X, WG>(x + at0 + CHUNK, t, w);
            } else {
#pragma unroll
                for (int u = 0; u < NV; ++u) sc_read<X>(x, at0 + (u * WG + t) * V, end, f + u * V);
            }
            const float m = sc_max<SC_PER_THREAD>(f, -INFINITY);
            if constexpr (TOP) sh.seg_max[c][t] = sc_order(m);
            sc_carry(st, fmaxf(st.m, m));
            sc_add<SC_PER_THREAD>(st, f);
        }
        const float lane_max = st.m;
        sc_join_block<WG>(st, wave_stat);
        const RowStat q = sc_row_stat(st);
        if (a.slices > 1) {
            if (t == 0) a.part[b] = st;
        } else {
            sc_put_row(a, r, st, q, tok, t);
        }
        if constexpr (TOP) {
            if (a.slices > 1) {
                uint64_t* keys = a.part_keys + b * a.top;
                if (q.bad) {
                    if (t < a.top) keys[t] = 0;
                } else {
                    sc_top_block<X, WG>(sh, x, begin, end, a.top, lane_max, [&](int k, uint64_t key) { keys[k] = key; });
                }
            } else if (q.bad || q.empty) {
                if (t < a.top) sc_put_top(a, r, t, q.bad ? 0 : sc_key(-INFINITY, t), q);
            } else {
                sc_top_block<X, WG>(sh, x, begin, end, a.top, lane_max, [&](int k, uint64_t key) { sc_put_top(a, r, k, key, q); });
            }
        }
        __syncthreads();  // wave_stat is written again
    }
}

// The slices of a row: their statistics by the rule above, their alternatives (each slice's in order) merged.  If the j-th keys
// of q slices reach a bound, at least q j keys do; the smallest j with q j >= top (q of the slices) makes the bound a close one:
// of 256 slices with 64 keys each some 75 reach the 64th largest of the first keys.  At most 256 slices (sc_cut).
#define SC_AHEAD 4

template <typename X>
__global__ __launch_bounds__(SC_WG) void k_token_logprobs_join(LogprobArgs a) {
    __shared__ uint64_t cand[SC_CAND], wave_key[SC_WAVES];
    __shared__ uint64_t heads[SC_WG];
    __shared__ uint32_t from;
    __shared__ Stat wave_stat[SC_WAVES];
    __shared__ int n_cand;
    const int t = threadIdx.x;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const typename X::E* x = (const typename X::E*)a.x + r * a.stride;
        const int n = sc_width(a.widths, r, a.cols);
        const RowToken tok = sc_row_token<X>(a, r, x, n, t);
        // everything the row needs is asked for at once: it comes from other XCDs' workgroups, by way of the memory
        const uint64_t* keys = a.part_keys + r * a.slices * a.top;
        const int total = a.slices * a.top;
        const int j = a.top ? (a.top + a.slices - 1) / a.slices : 1, reach = (a.top + j - 1) / j;
        uint64_t ahead[SC_AHEAD];
#pragma unroll
        for (int i = 0; i < SC_AHEAD; ++i) ahead[i] = t + i * SC_WG < total ? keys[t + i * SC_WG] : 0;
        uint64_t head = 0;  // two slices without a j-th key differ by the thread
        if (a.top && t < a.slices) heads[t] = head = (keys[t * a.top + j - 1] >> 32 << 32) | t;
        Stat st = {-INFINITY, 0, 0};
        for (int i = t; i < a.slices; i += SC_WG) {
            Stat o = a.part[r * a.slices + i];
            const float m = fmaxf(st.m, o.m);
            sc_carry(st, m);
            sc_carry(o, m);
            st.s += o.s;
            st.w += o.w;
        }
        if (t == 0) n_cand = 0;
        sc_join_block<SC_WG>(st, wave_stat);
        const RowStat q = sc_row_stat(st);
        sc_put_row(a, r, st, q, tok, t);
        if (a.top && (q.bad || q.empty)) {
            if (t < a.top) sc_put_top(a, r, t, q.bad ? 0 : sc_key(-INFINITY, t), q);
        } else if (a.top) {
            if (t < a.slices && sc_rank(heads, a.slices, head) == reach - 1) from = (uint32_t)(head >> 32);
            __syncthreads();
            const auto collect = [&](uint64_t key) {
                if (key && (uint32_t)(key >> 32) >= from) {
                    const int to = atomicAdd(&n_cand, 1);
                    if (to < SC_CAND) cand[to] = key;
                }
            };
#pragma unroll
            for (int i = 0; i < SC_AHEAD; ++i) collect(ahead[i]);
            for (int i = t + SC_AHEAD * SC_WG; i < total; i += SC_WG) collect(keys[i]);
            __syncthreads();
            const int have = n_cand;
            if (have <= SC_CAND) {
                for (int i = t; i < have; i += SC_WG) {
                    const uint64_t key = cand[i];
                    const int rank = sc_rank(cand, have, key);
                    if (rank < a.top) sc_put_top(a, r, rank, key, q);
                }
                if (t >= have && t < a.top) sc_put_top(a, r, t, 0, q);
            } else {
                // too many equal scores: the largest of the slices' next keys, one after the other
                uint64_t next = t < a.slices ? keys[t * a.top] : 0;
                for (int k = 0, at = 0; k < a.top; ++k) {
                    const uint64_t best = sc_block<SC_WG>(next, MaxOp(), wave_key);
                    if (t == 0) sc_put_top(a, r, k, best, q);
                    if (next == best && best) next = ++at < a.top ? keys[t * a.top + at] : 0;
                }
            }
        }
        __syncthreads();
    }
}

struct LogprobGradArgs {
    const void* x;
    int64_t rows, stride;
    int cols;
    const int32_t* widths;
    const float* stats;
    const int64_t* tokens;
    int n_tok;
    const float *g_logp, *g_entropy;
    void* out;
    int64_t out_stride;
};

// dx_j = -p_j (sum g + gH (log p_j + H)) + the tokens' own g, with t = log2 p_j = (x_j - m) log2 e - log2 S:
// one read and one write of the row, some eleven instructions a score, bound by the memory; short 16-bit rows by the number of
// wavefronts, one to a row (bfloat16, 65536 x 40 24.5 us, x 128 25.8, x 1000 61, x 2000 120; floors 2, 6.7, 52, 104).  A lane holds
// a token (n_tok <= 64), so that the row's scores are compared with none: the one lane that holds a token's column adds
// its g before the value is rounded, the tokens in their order.
struct GradRow {
    float base, log2_sum, c0, c1;  // dx = -p (c0 + c1 t)
    bool empty;
    int tok;      // this lane's token, -1: none, or not in the row
    float g;
};

__device__ __forceinline__ GradRow sc_grad_row(const LogprobGradArgs& a, int64_t r, int n, int lane) {
    GradRow q;
    const float m = a.stats[3 * r], log_sum = a.stats[3 * r + 1], h = a.stats[3 * r + 2];
    const float ge = a.g_entropy ? a.g_entropy[r] : 0.0f;
    q.empty = m == -INFINITY && log_sum == 0;
    q.base = m;
    q.log2_sum = log_sum * SC_LOG2E;
    q.tok = -1;
    q.g = 0;
    if (lane < a.n_tok) {
        const int64_t tok = a.tokens[r * a.n_tok + lane];
        if (tok >= 0) q.g = a.g_logp[r * a.n_tok + lane];
        if (tok >= 0 && tok < n) q.tok = (int)tok;
    }
    q.c0 = fmaf(ge, h, a.n_tok > 1 ? sc_wave(q.g, SumOp()) : __shfl(q.g, 0));
    q.c1 = ge * SC_LN2;
    return q;
}

// The gradient of NV vectors of V columns, vector u at at0 + u * step, from the scores f, in their place.
template <typename X, int NV>
__device__ __forceinline__ void sc_grad_values(const GradRow& q, float* f, int at0, int step, int begin, int end) {
    constexpr int V = X::V;
#pragma unroll
    for (int i = 0; i < NV * V; ++i) {
        const float t = fmaf(f[i] - q.base, SC_LOG2E, -q.log2_sum);
        f[i] = -__builtin_amdgcn_exp2f(t) * fmaf(q.c1, sc_floor_t(t), q.c0);
    }
    // the tokens whose column one of this wavefront's lanes holds: piece (tok - begin) / V goes to lane (..) mod 64, of
    // wavefront (..) / 64 mod the number of them (step / (64 V))
    const int piece = (q.tok - begin) / V, wave = (at0 - begin) / (64 * V);
    uint64_t mine = __ballot(q.tok >= begin && q.tok < end && (piece / 64) % (step / (64 * V)) == wave);
    for (; mine; mine &= mine - 1) {
        const int k = __ffsll((unsigned long long)mine) - 1;
        const int tok = __builtin_amdgcn_readlane(q.tok, k);
        const float g = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(q.g), k));
#pragma unroll
        for (int i = 0; i < NV * V; ++i)
            if (tok == at0 + (i / V) * step + i % V) f[i] += g;
    }
}

template <typename X>
__device__ __forceinline__ void sc_grad_store(typename X::E* out, int at, int n, int cols, bool empty, float* f) {
    constexpr int V = X::V;
    if (empty || at + V > n)
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = empty || at + e >= n ? 0.0f : f[e];
    if (at + V <= cols) {
        sc_store<X>(out + at, X::pack(f));
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (at + e < cols) X::put(out + at + e, f[e]);
    }
}

template <typename X, int NV>
__global__ __launch_bounds__(SC_WG) void k_token_logprobs_grad_wave(LogprobGradArgs a) {
    constexpr int V = X::V;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t r = (int64_t)blockIdx.x * SC_WAVES + wave; r < a.rows; r += (int64_t)gridDim.x * SC_WAVES) {
        const typename X::E* x = (const typename X::E*)a.x + r * a.stride;
        typename X::E* out = (typename X::E*)a.out + r * a.out_stride;
        const int n = sc_width(a.widths, r, a.cols);
        float f[NV * V];
#pragma unroll
        for (int u = 0; u < NV; ++u) sc_read<X>(x, (u * 64 + lane) * V, n, f + u * V);
        const GradRow q = sc_grad_row(a, r, n, lane);
        sc_grad_values<X, NV>(q, f, lane * V, 64 * V, 0, a.cols);
#pragma unroll
        for (int u = 0; u < NV; ++u) sc_grad_store<X>(out, (u * 64 + lane) * V, n, a.cols, q.empty, f + u * V);
    }
}

#define SC_CHUNK (SC_WG * SC_PER_THREAD)

template <typename X>
__global__ __launch_bounds__(SC_WG) void k_token_logprobs_grad_block(LogprobGradArgs a) {
    constexpr int V = X::V, NV = SC_PER_THREAD / V;
    const int t = threadIdx.x;
    const int chunks = (a.cols + SC_CHUNK - 1) / SC_CHUNK;
    for (int64_t b = blockIdx.x; b < a.rows * chunks; b += gridDim.x) {
        const int64_t r = b / chunks;
        const int at0 = (int)(b - r * chunks) * SC_CHUNK;
        const typename X::E* x = (const typename X::E*)a.x + r * a.stride;
        typename X::E* out = (typename X::E*)a.out + r * a.out_stride;
        const int n = sc_width(a.widths, r, a.cols);
        const bool whole = at0 + SC_CHUNK <= n;
        float f[SC_PER_THREAD];
        if (whole) {
            sc_u4 w[NV];
#pragma unroll
            for (int u = 0; u < NV; ++u) w[u] = sc_load_once<X>(x + at0 + (u * SC_WG + t) * V);
#pragma unroll
            for (int u = 0; u < NV; ++u) X::unpack(w[u], f + u * V);
        } else {
#pragma unroll
            for (int u = 0; u < NV; ++u) sc_read<X>(x, at0 + (u * SC_WG + t) * V, n, f + u * V);
        }
        const GradRow q = sc_grad_row(a, r, n, t & 63);
        sc_grad_values<X, NV>(q, f, at0 + t * V, SC_WG * V, at0, at0 + SC_CHUNK);
        if (whole && !q.empty) {
#pragma unroll
            for (int u = 0; u < NV; ++u) sc_store_once<X>(out + at0 + (u * SC_WG + t) * V, X::pack(f + u * V));
        } else {
#pragma unroll
            for (int u = 0; u < NV; ++u) sc_grad_store<X>(out, at0 + (u * SC_WG + t) * V, n, a.cols, q.empty, f + u * V);
        }
    }
}

// ---- routing -------------------------------------------------------------------------------
//
// The order of the experts is that of float64 arithmetic, so that it does not depend on how a kernel forms its sums.
// Without a bias it is the order of the logits, which float32 holds exactly.  With one, the scores p + bias are formed
// in float32 with a known error; a row in which that error could decide is done again in float64 (k_route calls
// sc_route_row for it, a wavefront to the row).  The same goes for the groups.
//
// A row belongs to L lanes (a power of two, whole groups to whole lanes), a lane holds EPL consecutive experts of one
// group, a wavefront 64 / L rows.  A score and its place are one number, the place in mantissa bits that the score does not
// use, so that one v_max orders both and no two are equal: bfloat16 and float16 logits leave 13 bits of 32, all else goes
// into a float64 (whose v_max issues at the same rate).  A lane sorts its experts KP at a time by
// a bitonic network, keeps the best KP, and the lanes merge theirs in log2 L exchanges.
//
// 65536 x 128 bfloat16 to eight: 11.5 us, 3.4 of them the launch and the first rows' latency, the rest 0.11 to 0.13 us for 1024
// rows, of which issue (630 instructions for eight rows) takes 0.08 and the bytes 0.06; the last 1024 of 8192 wavefronts wait
// for a place (65 registers leave seven to a SIMD): 0.6 us.  By p + bias and in groups issue is 36 of 57 us at 65536 x 256 (1697
// instructions for four rows), and three wavefronts a SIMD (161 registers) cover the latency badly.  Groups with the same sum
// go to float64, 5 us of a wavefront for a row: 65536 x 256 equal logits 277 us, a tenth of the rows equal 91.

struct RouteArgs {
    const void* x;
    int dtype;
    int64_t rows, stride;
    int experts, top, sigmoid;
    const float* bias;
    int groups, per_group, top_groups, top2, renorm;
    float scale;
    float* weights;
    int32_t* index;
    int lanes, group_lanes;  // to a row, to a group
};

__device__ __forceinline__ float sc_logit(const void* x, int dtype, int64_t at) {
    if (dtype == PD_F32) return F32::get((const float*)x + at);
    if (dtype == PD_BF16) return BF16::get((const uint16_t*)x + at);
    return F16::get((const _Float16*)x + at);
}

// p of a chosen expert relative to the others': lane i < top of a row's lanes holds the i-th one's logit (-inf: none).
// Sums of tiny sigmoids are formed relative to the largest, so that they do not all come to 0.
__device__ __forceinline__ float sc_chosen_share(float xi, bool have, int sigmoid, int renorm, int lanes) {
    float w;
    if (sigmoid) {
        float shift = 0;
        if (renorm) {
            const float big = sc_lanes(have ? xi : -INFINITY, lanes, FMaxOp());
            if (big < 0 && big > -INFINITY) shift = big;
        }
        w = xi < 0 ? expf(xi - shift) / (1 + expf(xi)) : 1 / (1 + expf(-xi));
    } else {
        const float big = sc_lanes(have ? xi : -INFINITY, lanes, FMaxOp());
        w = big == -INFINITY ? 0.0f : expf(xi - big);
    }
    if (!have) w = 0;
    if (renorm) {
        const float sum = sc_lanes(w, lanes, SumOp());
        w = sum == 0 ? 0.0f : w / sum;
    }
    return w;
}

// Lane i < top of the `lanes` lanes of a row writes the i-th expert and its weight, from its logit; m and total: the
// softmax's, where it is not renormalised.  idx < 0: the row has no order.
__device__ __forceinline__ void sc_route_put(const RouteArgs& a, int64_t r, int i, int lanes, bool have, int idx, float xi,
                                             float m, float total) {
    have &= i < a.top;
    float w;
    if (a.sigmoid || a.renorm)
        w = sc_chosen_share(have ? xi : -INFINITY, have, a.sigmoid, a.renorm, lanes);
    else
        w = total == 0 ? 0.0f : expf(xi - m) / total;
    if (have) {
        a.weights[r * a.top + i] = idx < 0 ? NAN : w * a.scale;
        a.index[r * a.top + i] = idx;
    }
}

// A row by one wavefront in float64, where p + bias or the groups' sums of p order the experts (ROUTE_CLOSE); by: PD_MAX_EXPERTS
// values of the wavefront's own.
__device__ __forceinline__ void sc_route_row(const RouteArgs& a, int64_t r, int lane, double* by) {
    const int E = a.experts;
    const int64_t row = r * a.stride;
    // (a lane's experts are lane, lane + 64, ..: nobody else's until the groups look at them; four loads in flight)
#pragma unroll 4
    for (int j = lane; j < E; j += 64) by[j] = sc_logit(a.x, a.dtype, row + j);
    double m = 0, total = 0;
    if (!a.sigmoid) {
        double big = -INFINITY;
#pragma nounroll
        for (int j = lane; j < E; j += 64) big = fmax(big, by[j]);
        big = sc_wave(big, DMaxOp());
        if (big > -INFINITY) {
            m = big;
#pragma nounroll
            for (int j = lane; j < E; j += 64) total += exp(by[j] - m);
        }
        total = sc_wave(total, SumOp());
    }
#pragma nounroll
        for (int j = lane; j < E; j += 64)
            by[j] = a.sigmoid ? 1 / (1 + exp(-by[j])) : total > 0 ? exp(by[j] - m) / total : 0.0;
    if (a.bias)
#pragma unroll 4
        for (int j = lane; j < E; j += 64) by[j] += a.bias[j];
#pragma nounroll
    for (int j = lane; j < E; j += 64) by[j] = by[j] >= -1e300 ? by[j] : -1e300;  // -inf and NaN behind all others
    pd_wave_sync();
    uint64_t kept = ~0ull;
    if (a.groups > 1) {
        double mine = -INFINITY;  // lane g: group g's
        if (lane < a.groups) {
            double b1 = -INFINITY, b2 = -INFINITY;
            const double* of = by + lane * a.per_group;
#pragma unroll 8
            for (int j = 0; j < a.per_group; ++j) {
                const double v = of[j];
                b2 = fmax(b2, fmin(b1, v));
                b1 = fmax(b1, v);
            }
            mine = b1;
            // (-1e300 stands for -inf, which a sum of finite ones never is; one of +inf and -inf counts as +inf)
            if (a.top2 && a.per_group > 1) mine = b2 > -1e300 || b1 == INFINITY ? b1 + b2 : -INFINITY;
        }
        int rank = 0;
#pragma nounroll
        for (int g = 0; g < a.groups; ++g) {
            const double o = __shfl(mine, g);
            rank += o > mine || (o == mine && g < lane);
        }
        kept = __ballot(lane < a.groups && rank < a.top_groups);
    }
#pragma nounroll
    for (int j = lane; j < E; j += 64) {
        if (!a.bias) by[j] = fmax((double)sc_logit(a.x, a.dtype, row + j), -1e300);  // p counted for the groups only
        if (!(kept >> (j / a.per_group) & 1)) by[j] = -INFINITY;
    }
    int chosen = -1;
#pragma nounroll
    for (int k = 0; k < a.top; ++k) {
        double best = -INFINITY;
        int at = E;
#pragma unroll 4
        for (int j = lane; j < E; j += 64) {
            const double v = by[j];
            at = v > best ? j : at;
            best = fmax(best, v);
        }
        const double top = sc_wave(best, DMaxOp());
        at = (int)sc_wave((uint32_t)(best == top ? at : E), MinOp());
        if ((at & 63) == lane && at < E) by[at] = -INFINITY;
        if (lane == k) chosen = at;
    }
    const float xi = lane < a.top ? sc_logit(a.x, a.dtype, row + chosen) : -INFINITY;
    sc_route_put(a, r, lane, 64, true, chosen, xi, (float)m, (float)total);
    pd_wave_sync();
}

// ---- sorting networks: descending, indexes known at compile time ------------------------------------

__device__ __forceinline__ double sc_hi(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ double sc_lo(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ uint32_t sc_hi(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t sc_lo(uint32_t a, uint32_t b) { return a < b ? a : b; }

template <typename K>
__device__ __forceinline__ void sc_exchange(K& a, K& b) {  // the larger first
    const K hi = sc_hi(a, b), lo = sc_lo(a, b);
    a = hi;
    b = lo;
}
// A bitonic sequence into descending order.
template <int N, typename K>
__device__ __forceinline__ void sc_bitonic(K* v) {
    if constexpr (N > 1) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) sc_exchange(v[i], v[i + N / 2]);
        sc_bitonic<N / 2>(v);
        sc_bitonic<N / 2>(v + N / 2);
    }
}
template <int N, typename K>
__device__ __forceinline__ void sc_sort(K* v) {
    if constexpr (N > 1) {
        sc_sort<N / 2>(v);
        sc_sort<N / 2>(v + N / 2);
        // two descending halves: the first step compares ends with ends, what is left is bitonic
#pragma unroll
        for (int i = 0; i < N / 2; ++i) sc_exchange(v[i], v[N - 1 - i]);
        sc_bitonic<N / 2>(v);
        sc_bitonic<N / 2>(v + N / 2);
    }
}
// The N largest of two descending lists, descending, into a.
template <int N, typename K>
__device__ __forceinline__ void sc_merge(K* a, const K* b) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = sc_hi(a[i], b[N - 1 - i]);
    sc_bitonic<N>(a);
}
template <int N, int STEP, typename K>
__device__ __forceinline__ void sc_merge_across(K* a) {
    K p[N], q[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sc_pair<STEP>(a[i], p[i], q[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = p[i];
    sc_merge<N>(a, q);
}

// Score and place as one number.  Of two equal scores the one of the lower place is the larger: where a float64 is negative
// the one with the smaller magnitude.  -inf (float64: and NaN) comes behind every finite score, NONE behind that.
#define SC_PLACES (PD_MAX_EXPERTS - 1)
struct Key32 {  // of a bfloat16 or float16 value: the order of its float32, whose lowest 13 bits are the same for all
    typedef uint32_t K;
    static constexpr K NONE = 0;
    static __device__ __forceinline__ K make(float s, int place) { return (sc_order(s) & ~(uint32_t)SC_PLACES) | (SC_PLACES - place); }
    static __device__ __forceinline__ int place(K key) { return SC_PLACES - (int)(key & SC_PLACES); }
    static __device__ __forceinline__ float score(K key) {
        return sc_unorder(key >> 31 ? key & ~(uint32_t)SC_PLACES : key | SC_PLACES);
    }
};
struct Key64 {
    typedef double K;
    static constexpr K NONE = -INFINITY;
    static __device__ __forceinline__ K make(float s, int place) {
        const double d = fmin(fmax((double)(s + 0.0f), -0x1p1000), 0x1p1000);
        const uint64_t u = __double_as_longlong(d);
        return __longlong_as_double(u | ((uint32_t)place ^ (~(uint32_t)((int64_t)u >> 63) & SC_PLACES)));
    }
    static __device__ __forceinline__ int place(K key) {
        const uint64_t u = __double_as_longlong(key);
        return (int)(((uint32_t)u ^ ~(uint32_t)((int64_t)u >> 63)) & SC_PLACES);
    }
    static __device__ __forceinline__ float score(K key) {  // +-2^1000 rounds to +-inf
        return (float)__longlong_as_double(__double_as_longlong(key) & ~(uint64_t)SC_PLACES);
    }
};

// `have` consecutive logits from element `at` on, -inf behind them.
template <typename X, int EPL>
__device__ __forceinline__ void sc_route_read(const void* base, int64_t at, int have, bool full, float* f) {
    const typename X::E* x = (const typename X::E*)base + at;
    if (full) {
        sc_u4 w[EPL / X::V];
#pragma unroll
        for (int u = 0; u < EPL / X::V; ++u) w[u] = sc_load<X>(x + u * X::V);
#pragma unroll
        for (int u = 0; u < EPL / X::V; ++u) X::unpack(w[u], f + u * X::V);
    } else {
#pragma unroll
        for (int u = 0; u < EPL / X::V; ++u) sc_read<X>(x, u * X::V, have, f + u * X::V);
    }
}

// PLAIN16, PLAIN32: the order is that of the logits (no bias, no sums of two p for the groups), 16-bit or float32 ones.
// CLOSE: p + bias, or groups by sums of p, take part in it, and close calls are taken to float64.
enum { ROUTE_PLAIN16, ROUTE_PLAIN32, ROUTE_CLOSE };

template <int EPL, int KP, int MODE>
__global__ __launch_bounds__(SC_WG) void k_route(RouteArgs a) {
    typedef typename std::conditional<MODE == ROUTE_PLAIN16, Key32, Key64>::type Key;
    typedef typename Key::K K;
    constexpr bool CLOSE = MODE == ROUTE_CLOSE;
    __shared__ double by[CLOSE ? SC_WAVES : 1][CLOSE ? PD_MAX_EXPERTS : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int L = a.lanes, l = lane & (L - 1), first = lane & ~(L - 1), per_wave = 64 / L;
    const uint64_t row_lanes = (L == 64 ? ~0ull : (1ull << L) - 1) << first;
    const int g = l / a.group_lanes, in_group = (l & (a.group_lanes - 1)) * EPL;
    const int place = g * a.per_group + in_group;
    const int have = g < a.groups ? pd_clampi(a.per_group - in_group, 0, EPL) : 0;
    const bool full = __ballot(have == EPL) == ~0ull;
    const bool biased = CLOSE && a.bias;
    const int64_t tiles = (a.rows + per_wave - 1) / per_wave;
    for (int64_t tile = (int64_t)blockIdx.x * SC_WAVES + wave; tile < tiles; tile += (int64_t)gridDim.x * SC_WAVES) {
        const int64_t r = tile * per_wave + lane / L, row = r < a.rows ? r : a.rows - 1;
        const bool on = r < a.rows;
        float x[EPL], s[EPL];
        if (MODE == ROUTE_PLAIN32 || (CLOSE && a.dtype == PD_F32))
            sc_route_read<F32, EPL>(a.x, row * a.stride + place, have, full, x);
        else if (a.dtype == PD_BF16)
            sc_route_read<BF16, EPL>(a.x, row * a.stride + place, have, full, x);
        else
            sc_route_read<F16, EPL>(a.x, row * a.stride + place, have, full, x);
        // rows without an order: NaN anywhere, +inf under a softmax
        bool bad = false;
        const int none = a.sigmoid ? 0x003 : 0x203;
#pragma unroll
        for (int j = 0; j < EPL; ++j) bad |= __builtin_amdgcn_classf(x[j], none);
        bad = (__ballot(bad) & row_lanes) != 0;

        float m = 0, total = 0, tol = 0;
        if (!a.sigmoid && (CLOSE || !a.renorm)) {
            m = sc_lanes(sc_max<EPL>(x, -INFINITY), L, FMaxOp());
            m = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                s[j] = __builtin_amdgcn_exp2f((x[j] - m) * SC_LOG2E);
                total += s[j];
            }
            total = sc_lanes(total, L, SumOp());
        }
        bool again = false, kept = true;
        if constexpr (CLOSE) {
            if (a.sigmoid) {
#pragma unroll
                for (int j = 0; j < EPL; ++j) s[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-SC_LOG2E * x[j]));
                // p is off by p (1 - p) times the exponent's and the exponential's error and a step each for the sum and
                // the reciprocal, together below 4 u (u = 2^-24); the difference of two by twice that
                tol = 0x1p-21f;
            } else {
                const float inv = total == 0 ? 0.0f : 1.0f / total;
#pragma unroll
                for (int j = 0; j < EPL; ++j) s[j] *= inv;
                // the largest p is 1 / total, and every p is off by at most (EPL + 27) u of it: 3 u for its exponent (1.6 |t| 2^t)
                // and exponential, EPL + 5 for the sum's steps and 17 for its terms (1.6 times the mean |t|, at most 10, and
                // 2), 2 for the division and the product; the difference of two by twice that
                tol = 0x1p-17f * inv;
            }
            if (biased) {  // (from the L1: the same for every row)
                float b[EPL];
                sc_route_read<F32, EPL>(a.bias, place, have, full, b);
#pragma unroll
                for (int j = 0; j < EPL; ++j) s[j] = fmaxf(s[j] + b[j], -INFINITY);  // a bias of NaN counts as -inf
            }
        }
        if (a.groups > 1) {
            float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                const float v = j < have ? (CLOSE ? s[j] : x[j]) : -INFINITY;
                b2 = fmaxf(b2, fminf(b1, v));
                b1 = fmaxf(b1, v);
            }
#define SC_TOP2_STEP(d)                                 \
    if (a.group_lanes > d) {                            \
        float p1, q1, p2, q2;                           \
        sc_pair<d>(b1, p1, q1);                         \
        sc_pair<d>(b2, p2, q2);                         \
        b2 = fmaxf(fminf(p1, q1), fmaxf(p2, q2));       \
        b1 = fmaxf(p1, q1);                             \
    }
            SC_TOP2_STEP(1) SC_TOP2_STEP(2) SC_TOP2_STEP(4) SC_TOP2_STEP(8) SC_TOP2_STEP(16) SC_TOP2_STEP(32)
#undef SC_TOP2_STEP
            const bool two = a.top2 && a.per_group > 1;
            const float mine = two ? b1 + b2 : b1;
            if constexpr (CLOSE) {
                // What the float64 score lies between.  Two p are off by tol together; b1 and b2 are off by a rounding of the
                // sum with the bias each, whatever is left of them in b1 + b2, that by one, and lo and hi by one: 3 u
                // (|b1| + |b2|), and 4 u are taken.  A bound past float32 leaves it open.  A term of -inf is that exactly.
                const float off = tol + 0x1p-22f * (fabsf(b1) + (two ? fabsf(b2) : 0.0f));
                const bool out = (two ? b2 : b1) == -INFINITY && b1 < INFINITY;
                const float lo = !out && off < INFINITY ? mine - off : -INFINITY, hi = off < INFINITY ? mine + off : out ? -INFINITY : INFINITY;
                int above = 0, maybe = 0;
                for (int k = 0; k < a.groups; ++k) {
                    const float o_lo = __shfl(lo, first + k * a.group_lanes), o_hi = __shfl(hi, first + k * a.group_lanes);
                    above += o_lo > hi;
                    maybe += k != g && !(o_hi < lo);
                }
                kept = maybe < a.top_groups;
                again = g < a.groups && !kept && above < a.top_groups;
            } else {
                int rank = 0;
                for (int k = 0; k < a.groups; ++k) {
                    const float o = __shfl(mine, first + k * a.group_lanes);
                    rank += o > mine || (o == mine && k < g);
                }
                kept = rank < a.top_groups;
            }
        }
        K best[KP];
        {
            constexpr int B = KP < EPL ? KP : EPL;
#pragma unroll
            for (int b = 0; b < EPL; b += B) {
                K v[B];
#pragma unroll
                for (int j = 0; j < B; ++j) v[j] = Key::make(CLOSE && biased ? s[b + j] : x[b + j], place + b + j);
                if (!full) {
#pragma unroll
                    for (int j = 0; j < B; ++j) v[j] = b + j < have ? v[j] : Key::NONE;
                }
                sc_sort<B>(v);
                if (b == 0) {
#pragma unroll
                    for (int j = 0; j < KP; ++j) best[j] = j < B ? v[j < B ? j : 0] : Key::NONE;
                } else if constexpr (B == KP) {
                    sc_merge<KP>(best, v);
                }
            }
        }
        if (a.groups > 1) {
#pragma unroll
            for (int j = 0; j < KP; ++j) best[j] = kept ? best[j] : Key::NONE;
        }
        if (L > 1) sc_merge_across<KP, 1>(best);
        if (L > 2) sc_merge_across<KP, 2>(best);
        if (L > 4) sc_merge_across<KP, 4>(best);
        if (L > 8) sc_merge_across<KP, 8>(best);
        if (L > 16) sc_merge_across<KP, 16>(best);
        if (L > 32) sc_merge_across<KP, 32>(best);

        K mine = best[0];
#pragma unroll
        for (int k = 1; k < KP; ++k) mine = l == k ? best[k] : mine;
        int idx = bad ? -1 : Key::place(mine);
        if constexpr (!CLOSE) {
            sc_route_put(a, r, l, L, on, idx, Key::score(mine), m, total);
        } else {
            if (biased) {
                bool redo = false;  // the list's order, or its end, is open
                // Two neighbours in the list that are too close: in order if they are equal by logit and bias.
                K last = best[0];
                uint32_t close = 0;
#pragma unroll
                for (int k = 0; k + 1 < KP; ++k) {
                    if (k + 1 < a.top && !(best[k] - best[k + 1] > tol + 0x1p-22 * fabs(best[k]))) close |= 1u << k;
                    last = k + 1 == a.top - 1 ? best[k + 1] : last;
                }
                if (!on || bad) close = 0;
                while (__any(close != 0)) {  // lane k of the row holds the k-th place
                    const int k = close ? __ffs((int)close) - 1 : 0, p0 = __shfl(idx, first + k), p1 = __shfl(idx, first + k + 1);
                    if (close)
                        redo |= sc_logit(a.x, a.dtype, row * a.stride + p0) != sc_logit(a.x, a.dtype, row * a.stride + p1) ||
                                 a.bias[p0] != a.bias[p1];
                    close &= close - 1;
                }
                // An expert too close to the last one chosen, on either side: the choice stands if they are equal.
                const float edge = (float)last, off = tol + 0x1p-22f * fabsf(edge);
                const int pl = Key::place(last);
                uint32_t near = 0;
#pragma unroll
                for (int j = EPL - 1; j >= 0; --j) near = near + near + !(fabsf(s[j] - edge) > off);
                if (pl >= place && pl < place + EPL) near &= ~(1u << (pl - place));
                if (on && !bad && near && kept) {
                    const float xl = sc_logit(a.x, a.dtype, row * a.stride + pl), bl = a.bias[pl];
                    for (; near; near &= near - 1) {
                        const int j = __ffs((int)near) - 1;
                        if (j < have)
                            redo |= sc_logit(a.x, a.dtype, row * a.stride + place + j) != xl || a.bias[place + j] != bl;
                    }
                }
                redo = (__ballot(redo) & row_lanes) != 0;
                again |= redo && !a.sigmoid;
                if (a.sigmoid && __any(redo)) {
                    // The experts that can be among the first `top` (not below the last one by more than the error): their
                    // scores in float64, and their ranks among themselves.
                    struct Cand {
                        double by;
                        int place;
                    };
                    Cand* cand = (Cand*)by[wave] + first / L * (2 * L);  // 64 / L rows of 2 L: 2 KB of the 8
                    uint32_t take = 0;
#pragma unroll
                    for (int j = EPL - 1; j >= 0; --j) take = take + take + (s[j] >= edge - off);
                    take = redo && kept ? take & (uint32_t)((1ull << have) - 1) : 0;
                    const int count = sc_lanes(__popc(take), L, SumOp());
                    const bool mend = redo && count <= 2 * L && fabsf(edge) < INFINITY;
                    again |= redo && !mend;
                    int to = __popc(take);  // an exclusive scan over the row's lanes
                    for (int d = 1; d < L; d <<= 1) {
                        const int o = __shfl_up(to, d, L);
                        if (l >= d) to += o;
                    }
                    to -= __popc(take);
                    if (mend)
                        for (; take; take &= take - 1) cand[to++].place = place + __ffs((int)take) - 1;
                    pd_wave_sync();
                    if (mend)
                        for (int i = l; i < count; i += L) {
                            const int at = cand[i].place;
                            const double v = 1 / (1 + exp(-(double)sc_logit(a.x, a.dtype, row * a.stride + at))) + (double)a.bias[at];
                            cand[i].by = v >= -1e300 ? v : -1e300;
                        }
                    pd_wave_sync();
                    int* order = (int*)(by[wave] + 2 * 64 * sizeof(Cand) / sizeof(double)) + first;
                    if (mend)
                        for (int i = l; i < count; i += L) {
                            int rank = 0;
                            for (int k = 0; k < count; ++k)
                                rank += cand[k].by > cand[i].by || (cand[k].by == cand[i].by && cand[k].place < cand[i].place);
                            if (rank < L) order[rank] = cand[i].place;
                        }
                    pd_wave_sync();
                    if (mend) idx = l < a.top ? order[l] : -1;
                    pd_wave_sync();  // the next rows go to the same place
                }
            }
            uint64_t todo = __ballot(again && on && !bad);
            const bool put = on && !(todo & row_lanes);
            const float xi = put && l < a.top && idx >= 0 ? sc_logit(a.x, a.dtype, row * a.stride + idx) : -INFINITY;
            sc_route_put(a, r, l, L, put, idx, xi, m, total);
            while (todo) {  // rows whose order float32 does not tell: here, where the sorting's registers are free again
                const int from = (__ffsll((unsigned long long)todo) - 1) & ~(L - 1);
                sc_route_row(a, tile * per_wave + from / L, lane, by[wave]);
                todo &= ~((L == 64 ? ~0ull : (1ull << L) - 1) << from);
            }
        }
    }
}

struct RouteGradArgs {
    const void* x;
    int64_t rows, stride;
    int experts, top, sigmoid, renorm;
    float scale;
    const int32_t* index;
    const float* g;
    void* out;
    int64_t out_stride;
    int lanes;
};

// With w the chosen experts' p, divided by their sum where they are renormalised:
//   renormalised, or sigmoid:  dx_i = w_i (g_i - sum g w) [renormalised, else w_i g_i], times 1 - p_i for a sigmoid, at the
//                              chosen; 0 elsewhere, and the other logits are not read;
//   softmax as it is:          dx_j = p_j ([j chosen] g_j - sum over the chosen of g_i p_i), which reaches every expert.
// A row's lanes put the chosen experts' values into the row's zeroes in LDS (an expert named twice adds up) and write it out
// in 16-byte pieces.  Bound by the memory and the latency of index -> logit; the softmax as it is (32768 x 160 9 to 10 us, floor
// 4.5) also by its 74 registers, six wavefronts a SIMD: 24576 rows, which all find a place, take 6.8 us, 28672 8.4.
template <typename X, int NV, bool DENSE>
__global__ __launch_bounds__(SC_WG) void k_route_grad(RouteGradArgs a) {
    constexpr int V = X::V;
    __shared__ __align__(16) float rows_acc[SC_WAVES][PD_MAX_EXPERTS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int L = a.lanes, l = lane & (L - 1), per_wave = 64 / L, E = a.experts;
    const int padded = (E + 7) & ~7;  // 64 / L rows of at most 16 L
    float* acc = rows_acc[wave] + lane / L * padded;
    const int64_t tiles = (a.rows + per_wave - 1) / per_wave;
    for (int64_t tile = (int64_t)blockIdx.x * SC_WAVES + wave; tile < tiles; tile += (int64_t)gridDim.x * SC_WAVES) {
        const int64_t r = tile * per_wave + lane / L;
        const bool on = r < a.rows;
        const typename X::E* x = (const typename X::E*)a.x + (on ? r : 0) * a.stride;
        const int idx = on && l < a.top ? a.index[r * a.top + l] : -1;
        const bool have = idx >= 0 && idx < E;
        const float g = have ? a.g[r * a.top + l] * a.scale : 0.0f;
        const float xi = have ? X::get(x + idx) : -INFINITY;
        for (int j = 4 * l; j < padded; j += 4 * L) *(float4*)(acc + j) = make_float4(0, 0, 0, 0);
        float f[DENSE ? NV * V : 1], m = 0, inv = 0, c, all = 0;
        if constexpr (DENSE) {
#pragma unroll
            for (int v = 0; v < NV; ++v) sc_read<X>(x, (v * L + l) * V, on ? E : 0, f + v * V);
            m = sc_lanes(sc_max<NV * V>(f, -INFINITY), L, FMaxOp());
            m = m == -INFINITY ? 0.0f : m;
            float total = 0;
#pragma unroll
            for (int i = 0; i < NV * V; ++i) {
                f[i] = __builtin_amdgcn_exp2f((f[i] - m) * SC_LOG2E);
                total += f[i];
            }
            total = sc_lanes(total, L, SumOp());
            inv = total == 0 ? 0.0f : 1.0f / total;
            c = have ? g * (__builtin_amdgcn_exp2f((xi - m) * SC_LOG2E) * inv) : 0.0f;
            all = inv * sc_lanes(c, L, SumOp());
        } else {
            const float w = sc_chosen_share(xi, have, a.sigmoid, a.renorm, L);
            c = w * (g - (a.renorm ? sc_lanes(w * g, L, SumOp()) : 0.0f));
            if (a.sigmoid) c *= xi > 0 ? expf(-xi) / (1 + expf(-xi)) : 1 / (1 + expf(xi));  // 1 - p
        }
        pd_wave_sync();
        if (have) unsafeAtomicAdd(acc + idx, c);
        pd_wave_sync();
        typename X::E* out = (typename X::E*)a.out + (on ? r : 0) * a.out_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * L + l) * V;
            if (!on || at >= E) continue;
            float d[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) *(float4*)(d + e) = *(const float4*)(acc + at + e);
            if constexpr (DENSE) {
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] -= f[v * V + e] * all;
            }
            if (at + V <= E) {
                sc_store_once<X>(out + at, X::pack(d));
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (at + e < E) X::put(out + at + e, d[e]);
            }
        }
        pd_wave_sync();  // the next rows' zeroes
    }
}

// ---- entry points --------------------------------------------------------------------------

static int sc_fail(const char* fn, const char* what) {
    pd_set_global_error("%s: %s", fn, what);
    return PD_E_INVALID;
}

static int sc_launched(const char* fn) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return PD_OK;
    pd_set_global_error("%s: launch failed: %s", fn, hipGetErrorString(e));
    return PD_E_HIP;
}

// Rows beyond this many workgroups are taken in turns.
static unsigned sc_grid(int64_t wanted) { return (unsigned)(wanted < 1 << 20 ? wanted : 1 << 20); }

static int sc_size(int dtype) { return dtype == PD_F32 ? 4 : dtype == PD_BF16 || dtype == PD_F16 ? 2 : 0; }

// What the calls have in common; 1: nothing to do.
static int sc_check_rows(const char* fn, const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, int64_t max_cols) {
    if (!sc_size(dtype)) return sc_fail(fn, "logits are PD_F32, PD_BF16 or PD_F16");
    if (rows < 0 || rows > INT32_MAX) return sc_fail(fn, "rows is outside 0..2^31-1");
    if (cols < 1 || cols > max_cols) {
        pd_set_global_error("%s: %lld columns are outside 1..%lld", fn, (long long)cols, (long long)max_cols);
        return PD_E_INVALID;
    }
    if (stride < 0 || stride > INT64_MAX / 8 / (rows > 0 ? rows : 1)) return sc_fail(fn, "bad row stride");
    if (rows == 0) return 1;
    if (!x) return sc_fail(fn, "logits are required");
    if ((uintptr_t)x % sc_size(dtype)) return sc_fail(fn, "logits are not aligned to their type");
    return 0;
}

// Whether one of `rows` intervals of `width` bytes from x on, x_step apart, meets one of as many from g on, g_step >= width
// apart.  Mostly told without the rows: by the whole ranges, or where the g lie in the gaps of every multiple of the steps' common
// divisor (columns next to each other, every other row); with equal steps that decides it.
static bool sc_rows_meet(uintptr_t x, int64_t x_step, uintptr_t g, int64_t g_step, int64_t rows, int64_t width) {
    const int64_t to_g = (int64_t)(g - x), x_end = (rows - 1) * x_step + width;  // from x on
    if (to_g >= x_end || to_g + (rows - 1) * g_step + width <= 0) return false;
    int64_t step = g_step;
    for (int64_t b = x_step; b; ) {
        const int64_t c = step % b;
        step = b;
        b = c;
    }
    const int64_t at = (to_g % step + step) % step;
    if (at >= width && at + width <= step) return false;
    if (x_step == g_step) return true;
    for (int64_t r = 0; r < rows; ++r) {
        const int64_t from = to_g + r * g_step;
        if (from >= x_end) break;
        if (from + width <= 0) continue;
        // the first x that ends behind `from`
        const int64_t k = from < width ? 0 : x_step ? (from - width) / x_step + 1 : rows;
        if (k < rows && k * x_step < from + width) return true;
    }
    return false;
}

// The gradient's rows: in the logits' own place, or clear of them.
static int sc_check_grad(const char* fn, const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, const void* grad,
                         int64_t grad_stride) {
    const int64_t size = sc_size(dtype);
    if ((uintptr_t)grad % size) return sc_fail(fn, "grad is not aligned to its type");
    if (grad_stride < cols || grad_stride > INT64_MAX / 8 / rows) return sc_fail(fn, "the rows of grad overlap");
    if (grad == x && (grad_stride == stride || rows == 1)) return PD_OK;
    if (sc_rows_meet((uintptr_t)x, stride * size, (uintptr_t)grad, grad_stride * size, rows, cols * size))
        return sc_fail(fn, "grad overlaps the logits without being them");
    return PD_OK;
}

// Lanes to a row of up to SC_WAVE_COLS columns: the fewest with at most 32 scores to a lane, as long as that leaves
// SC_ROW_WAVES wavefronts, four to a SIMD, and as the lanes' maxima bound the alternatives well.
#define SC_ROW_WAVES 4096

static int sc_row_lanes(int64_t rows, int64_t cols, int top) {
    int lanes = 64;
    const int least = top <= 8 ? 16 : top <= 16 ? 32 : 64;
    while (lanes > least && cols <= lanes / 2 * 32 && rows * (lanes / 2) >= 64 * SC_ROW_WAVES) lanes /= 2;
    return lanes;
}

// How a call with a workgroup to the row is cut.  Measured in the kernel, five alternatives, bfloat16, 64 / 256 / 1024
// threads: 8192 x 4096 22 / 43 / 224 us, 16 x 4096 6.1 / 6.2 / 8.1, 4096 x 16384 28 / 31 / 117, 1400 x 16384 17 / 15 / 45,
// 200 x 16384 10.7 / 6.8 / 8.6, 4096 x 131072 233 / 214 / 261, 255 x 131072 25 / 24 / 19.  So: one wavefront for rows of up to
// 4096 columns, and up to 32768 where there are eight for every CU (it waits for no other at a row's end); 1024 threads for
// long rows that leave CUs idle; 256 otherwise.  More than 32 alternatives need 256 parts.
// A row alone keeps one CU busy for 9 us per 131072 columns, and the join of slices costs 4 us: where few rows leave CUs for
// eight slices of SC_SLICE_COLS they are cut into as many as there are CUs for (1 x 131072 15.8 -> 12.5 us, 1 x 1000000 float32
// 21 -> 14; 100 x 131072 in two would go from 15 to 17).
#define SC_WAVE_COLS 2048
#define SC_CUS 256
#define SC_SLICE_COLS 16384

struct Cut {
    int wg, slices, slice_cols;
};

static Cut sc_cut(int64_t rows, int64_t cols, int top) {
    Cut c;
    int64_t want = SC_CUS / rows < cols / SC_SLICE_COLS ? SC_CUS / rows : cols / SC_SLICE_COLS;
    if (want < 8) want = 1;
    if (top <= 32 && (cols <= 4096 || (cols <= 32768 && rows >= 8 * SC_CUS)))
        c.wg = 64;
    else
        c.wg = rows < SC_CUS && cols > 32768 && want == 1 ? 1024 : SC_WG;
    const int64_t chunk = (int64_t)c.wg * SC_PER_THREAD, chunks = (cols + chunk - 1) / chunk;
    const int64_t least = (chunks + SC_MAX_CHUNKS(c.wg) - 1) / SC_MAX_CHUNKS(c.wg);  // what the segments' LDS holds
    if (want < least) want = least;
    const int64_t each = (chunks + want - 1) / want;
    c.slices = (int)((chunks + each - 1) / each);
    c.slice_cols = (int)(each * chunk);
    return c;
}

extern "C" uint64_t pd_token_logprobs_workspace(int dtype, int64_t rows, int64_t columns, int top) {
    if (!sc_size(dtype) || rows < 1 || rows > INT32_MAX || columns <= SC_WAVE_COLS || columns > PD_MAX_COLUMNS || top < 0 ||
        top > PD_MAX_ALTERNATIVES)
        return 0;
    const Cut c = sc_cut(rows, columns, top);
    if (c.slices == 1) return 0;
    return (((uint64_t)rows * c.slices * sizeof(Stat) + 15) & ~15ull) + (uint64_t)rows * c.slices * top * sizeof(uint64_t);
}

template <typename X, int WG>
static void sc_launch_logprobs_block(const LogprobArgs& a, hipStream_t stream) {
    const dim3 grid(sc_grid(a.rows * a.slices)), wg(WG);
    if (a.top)
        hipLaunchKernelGGL((k_token_logprobs_block<X, WG, true>), grid, wg, 0, stream, a);
    else
        hipLaunchKernelGGL((k_token_logprobs_block<X, WG, false>), grid, wg, 0, stream, a);
    if (a.slices > 1) hipLaunchKernelGGL((k_token_logprobs_join<X>), dim3(sc_grid(a.rows)), dim3(SC_WG), 0, stream, a);
}

template <typename X>
static void sc_launch_logprobs(const LogprobArgs& a, int wg_size, hipStream_t stream) {
    if (a.cols <= SC_WAVE_COLS) {
        const dim3 grid(sc_grid((a.rows * a.lanes + SC_WG - 1) / SC_WG)), wg(SC_WG);
        const int vecs = (a.cols + a.lanes * X::V - 1) / (a.lanes * X::V);
        if (vecs <= 1)
            hipLaunchKernelGGL((k_token_logprobs_rows<X, 1>), grid, wg, 0, stream, a);
        else if (vecs <= 2)
            hipLaunchKernelGGL((k_token_logprobs_rows<X, 2>), grid, wg, 0, stream, a);
        else if (vecs <= 3)
            hipLaunchKernelGGL((k_token_logprobs_rows<X, 3>), grid, wg, 0, stream, a);
        else if (vecs <= 4)
            hipLaunchKernelGGL((k_token_logprobs_rows<X, 4>), grid, wg, 0, stream, a);
        else if (vecs <= 6)  // float32 from here on: 16-bit rows have four at most
            hipLaunchKernelGGL((k_token_logprobs_rows<X, 24 / X::V>), grid, wg, 0, stream, a);
        else
            hipLaunchKernelGGL((k_token_logprobs_rows<X, 32 / X::V>), grid, wg, 0, stream, a);
        return;
    }
    if (wg_size == 64)
        sc_launch_logprobs_block<X, 64>(a, stream);
    else if (wg_size == SC_WG)
        sc_launch_logprobs_block<X, SC_WG>(a, stream);
    else
        sc_launch_logprobs_block<X, 1024>(a, stream);
}

extern "C" int pd_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t columns, int64_t row_stride,
                                 const int32_t* widths, const int64_t* tokens, int n_tokens, int top, float* logp,
                                 float* entropy, float* stats, float* top_logp, int32_t* top_index, void* workspace,
                                 uint64_t workspace_bytes, void* stream) {
    static const char fn[] = "pd_token_logprobs";
    const int rc = sc_check_rows(fn, logits, dtype, rows, columns, row_stride, PD_MAX_COLUMNS);
    if (rc < 0) return rc;
    if (n_tokens < 0 || n_tokens > PD_MAX_TOKENS) return sc_fail(fn, "n_tokens is outside 0..64");
    if (top < 0 || top > PD_MAX_ALTERNATIVES || top > columns) return sc_fail(fn, "top is outside 0..64 or larger than a row");
    if (rc == 1) return PD_OK;
    if (n_tokens && (!tokens || !logp)) return sc_fail(fn, "tokens and logp are required with n_tokens");
    if (top && (!top_logp || !top_index)) return sc_fail(fn, "top_logp and top_index are required with top");
    const uint64_t need = pd_token_logprobs_workspace(dtype, rows, columns, top);
    if (need && (!workspace || workspace_bytes < need)) {
        pd_set_global_error("%s: a workspace of %llu bytes is needed", fn, (unsigned long long)need);
        return PD_E_INVALID;
    }
    if (need && ((uintptr_t)workspace & 15)) return sc_fail(fn, "the workspace is not 16-byte aligned");
    LogprobArgs a = {logits, rows, row_stride, (int)columns, widths, tokens, n_tokens, top, logp, entropy, stats, top_logp, top_index};
    const Cut cut = sc_cut(rows, columns, top);
    a.lanes = sc_row_lanes(rows, columns, top);
    a.slices = cut.slices;
    a.slice_cols = cut.slice_cols;
    if (need) {
        a.part = (Stat*)workspace;
        a.part_keys = (uint64_t*)((char*)workspace + (((uint64_t)rows * a.slices * sizeof(Stat) + 15) & ~15ull));
    }
    if (dtype == PD_F32)
        sc_launch_logprobs<F32>(a, cut.wg, (hipStream_t)stream);
    else if (dtype == PD_BF16)
        sc_launch_logprobs<BF16>(a, cut.wg, (hipStream_t)stream);
    else
        sc_launch_logprobs<F16>(a, cut.wg, (hipStream_t)stream);
    return sc_launched(fn);
}

template <typename X>
static void sc_launch_logprobs_grad(const LogprobGradArgs& a, hipStream_t stream) {
    const dim3 wg(SC_WG);
    if (a.cols <= SC_WAVE_COLS) {
        const dim3 grid(sc_grid((a.rows + SC_WAVES - 1) / SC_WAVES));
        const int vecs = (a.cols + 64 * X::V - 1) / (64 * X::V);
        if (vecs <= 1)
            hipLaunchKernelGGL((k_token_logprobs_grad_wave<X, 1>), grid, wg, 0, stream, a);
        else if (vecs <= 2)
            hipLaunchKernelGGL((k_token_logprobs_grad_wave<X, 2>), grid, wg, 0, stream, a);
        else if (vecs <= 4)
            hipLaunchKernelGGL((k_token_logprobs_grad_wave<X, 4>), grid, wg, 0, stream, a);
        else
            hipLaunchKernelGGL((k_token_logprobs_grad_wave<X, SC_WAVE_COLS / 64 / X::V>), grid, wg, 0, stream, a);
        return;
    }
    const int64_t chunks = (a.cols + SC_CHUNK - 1) / SC_CHUNK;
    hipLaunchKernelGGL((k_token_logprobs_grad_block<X>), dim3(sc_grid(a.rows * chunks)), wg, 0, stream, a);
}

extern "C" int pd_token_logprobs_grad(const void* logits, int dtype, int64_t rows, int64_t columns, int64_t row_stride,
                                      const int32_t* widths, const float* stats, const int64_t* tokens, int n_tokens,
                                      const float* grad_logp, const float* grad_entropy, void* grad, int64_t grad_stride,
                                      void* stream) {
    static const char fn[] = "pd_token_logprobs_grad";
    const int rc = sc_check_rows(fn, logits, dtype, rows, columns, row_stride, PD_MAX_COLUMNS);
    if (rc < 0) return rc;
    if (n_tokens < 0 || n_tokens > PD_MAX_TOKENS) return sc_fail(fn, "n_tokens is outside 0..64");
    if (rc == 1) return PD_OK;
    if (!stats || !grad) return sc_fail(fn, "stats and grad are required");
    if (n_tokens && (!tokens || !grad_logp)) return sc_fail(fn, "tokens and grad_logp are required with n_tokens");
    if (sc_check_grad(fn, logits, dtype, rows, columns, row_stride, grad, grad_stride)) return PD_E_INVALID;
    LogprobGradArgs a = {logits, rows, row_stride, (int)columns, widths, stats, tokens, n_tokens, grad_logp, grad_entropy, grad, grad_stride};
    if (dtype == PD_F32)
        sc_launch_logprobs_grad<F32>(a, (hipStream_t)stream);
    else if (dtype == PD_BF16)
        sc_launch_logprobs_grad<BF16>(a, (hipStream_t)stream);
    else
        sc_launch_logprobs_grad<F16>(a, (hipStream_t)stream);
    return sc_launched(fn);
}

static int sc_check_route(const char* fn, int64_t experts, int top, int score) {
    if (score != PD_SCORE_SOFTMAX && score != PD_SCORE_SIGMOID) return sc_fail(fn, "score is PD_SCORE_SOFTMAX or PD_SCORE_SIGMOID");
    if (top < 1 || top > PD_MAX_ROUTES || top > experts) return sc_fail(fn, "top is outside 1..32 or larger than the number of experts");
    return 0;
}

#define SC_ROUTE_WAVES 2048

static int sc_pow2(int v) {
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

template <int EPL, int MODE>
static void sc_launch_route_epl(const RouteArgs& a, int kp, unsigned grid, hipStream_t stream) {
    const dim3 wg(SC_WG);
    if (kp == 2)
        hipLaunchKernelGGL((k_route<EPL, 2, MODE>), dim3(grid), wg, 0, stream, a);
    else if (kp == 4)
        hipLaunchKernelGGL((k_route<EPL, 4, MODE>), dim3(grid), wg, 0, stream, a);
    else if (kp == 8)
        hipLaunchKernelGGL((k_route<EPL, 8, MODE>), dim3(grid), wg, 0, stream, a);
    else if (kp == 16)
        hipLaunchKernelGGL((k_route<EPL, 16, MODE>), dim3(grid), wg, 0, stream, a);
    else
        hipLaunchKernelGGL((k_route<EPL, 32, MODE>), dim3(grid), wg, 0, stream, a);
}

template <int MODE>
static void sc_launch_route(const RouteArgs& a, int epl, int kp, hipStream_t stream) {
    const int64_t rows_wg = 64 / a.lanes * SC_WAVES;
    const unsigned grid = sc_grid((a.rows + rows_wg - 1) / rows_wg);
    if (epl <= 8)
        sc_launch_route_epl<8, MODE>(a, kp, grid, stream);
    else if (epl <= 16)
        sc_launch_route_epl<16, MODE>(a, kp, grid, stream);
    else
        sc_launch_route_epl<32, MODE>(a, kp, grid, stream);
}

extern "C" int pd_route_experts(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t row_stride,
                                const float* bias, int score, int groups, int top_groups, int group_score, int top,
                                int renormalise, float scale, float* weights, int32_t* index, void* stream) {
    static const char fn[] = "pd_route_experts";
    int rc = sc_check_rows(fn, logits, dtype, rows, experts, row_stride, PD_MAX_EXPERTS);
    if (rc < 0) return rc;
    if (sc_check_route(fn, experts, top, score)) return PD_E_INVALID;
    if (groups < 1 || groups > PD_MAX_GROUPS || experts % groups) return sc_fail(fn, "groups is outside 1..64 or does not divide the experts");
    if (top_groups < 1 || top_groups > groups) return sc_fail(fn, "top_groups is outside 1..groups");
    if (top > top_groups * (experts / groups)) return sc_fail(fn, "the chosen groups hold fewer than top experts");
    if (group_score != PD_GROUP_MAX && group_score != PD_GROUP_TOP2) return sc_fail(fn, "group_score is PD_GROUP_MAX or PD_GROUP_TOP2");
    if (rc == 1) return PD_OK;
    if (!weights || !index) return sc_fail(fn, "weights and index are required");
    RouteArgs a = {logits, dtype, rows, row_stride, (int)experts, top, score == PD_SCORE_SIGMOID, bias, groups, (int)experts / groups,
                   top_groups, group_score == PD_GROUP_TOP2, renormalise != 0, scale, weights, index};
    // The fewest lanes that hold a row, 16 experts each at most: a lane's work grows more slowly with its experts than the
    // rows of a wavefront fall with its lanes.  Where the rows leave most of the chip idle anyway a lane takes 8; 32 where
    // an odd number of groups would take more than the 64 lanes (G > gp / 2 groups of at most 1024 / G always fit then).
    const int kp = sc_pow2(top < 2 ? 2 : top), gp = sc_pow2(groups);
    a.lanes = kp > gp ? kp : gp;
    while (a.lanes < 64 && a.lanes / gp * 16 < a.per_group) a.lanes *= 2;
    if (a.lanes < 64 && a.lanes / gp * 8 < a.per_group && rows * a.lanes < 64 * SC_ROUTE_WAVES) a.lanes *= 2;
    a.group_lanes = a.lanes / gp;
    const int epl = (a.per_group + a.group_lanes - 1) / a.group_lanes;
    if (bias || (groups > 1 && a.top2))
        sc_launch_route<ROUTE_CLOSE>(a, epl, kp, (hipStream_t)stream);
    else if (dtype == PD_F32)
        sc_launch_route<ROUTE_PLAIN32>(a, epl, kp, (hipStream_t)stream);
    else
        sc_launch_route<ROUTE_PLAIN16>(a, epl, kp, (hipStream_t)stream);
    return sc_launched(fn);
}

template <typename X, int NV>
static void sc_launch_route_grad_nv(const RouteGradArgs& a, hipStream_t stream) {
    const int64_t rows_wg = 64 / a.lanes * SC_WAVES;
    const dim3 grid(sc_grid((a.rows + rows_wg - 1) / rows_wg)), wg(SC_WG);
    if (!a.sigmoid && !a.renorm)
        hipLaunchKernelGGL((k_route_grad<X, NV, true>), grid, wg, 0, stream, a);
    else
        hipLaunchKernelGGL((k_route_grad<X, NV, false>), grid, wg, 0, stream, a);
}

template <typename X>
static void sc_launch_route_grad(RouteGradArgs& a, hipStream_t stream) {
    // A 16-byte piece of the row to a lane, two where there are many rows, and a lane to every chosen expert; 16 experts to
    // a lane at most (the LDS rows).
    a.lanes = sc_pow2(a.top);
    while (a.lanes < 64 && a.lanes * X::V * (a.rows >= SC_ROUTE_WAVES * 8 ? 2 : 1) < a.experts) a.lanes *= 2;
    const int pieces = (a.experts + a.lanes * X::V - 1) / (a.lanes * X::V);
    if (pieces <= 1)
        sc_launch_route_grad_nv<X, 1>(a, stream);
    else if (pieces <= 2)
        sc_launch_route_grad_nv<X, 2>(a, stream);
    else
        sc_launch_route_grad_nv<X, 16 / X::V>(a, stream);
}

extern "C" int pd_route_experts_grad(const void* logits, int dtype, int64_t rows, int64_t experts, int64_t row_stride,
                                     const int32_t* index, const float* grad_weights, int score, int top, int renormalise,
                                     float scale, void* grad, int64_t grad_stride, void* stream) {
    static const char fn[] = "pd_route_experts_grad";
    const int rc = sc_check_rows(fn, logits, dtype, rows, experts, row_stride, PD_MAX_EXPERTS);
    if (rc < 0) return rc;
    if (sc_check_route(fn, experts, top, score)) return PD_E_INVALID;
    if (rc == 1) return PD_OK;
    if (!index || !grad_weights || !grad) return sc_fail(fn, "index, grad_weights and grad are required");
    if (sc_check_grad(fn, logits, dtype, rows, experts, row_stride, grad, grad_stride)) return PD_E_INVALID;
    RouteGradArgs a = {logits, rows, row_stride, (int)experts, top, score == PD_SCORE_SIGMOID, renormalise != 0, scale,
                       index, grad_weights, grad, grad_stride};
    if (dtype == PD_F32)
        sc_launch_route_grad<F32>(a, (hipStream_t)stream);
    else if (dtype == PD_BF16)
        sc_launch_route_grad<BF16>(a, (hipStream_t)stream);
    else
        sc_launch_route_grad<F16>(a, (hipStream_t)stream);
    return sc_launched(fn);
}
