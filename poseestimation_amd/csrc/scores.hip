// Operators on rows of scores: log probabilities of given tokens with entropy and top
// alternatives, the routing of rows to experts, and the gradients of both.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

#define SC_WG 256
#define SC_LOG2E 1.44269504088896340736f
#define SC_LN2 0.69314718055994530942f

// ---- elements ------------------------------------------------------------------------------

__device__ __forceinline__ float sc_get(const float* p) { return *p; }
__device__ __forceinline__ float sc_get(const __hip_bfloat16* p) {
    return __uint_as_float((uint32_t)*(const uint16_t*)p << 16);
}
__device__ __forceinline__ float sc_get(const _Float16* p) { return (float)*p; }

__device__ __forceinline__ void sc_put(float* p, float v) { *p = v; }
// round to nearest, ties to even; a NaN stays one
__device__ __forceinline__ void sc_put(__hip_bfloat16* p, float v) {
    const uint32_t u = __float_as_uint(v);
    *(uint16_t*)p = (uint16_t)(v != v ? (u >> 16) | 0x40 : (u + 0x7fff + ((u >> 16) & 1)) >> 16);
}
__device__ __forceinline__ void sc_put(_Float16* p, float v) { *p = (_Float16)v; }

// One whole number per (score, place): larger for the larger score, then for the lower place.
__device__ __forceinline__ uint64_t sc_key(float x, uint32_t at) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 counts as 0
    const uint32_t o = (u >> 31) ? ~u : (u | 0x80000000u);
    return ((uint64_t)o << 32) | (uint32_t)~at;
}
__device__ __forceinline__ float sc_key_score(uint64_t k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o >> 31) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint32_t sc_key_place(uint64_t k) { return ~(uint32_t)k; }

template <typename V, typename F>
__device__ __forceinline__ V sc_wave(V v, F f) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = f(v, __shfl_xor(v, d));
    return v;
}
struct SumOp { template <typename V> __device__ V operator()(V a, V b) const { return a + b; } };
struct MaxOp { template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; } };

template <typename V, typename F>
__device__ V sc_block(V v, F f, V* lds) {  // lds: SC_WG / 64 values
    v = sc_wave(v, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < SC_WG / 64; ++i) v = f(v, lds[i]);
    return v;
}

// ---- log probabilities ---------------------------------------------------------------------

struct LogprobArgs {
    const void* x;
    int64_t rows, stride;
    int cols;
    const int32_t* widths;
    const int64_t* tokens;
    int n_tok, top;
    float *logp, *entropy, *stats, *top_logp;
    int32_t* top_index;
};

__device__ __forceinline__ int sc_width(const int32_t* widths, int64_t r, int cols) {
    return widths ? pd_clampi(widths[r], 0, cols) : cols;
}

template <typename X>
__global__ __launch_bounds__(SC_WG) void k_token_logprobs(LogprobArgs a) {
    __shared__ float lf[SC_WG / 64];
    __shared__ uint64_t lk[SC_WG / 64];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const X* x = (const X*)a.x + r * a.stride;
        const int n = sc_width(a.widths, r, a.cols);
        float m = -INFINITY;
        for (int j = threadIdx.x; j < n; j += SC_WG) m = fmaxf(m, sc_get(x + j));
        m = sc_block(m, MaxOp(), lf);
        const float mb = m == -INFINITY ? 0.0f : m;
        float s = 0, w = 0;
        for (int j = threadIdx.x; j < n; j += SC_WG) {
            const float t = (sc_get(x + j) - mb) * SC_LOG2E, e = exp2f(t);
            s += e;
            w = fmaf(e, fmaxf(t, -256.0f), w);
        }
        s = sc_block(s, SumOp(), lf);
        w = sc_block(w, SumOp(), lf);
        const bool empty = s == 0, bad = s != s;
        const float log_sum = empty ? 0.0f : logf(s), h = empty ? 0.0f : log_sum - SC_LN2 * w / s;
        if (threadIdx.x == 0) {
            if (a.stats) {
                a.stats[3 * r] = m;
                a.stats[3 * r + 1] = log_sum;
                a.stats[3 * r + 2] = h;
            }
            if (a.entropy) a.entropy[r] = h;
        }
        for (int t = threadIdx.x; t < a.n_tok; t += SC_WG) {
            const int64_t tok = a.tokens[r * a.n_tok + t];
            float v = 0;
            if (tok >= 0) v = empty ? -INFINITY : ((tok < n ? sc_get(x + tok) : -INFINITY) - mb) - log_sum;
            a.logp[r * a.n_tok + t] = v;
        }
        uint64_t prev = ~0ull;
        for (int k = 0; k < a.top; ++k) {
            uint64_t best = 0;
            if (!bad && !empty)
                for (int j = threadIdx.x; j < n; j += SC_WG) {
                    const uint64_t key = sc_key(sc_get(x + j), j);
                    if (key < prev && key > best) best = key;
                }
            best = sc_block(best, MaxOp(), lk);
            prev = best;
            if (threadIdx.x == 0) {
                a.top_index[r * a.top + k] = bad ? -1 : best ? (int)sc_key_place(best) : k;
                a.top_logp[r * a.top + k] = bad ? NAN : best ? (sc_key_score(best) - mb) - log_sum : -INFINITY;
            }
        }
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

template <typename X>
__global__ __launch_bounds__(SC_WG) void k_token_logprobs_grad(LogprobGradArgs a) {
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const X* x = (const X*)a.x + r * a.stride;
        X* out = (X*)a.out + r * a.out_stride;
        const int n = sc_width(a.widths, r, a.cols);
        const float m = a.stats[3 * r], log_sum = a.stats[3 * r + 1], h = a.stats[3 * r + 2];
        const bool empty = m == -INFINITY && log_sum == 0;
        const float ge = a.g_entropy ? a.g_entropy[r] : 0.0f;
        float g = 0;
        for (int t = 0; t < a.n_tok; ++t)
            if (a.tokens[r * a.n_tok + t] >= 0) g += a.g_logp[r * a.n_tok + t];
        for (int j = threadIdx.x; j < a.cols; j += SC_WG) {
            float d = 0;
            if (j < n && !empty) {
                const float lp = (sc_get(x + j) - m) - log_sum, p = exp2f(lp * SC_LOG2E);
                d = -p * (g + ge * (fmaxf(lp, -256.0f) + h));
                for (int t = 0; t < a.n_tok; ++t)
                    if (a.tokens[r * a.n_tok + t] == j) d += a.g_logp[r * a.n_tok + t];
            }
            sc_put(out + j, d);
        }
    }
}

// ---- routing -------------------------------------------------------------------------------

struct RouteArgs {
    const void* x;
    int64_t rows, stride;
    int experts, top, sigmoid;
    const float* bias;
    int groups, top_groups, top2, renorm;
    float scale;
    float* weights;
    int32_t* index;
};

#define SC_PER_LANE (PD_MAX_EXPERTS / 64)

// The weights of the chosen experts of one row; lane i < top holds the i-th one's logit.
__device__ __forceinline__ void sc_route_weights(const RouteArgs& a, int64_t r, int lane, int idx, float xi, float m,
                                                 float total) {
    const bool have = lane < a.top;
    float wgt;
    if (a.sigmoid) {
        float big = sc_wave(have ? xi : -INFINITY, MaxOp());
        // a sum of tiny values is formed relative to the largest of them
        const float shift = a.renorm && big < 0 && big > -INFINITY ? big : 0.0f;
        wgt = xi < 0 ? expf(xi - shift) / (1 + expf(xi)) : 1 / (1 + expf(-xi));
    } else if (a.renorm) {
        float big = sc_wave(have ? xi : -INFINITY, MaxOp());
        wgt = big == -INFINITY ? 0.0f : expf(xi - big);
    } else {
        wgt = total == 0 ? 0.0f : expf(xi - m) / total;
    }
    if (!have) wgt = 0;
    if (a.renorm) {
        const float sum = sc_wave(wgt, SumOp());
        wgt = sum == 0 ? 0.0f : wgt / sum;
    }
    if (have) {
        a.weights[r * a.top + lane] = idx < 0 ? NAN : wgt * a.scale;
        a.index[r * a.top + lane] = idx;
    }
}

// One row by one wavefront, the order decided in float64.
template <typename X>
__device__ void sc_route_row(const RouteArgs& a, int64_t r, int lane) {
    const X* x = (const X*)a.x + r * a.stride;
    const int E = a.experts, per_group = E / a.groups;
    float m = -INFINITY;
    bool nan = false;
    for (int j = lane; j < E; j += 64) {
        const float v = sc_get(x + j);
        nan |= v != v || (v == INFINITY && !a.sigmoid);
        m = fmaxf(m, v);
    }
    nan = __any(nan);
    m = sc_wave(m, MaxOp());
    double total = 0;
    if (!a.sigmoid && m > -INFINITY)
        for (int j = lane; j < E; j += 64) total += exp((double)sc_get(x + j) - m);
    total = sc_wave(total, SumOp());
    double p[SC_PER_LANE], by[SC_PER_LANE];
#pragma unroll
    for (int i = 0; i < SC_PER_LANE; ++i) {
        const int j = lane + 64 * i;
        p[i] = by[i] = -INFINITY;
        if (j >= E) continue;
        const double v = sc_get(x + j);
        p[i] = a.sigmoid ? 1 / (1 + exp(-v)) : total > 0 ? exp(v - m) / total : 0.0;
        by[i] = a.bias ? p[i] + (double)a.bias[j] : v;
        if (!(by[i] >= -1e300)) by[i] = -1e300;  // -inf or NaN: behind every other, before what no group offers
    }
    if (a.groups > 1) {
        // lane g holds group g's score
        double mine = -INFINITY;
        for (int g = 0; g < a.groups; ++g) {
            double b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
            for (int i = 0; i < SC_PER_LANE; ++i) {
                const int j = lane + 64 * i;
                if (j >= E || j / per_group != g) continue;
                const double v = a.top2 && !a.bias ? p[i] : by[i];
                b2 = fmax(b2, fmin(b1, v));
                b1 = fmax(b1, v);
            }
#pragma unroll
            for (int d = 32; d; d >>= 1) {
                const double o1 = __shfl_xor(b1, d), o2 = __shfl_xor(b2, d);
                b2 = fmax(fmin(b1, o1), fmax(b2, o2));
                b1 = fmax(b1, o1);
            }
            const double s = a.top2 && per_group > 1 ? b1 + b2 : b1;
            if (lane == g) mine = s;
        }
        int rank = 0;
        for (int g = 0; g < a.groups; ++g) {
            const double o = __shfl(mine, g);
            rank += o > mine || (o == mine && g < lane);
        }
        const uint64_t kept = __ballot(lane < a.groups && rank < a.top_groups);
#pragma unroll
        for (int i = 0; i < SC_PER_LANE; ++i) {
            const int j = lane + 64 * i;
            if (j < E && !(kept >> (j / per_group) & 1)) by[i] = -INFINITY;
        }
    }
    int chosen = -1;
    for (int k = 0; k < a.top; ++k) {
        double best = -INFINITY;
        int at = E;
#pragma unroll
        for (int i = 0; i < SC_PER_LANE; ++i)
            if (by[i] > best) best = by[i], at = lane + 64 * i;
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            const double o = __shfl_xor(best, d);
            const int oa = __shfl_xor(at, d);
            if (o > best || (o == best && oa < at)) best = o, at = oa;
        }
#pragma unroll
        for (int i = 0; i < SC_PER_LANE; ++i)
            if (lane + 64 * i == at) by[i] = -INFINITY;
        if (lane == k) chosen = at;
    }
    const int idx = nan ? -1 : chosen;
    const float xi = lane < a.top && idx >= 0 ? sc_get(x + idx) : -INFINITY;
    sc_route_weights(a, r, lane, idx, xi, m, (float)total);
}

template <typename X>
__global__ __launch_bounds__(SC_WG) void k_route(RouteArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * (SC_WG / 64) + (threadIdx.x >> 6); r < a.rows; r += (int64_t)gridDim.x * (SC_WG / 64))
        sc_route_row<X>(a, r, lane);
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
};

template <typename X>
__global__ __launch_bounds__(SC_WG) void k_route_grad(RouteGradArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * (SC_WG / 64) + (threadIdx.x >> 6); r < a.rows; r += (int64_t)gridDim.x * (SC_WG / 64)) {
        const X* x = (const X*)a.x + r * a.stride;
        X* out = (X*)a.out + r * a.out_stride;
        const int E = a.experts;
        const int idx = lane < a.top ? a.index[r * a.top + lane] : -1;
        const bool have = idx >= 0 && idx < E;
        const float g = have ? a.g[r * a.top + lane] * a.scale : 0.0f;
        const float xi = have ? sc_get(x + idx) : -INFINITY;
        const bool dense = !a.sigmoid && !a.renorm;
        float m = 0, total = 0, wgt, c;
        if (a.sigmoid || a.renorm) {
            const float big = sc_wave(xi, MaxOp());
            if (a.sigmoid) {
                const float shift = a.renorm && big < 0 && big > -INFINITY ? big : 0.0f;
                wgt = xi < 0 ? expf(xi - shift) / (1 + expf(xi)) : 1 / (1 + expf(-xi));
            } else {
                wgt = big == -INFINITY ? 0.0f : expf(xi - big);
            }
            if (!have) wgt = 0;
            float sum = 0;
            if (a.renorm) {
                sum = sc_wave(wgt, SumOp());
                wgt = sum == 0 ? 0.0f : wgt / sum;
                sum = sc_wave(wgt * g, SumOp());
            }
            c = wgt * (g - sum);
            if (a.sigmoid) c *= xi > 0 ? expf(-xi) / (1 + expf(-xi)) : 1 / (1 + expf(xi));  // 1 - p
        } else {
            m = -INFINITY;
            for (int j = lane; j < E; j += 64) m = fmaxf(m, sc_get(x + j));
            m = sc_wave(m, MaxOp());
            if (m > -INFINITY)
                for (int j = lane; j < E; j += 64) total += expf(sc_get(x + j) - m);
            total = sc_wave(total, SumOp());
            wgt = have && total != 0 ? expf(xi - m) / total : 0.0f;
            c = wgt * g;
        }
        const float all = dense ? sc_wave(c, SumOp()) : 0.0f;
        for (int j0 = 0; j0 < E; j0 += 64) {
            const int j = j0 + lane;
            float d = 0;
            if (dense && j < E && total != 0) d = -(expf(sc_get(x + j) - m) / total) * all;
            for (int k = 0; k < a.top; ++k) {
                const int at = __shfl(have ? idx : -1, k);
                const float v = __shfl(c, k);
                if (at == j) d += v;
            }
            if (j < E) sc_put(out + j, d);
        }
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

static int sc_size(int dtype) { return dtype == PD_F32 ? 4 : dtype == PD_BF16 || dtype == PD_F16 ? 2 : 0; }

static unsigned sc_grid(int64_t wanted) { return (unsigned)(wanted < 1 << 20 ? wanted : 1 << 20); }

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

// The gradient's rows: in the logits' own place, or clear of them.
static int sc_check_grad(const char* fn, const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, const void* grad,
                         int64_t grad_stride) {
    if ((uintptr_t)grad % sc_size(dtype)) return sc_fail(fn, "grad is not aligned to its type");
    if (grad_stride < cols || grad_stride > INT64_MAX / 8 / rows) return sc_fail(fn, "the rows of grad overlap");
    const uintptr_t x0 = (uintptr_t)x, x1 = x0 + ((rows - 1) * stride + cols) * sc_size(dtype);
    const uintptr_t g0 = (uintptr_t)grad, g1 = g0 + ((rows - 1) * grad_stride + cols) * sc_size(dtype);
    if (g0 < x1 && x0 < g1 && !(g0 == x0 && (grad_stride == stride || rows == 1)))
        return sc_fail(fn, "grad overlaps the logits without being them");
    return PD_OK;
}

#define SC_BY_TYPE(dtype, kernel, grid, stream, args)                                                          \
    do {                                                                                                       \
        if ((dtype) == PD_F32)                                                                                 \
            hipLaunchKernelGGL((kernel<float>), dim3(grid), dim3(SC_WG), 0, (hipStream_t)(stream), args);      \
        else if ((dtype) == PD_BF16)                                                                           \
            hipLaunchKernelGGL((kernel<__hip_bfloat16>), dim3(grid), dim3(SC_WG), 0, (hipStream_t)(stream), args); \
        else                                                                                                   \
            hipLaunchKernelGGL((kernel<_Float16>), dim3(grid), dim3(SC_WG), 0, (hipStream_t)(stream), args);   \
    } while (0)

extern "C" uint64_t pd_token_logprobs_workspace(int dtype, int64_t rows, int64_t columns, int top) { return 0; }

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
    if (workspace_bytes < pd_token_logprobs_workspace(dtype, rows, columns, top)) return sc_fail(fn, "the workspace is too small");
    LogprobArgs a = {logits, rows, row_stride, (int)columns, widths, tokens, n_tokens, top, logp, entropy, stats, top_logp, top_index};
    SC_BY_TYPE(dtype, k_token_logprobs, sc_grid(rows), stream, a);
    return sc_launched(fn);
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
    SC_BY_TYPE(dtype, k_token_logprobs_grad, sc_grid(rows), stream, a);
    return sc_launched(fn);
}

static int sc_check_route(const char* fn, int64_t experts, int top, int score) {
    if (score != PD_SCORE_SOFTMAX && score != PD_SCORE_SIGMOID) return sc_fail(fn, "score is PD_SCORE_SOFTMAX or PD_SCORE_SIGMOID");
    if (top < 1 || top > PD_MAX_ROUTES || top > experts) return sc_fail(fn, "top is outside 1..32 or larger than the number of experts");
    return 0;
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
    RouteArgs a = {logits, rows, row_stride, (int)experts, top, score == PD_SCORE_SIGMOID, bias, groups, top_groups,
                   group_score == PD_GROUP_TOP2, renormalise != 0, scale, weights, index};
    SC_BY_TYPE(dtype, k_route, sc_grid((rows + 3) / 4), stream, a);
    return sc_launched(fn);
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
    SC_BY_TYPE(dtype, k_route_grad, sc_grid((rows + 3) / 4), stream, a);
    return sc_launched(fn);
}
