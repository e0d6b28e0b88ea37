// route.hip -- the experts of every column of logits, their weights, and the
// logits' gradient.
//
//   s_e = exp(l_e) / sum exp(l)  or  1 / (1 + exp(-l_e)),     key_e = s_e + bias_e
//   the best `keep` groups, of their experts the best `copies` keys, ties to the lowest
//   w_c = scale s_c  or  scale s_c / (sum of the chosen s)
//
// Keys are Float64: which of two experts is chosen goes by the scores and not by
// their rounding.  Without a bias the logits are the keys, in the same order.
#include "column_chunks.hpp"
#include "lanes.hpp"
#include "wave.hpp"

#include <cmath>

namespace jlust {
namespace {

constexpr int64_t MAX_EXPERTS = 4095, MAX_COPIES = 64, MAX_ROUTE_GROUPS = 64;
constexpr int64_t ROUTE_FEW = 4096;            // columns, up to which a wave takes one

struct RouteArgs {
    int64_t cols;
    int experts, groups, size, keep, best, copies, origin, score, renormalize;
    int lane_shift, per;                // lanes of a group (a power of two), experts of a lane
    bool whole;                         // every lane of a group has as many as the kernel holds
    const void *L;
    int64_t ldl;
    const void *bias;
    int32_t *ids;
    int64_t ldi;
    void *weights;
    int64_t ldw;
    double scale;
};

template <int LANES, typename A>
__device__ __forceinline__ A lanes_max(A v)
{
    return over_lanes<LANES>(v, Larger());
}

template <int LANES, typename A>
__device__ __forceinline__ A lanes_sum(A v)
{
    return over_lanes<LANES>(v, Plus());
}

// The first of a column's lanes where `is` holds, -1 if none.
template <int LANES>
__device__ __forceinline__ int first_lane(bool is)
{
    uint64_t mask = __ballot(is);
    if constexpr (LANES < 64) mask = mask >> (threadIdx.x & (64 - LANES)) & ((1ull << LANES) - 1);
    return __ffsll((unsigned long long)mask) - 1;
}

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// exp(l - top), 1 where both are the same infinity.
template <typename A>
__device__ __forceinline__ A exp_below(A l, A top)
{
    return l == top ? A(1) : exp_of(l - top);
}

// The chosen experts' scores up to a factor that they share, from their logits: NP
// each of LANES lanes (-inf: none).  Softmax: exp(l - m) with m the largest.  Sigmoid
// renormalised: times exp(-m) with m the largest, 0 at most, so that scores below the
// type's range keep their ratios; else as it is.
template <int LANES, int NP, typename A>
__device__ __forceinline__ void chosen_scores(int score, bool relative, const A (&l)[NP], A (&p)[NP])
{
    A m = -INFINITY;
#pragma unroll
    for (int q = 0; q < NP; ++q) m = l[q] > m ? l[q] : m;
    m = lanes_max<LANES>(m);
    if (score == JLUST_SCORE_SIGMOID) m = !relative || m > A(0) ? A(0) : m;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        if (!(l[q] > A(-INFINITY))) p[q] = A(0);
        else if (score == JLUST_SCORE_SOFTMAX) p[q] = exp_below(l[q], m);
        else p[q] = l[q] > A(0) ? A(1) / (A(1) + exp_of(-l[q])) : exp_below(l[q], m) / (A(1) + exp_of(l[q]));
    }
}

// LANES lanes take a column, `1 << lane_shift` of them a group, PER experts at most
// each: lane's experts and then the lanes' are in the experts' order, so the first
// lane with the best key holds the lowest expert that has it.  K: the keys' type,
// Float64 but for logits that are the keys themselves.  PER 0: any number of them, in
// LDS, a wave a workgroup.
template <typename T, typename K, int LANES, int PER>
__global__ __launch_bounds__(PER ? 256 : 64, PER ? 3 : 1) void route_kernel(const RouteArgs a)
{
    using A = typename Elem<T>::Acc;
    constexpr int NT = PER ? 256 : 64, COLS = NT / LANES, NP = MAX_COPIES / LANES, HELD = PER ? PER : 1;
    constexpr K NONE = -INFINITY;
    __shared__ int s_chosen[COLS][MAX_COPIES];
    extern __shared__ double s_keys[];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES, of_group = 1 << a.lane_shift;
    const int group = lane >> a.lane_shift, place = (lane & (of_group - 1)) * a.per;
    const int first = group * a.size + place;
    const bool softmax = a.score == JLUST_SCORE_SOFTMAX;
    const A *bias = (const A *)a.bias;
    K held[HELD];
    // f(j, key) of this lane's keys, which it may change.
    auto each = [&](auto &&f) {
        if constexpr (PER > 0) {
#pragma unroll
            for (int j = 0; j < PER; ++j) f(j, held[j]);
        } else {
            K *keys = (K *)s_keys + lane;
            for (int j = 0; j < a.per; ++j) {
                K k = keys[j * 64];
                f(j, k);
                keys[j * 64] = k;
            }
        }
    };
    for (int64_t c0 = (int64_t)blockIdx.x * COLS; c0 < a.cols; c0 += (int64_t)gridDim.x * COLS) {
        const int64_t c = c0 + sub;
        const T *L = (const T *)a.L + c * a.ldl;
        int count = a.size - place < a.per ? a.size - place : a.per;
        if (group >= a.groups || c >= a.cols || count < 0) count = 0;
        double top = -INFINITY, total = 1;
        if (PER > 0 && a.whole) {
            T raw[HELD] = {};
            if (count) load_vec<HELD>(L + first, raw);
#pragma unroll
            for (int j = 0; j < PER; ++j) held[j] = count && A(raw[j]) > A(-INFINITY) ? K(A(raw[j])) : NONE;
        } else {
            each([&](int j, K &k) {
                const K l = j < count ? K(A(L[first + j])) : NONE;
                k = l > NONE ? l : NONE;
            });
        }
        // Softmax's sum is needed where scores are compared or left as they are.
        if (softmax && (bias || !a.renormalize)) {
            K m = NONE;
            A sum = A(0);
            each([&](int, K &k) { m = k > m ? k : m; });
            m = lanes_max<LANES>(m);
            top = (double)m;
            if (bias) {
                double wide = 0;
                each([&](int, K &k) { wide += k > NONE ? exp_below((double)k, top) : 0; });
                total = lanes_sum<LANES>(wide);
            } else {
                each([&](int, K &k) { sum += k > NONE ? exp_below(A(k), A(m)) : A(0); });
                total = (double)lanes_sum<LANES>(sum);
            }
        }
        auto score_of = [&](double l, double m, double all) { return softmax ? exp_below(l, m) / all : 1 / (1 + exp(-l)); };
        if (bias) {
            auto keyed = [&](K &k, A b) {
                const K v = k > NONE ? K(score_of((double)k, top, total) + (double)b) : NONE;
                k = v > NONE ? v : NONE;
            };
            if (PER > 0 && a.whole) {
                A add[HELD] = {};
                if (count) load_vec<HELD>(bias + first, add);
#pragma unroll
                for (int j = 0; j < PER; ++j) keyed(held[j], add[j]);
            } else {
                each([&](int j, K &k) { keyed(k, j < count ? bias[first + j] : A(0)); });
            }
        }
        if (a.keep < a.groups) {
            K v1 = NONE, v2 = NONE;
            each([&](int, K &k) {
                v2 = k > v1 ? v1 : k > v2 ? k : v2;
                v1 = k > v1 ? k : v1;
            });
            K rank;
            if (a.best == 1) {
                rank = over_lanes<LANES>(v1, Larger(), of_group);
            } else {
                // The best of all the lanes' firsts, and of what is left of them and their seconds.
                const K m = over_lanes<LANES>(v1, Larger(), of_group);
                const uint64_t mine = __ballot(v1 == m) >> (threadIdx.x & 63 & ~(of_group - 1));
                const bool holds = (__ffsll((unsigned long long)mine) - 1) == (lane & (of_group - 1));
                const K rest = over_lanes<LANES>(holds ? v2 : v1, Larger(), of_group);
                double x = (double)m, y = (double)rest;
                if (!bias) {
                    const double most = softmax ? (double)lanes_max<LANES>(m) : 0;
                    x = m > NONE ? score_of(x, most, 1) : x;
                    y = rest > NONE ? score_of(y, most, 1) : y;
                }
                const double sum = m > NONE ? x + (rest > NONE ? y : 0) : (double)NONE;
                rank = K(sum);
                if constexpr (sizeof(K) == 4) {
                    // Sums are compared in 64 bits: each group's place among them instead.
                    int above = 0;
                    for (int g = 0; g < a.groups; ++g) {
                        const double o = __shfl(sum, (threadIdx.x & 63 & ~(LANES - 1)) + (g << a.lane_shift), 64);
                        above += o > sum || (o == sum && g < group);
                    }
                    rank = m > NONE ? K(-above) : NONE;
                }
            }
            bool kept = false;
            for (int r = 0; r < a.keep; ++r) {
                const K m = lanes_max<LANES>(rank);
                const int winner = first_lane<LANES>(rank == m && m > NONE);
                if (winner >= 0 && winner >> a.lane_shift == group) {
                    kept = true;
                    rank = NONE;
                }
            }
            each([&](int, K &k) { k = kept ? k : NONE; });
        }
        K best = NONE;
        int at = -1;
        each([&](int j, K &k) {
            if (k > best) {
                best = k;
                at = j;
            }
        });
        for (int r = 0; r < a.copies; ++r) {
            const K m = lanes_max<LANES>(best);
            const int winner = first_lane<LANES>(best == m && m > NONE);
            if (winner < 0 && lane == 0) s_chosen[sub][r] = -1;
            if (winner == lane) {
                s_chosen[sub][r] = first + at;
                const int gone = at;
                best = NONE;
                at = -1;
                each([&](int j, K &k) {
                    k = j == gone ? NONE : k;
                    if (k > best) {
                        best = k;
                        at = j;
                    }
                });
            }
        }
        wave_sync();
        A l[NP], p[NP];
        int e[NP];
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int i = lane + q * LANES;
            e[q] = i < a.copies && c < a.cols ? s_chosen[sub][i] : -1;
            l[q] = e[q] >= 0 ? A(L[e[q]]) : A(-INFINITY);
        }
        wave_sync();
        A sum = A(0);
        if (softmax && !a.renormalize) {
#pragma unroll
            for (int q = 0; q < NP; ++q) p[q] = e[q] >= 0 ? exp_below(l[q], A(top)) / A(total) : A(0);
        } else {
            chosen_scores<LANES>(a.score, a.renormalize, l, p);
        }
#pragma unroll
        for (int q = 0; q < NP; ++q) sum += p[q];
        sum = a.renormalize ? lanes_sum<LANES>(sum) : A(1);
        if (c >= a.cols) continue;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int i = lane + q * LANES;
            if (i >= a.copies) continue;
            a.ids[c * a.ldi + i] = e[q] + a.origin;
            ((A *)a.weights)[c * a.ldw + i] = e[q] >= 0 ? A(a.scale) * (p[q] / sum) : A(0);
        }
    }
}

// ------------------------------------------------------------------- gradient

struct RouteGradArgs {
    int64_t cols;
    int experts, copies, origin, score, renormalize;
    const void *L;
    int64_t ldl;
    const int32_t *ids;
    int64_t ldi;
    const void *dw;
    int64_t lddw;
    void *dL;
    int64_t lddl;
    double scale;
};

// exp(l - top) of many scores, where 16-bit results take no more than the hardware's.
template <typename T, typename A>
__device__ __forceinline__ A score_below(A l, A top)
{
    if constexpr (sizeof(T) == 2) return l == top ? A(1) : __expf(l - top);
    else return exp_below(l, top);
}

// With t = scale dw and p the weights' shares of the chosen: softmax renormalised
// p (t - sum p t), sigmoid renormalised the same times 1 - s, sigmoid t s (1 - s) at the
// chosen and 0 elsewhere; softmax as it is s_e (t_e - sum s t) everywhere.  LANES lanes
// take a column, CPL chunks of 16 bytes each in registers, so logits are read once (CPL
// 0: any number, read again).
template <typename T, int LANES, int CPL>
__global__ __launch_bounds__(256) void route_grad_kernel(const RouteGradArgs a)
{
    constexpr int CH = 16 / sizeof(T), HELD = CPL ? CPL : 1;
    using A = typename Elem<T>::Acc;
    constexpr int COLS = 256 / LANES, NP = MAX_COPIES / LANES;
    __shared__ int s_expert[COLS][MAX_COPIES];
    __shared__ A s_part[COLS][MAX_COPIES];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const bool softmax = a.score == JLUST_SCORE_SOFTMAX, dense = softmax && !a.renormalize;
    for (int64_t c0 = (int64_t)blockIdx.x * COLS; c0 < a.cols; c0 += (int64_t)gridDim.x * COLS) {
        const int64_t c = c0 + sub;
        const bool live = c < a.cols;
        const T *L = (const T *)a.L + c * a.ldl;
        A top = -INFINITY, total = A(0), s[HELD][CH];
        if (CPL > 0 && dense) {
            uint32x4 raw[HELD];
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                const int at = (lane + LANES * i) * CH;
                raw[i] = read_raw(L + at, live ? a.experts - at : 0);
            }
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                values<T>(raw[i], s[i]);
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    const bool some = live && (lane + LANES * i) * CH + j < a.experts && s[i][j] > A(-INFINITY);
                    s[i][j] = some ? s[i][j] : A(-INFINITY);
                    top = s[i][j] > top ? s[i][j] : top;
                }
            }
            top = lanes_max<LANES>(top);
#pragma unroll
            for (int i = 0; i < CPL; ++i)
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    s[i][j] = s[i][j] > A(-INFINITY) ? score_below<T>(s[i][j], top) : A(0);
                    total += s[i][j];
                }
            total = lanes_sum<LANES>(total);
        } else if (dense) {
            if (live)
                for (int e = lane; e < a.experts; e += LANES) top = A(L[e]) > top ? A(L[e]) : top;
            top = lanes_max<LANES>(top);
            if (live)
                for (int e = lane; e < a.experts; e += LANES)
                    if (A(L[e]) > A(-INFINITY)) total += score_below<T>(A(L[e]), top);
            total = lanes_sum<LANES>(total);
        }
        A l[NP], t[NP], p[NP];
        int at[NP];
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int i = lane + q * LANES;
            at[q] = -1;
            l[q] = -INFINITY;
            t[q] = A(0);
            if (live && i < a.copies) {
                const int64_t e = (int64_t)a.ids[c * a.ldi + i] - a.origin;
                if (e >= 0 && e < a.experts) {
                    at[q] = (int)e;
                    l[q] = A(L[e]);
                    t[q] = A(a.scale) * ((const A *)a.dw)[c * a.lddw + i];
                }
            }
        }
        A sum = A(0), dot = A(0);
        if (dense) {
#pragma unroll
            for (int q = 0; q < NP; ++q) p[q] = l[q] > A(-INFINITY) ? exp_below(l[q], top) / total : A(0);
        } else {
            chosen_scores<LANES>(a.score, a.renormalize, l, p);
            if (a.renormalize) {
#pragma unroll
                for (int q = 0; q < NP; ++q) sum += p[q];
                sum = lanes_sum<LANES>(sum);
#pragma unroll
                for (int q = 0; q < NP; ++q) p[q] = p[q] > A(0) ? p[q] / sum : A(0);
            }
        }
        if (softmax || a.renormalize) {
#pragma unroll
            for (int q = 0; q < NP; ++q) dot += p[q] * t[q];
            dot = lanes_sum<LANES>(dot);
        }
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const int i = lane + q * LANES;
            if (i >= a.copies) continue;
            A g = dense ? t[q] : p[q] * (t[q] - dot);
            if (!softmax) g *= A(1) / (A(1) + exp_of(l[q]));
            s_expert[sub][i] = at[q];
            s_part[sub][i] = at[q] >= 0 ? g : A(0);
        }
        wave_sync();
        if constexpr (CPL > 0) {
            const A inv = total > A(0) ? A(1) / total : A(0);
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                const int at = (lane + LANES * i) * CH;
                A g[CH];
#pragma unroll
                for (int j = 0; j < CH; ++j) g[j] = A(0);
                for (int k = 0; k < a.copies; ++k) {
                    const int e = s_expert[sub][k] - at;
                    const A v = s_part[sub][k];
#pragma unroll
                    for (int j = 0; j < CH; ++j) g[j] += e == j ? v : A(0);
                }
                if (dense) {
#pragma unroll
                    for (int j = 0; j < CH; ++j) g[j] = s[i][j] * inv * (g[j] - dot);
                }
                if (live) write_chunk((T *)a.dL + c * a.lddl + at, a.experts - at, g);
            }
        } else if (live) {
            for (int e = lane; e < a.experts; e += LANES) {
                A g = A(0);
                for (int i = 0; i < a.copies; ++i) g += s_expert[sub][i] == e ? s_part[sub][i] : A(0);
                if (dense) {
                    const A v = A(L[e]);
                    g = v > A(-INFINITY) ? score_below<T>(v, top) / total * (g - dot) : A(0);
                }
                ((T *)a.dL)[c * a.lddl + e] = T(g);
            }
        }
        wave_sync();
    }
}

// ----------------------------------------------------------------------- host

// The lanes of a group (their binary logarithm) and the experts of a lane when `lanes`
// take a column; false where they do not hold the groups.
bool route_lanes(int lanes, RouteArgs *a)
{
    if (a->groups > lanes) return false;
    a->lane_shift = 0;
    while (a->groups << (a->lane_shift + 1) <= lanes) ++a->lane_shift;
    a->per = (a->size + (1 << a->lane_shift) - 1) >> a->lane_shift;
    return true;
}

template <typename T, typename K, int LANES, int PER>
int launch_route(RouteArgs a, hipStream_t s)
{
    constexpr int NT = PER ? 256 : 64;
    a.whole = a.per == PER && a.size % (PER ? PER : 1) == 0;
    hipLaunchKernelGGL((route_kernel<T, K, LANES, PER>), dim3(column_blocks(a.cols, NT / LANES)), dim3(NT),
                       PER ? 0 : sizeof(K) * 64 * a.per, s, a);
    return check_launch("route_kernel");
}

// 16 lanes a column where it fits them and the columns fill the CUs (a round of the
// best key then serves four columns), else a wave.
template <typename T, typename K>
int route(RouteArgs a, hipStream_t s)
{
    if (a.cols > ROUTE_FEW && route_lanes(16, &a) && a.per <= 16) {
        if (a.per <= 1) return launch_route<T, K, 16, 1>(a, s);
        if (a.per <= 2) return launch_route<T, K, 16, 2>(a, s);
        if (a.per <= 4) return launch_route<T, K, 16, 4>(a, s);
        if (a.per <= 8) return launch_route<T, K, 16, 8>(a, s);
        return launch_route<T, K, 16, 16>(a, s);
    }
    route_lanes(64, &a);
    if (a.per <= 1) return launch_route<T, K, 64, 1>(a, s);
    if (a.per <= 2) return launch_route<T, K, 64, 2>(a, s);
    if (a.per <= 4) return launch_route<T, K, 64, 4>(a, s);
    if (a.per <= 16) return launch_route<T, K, 64, 16>(a, s);
    return launch_route<T, K, 64, 0>(a, s);
}

int check_route(const char *who, int32_t value_type, int32_t score, int64_t experts, int64_t cols, int64_t copies, double scale)
{
    if (int st = check_extents(who, value_type, experts, cols)) return st;
    if (score != JLUST_SCORE_SOFTMAX && score != JLUST_SCORE_SIGMOID)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: unknown score %d", who, score);
    if (experts < 1 || experts > MAX_EXPERTS)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %lld experts are not within [1, %lld]", who, (long long)experts,
                    (long long)MAX_EXPERTS);
    if (copies < 1 || copies > MAX_COPIES || copies > experts)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %lld of %lld experts are not within [1, %lld]", who, (long long)copies,
                    (long long)experts, (long long)MAX_COPIES);
    if (!std::isfinite(scale)) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: scale is not finite", who);
    return JLUST_STATUS_SUCCESS;
}

}  // namespace
}  // namespace jlust

using namespace jlust;

extern "C" int jlust_hip_route(const jlust_route *op, jlust_stream_t stream)
{
    clear_error();
    const char *who = "route";
    if (!op) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: null argument", who);
    if (int st = check_route(who, op->value_type, op->score, op->experts, op->cols, op->copies, op->scale)) return st;
    if (int st = check_origin(op->origin)) return st;
    if (op->groups < 1 || op->groups > MAX_ROUTE_GROUPS || op->experts % op->groups)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %lld experts do not make %lld equal groups of at most %lld", who,
                    (long long)op->experts, (long long)op->groups, (long long)MAX_ROUTE_GROUPS);
    if (op->keep < 1 || op->keep > op->groups || op->copies > op->experts / op->groups * op->keep)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %lld of %lld groups do not hold %lld of the experts", who,
                    (long long)op->keep, (long long)op->groups, (long long)op->copies);
    if (op->best != 1 && op->best != 2)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: a group is ranked by its best 1 or 2 experts, not %lld", who, (long long)op->best);
    if (int st = check_matrix(who, "L", op->L, op->experts, op->cols, op->ldl, true)) return st;
    if (int st = check_matrix(who, "ids", op->ids, op->copies, op->cols, op->ldi, true)) return st;
    if (int st = check_matrix(who, "weights", op->weights, op->copies, op->cols, op->ldw, true)) return st;
    if (int st = require_device(nullptr)) return st;
    if (op->cols == 0) return JLUST_STATUS_SUCCESS;
    RouteArgs a;
    a.cols = op->cols;
    a.experts = (int)op->experts;
    a.groups = (int)op->groups;
    a.size = (int)(op->experts / op->groups);
    a.keep = (int)op->keep;
    a.best = (int)op->best;
    a.copies = (int)op->copies;
    a.origin = op->origin;
    a.score = op->score;
    a.renormalize = op->renormalize;
    a.lane_shift = a.per = 0;
    a.whole = false;
    a.L = op->L;
    a.ldl = op->ldl;
    a.bias = op->bias;
    a.ids = op->ids;
    a.ldi = op->ldi;
    a.weights = op->weights;
    a.ldw = op->ldw;
    a.scale = op->scale;
    return with_type(op->value_type, [&](auto t) {
        using T = decltype(t);
        if constexpr (sizeof(T) < 8)
            if (!a.bias) return route<T, float>(a, (hipStream_t)stream);
        return route<T, double>(a, (hipStream_t)stream);
    });
}

extern "C" int jlust_hip_route_grad(const jlust_route_grad *op, jlust_stream_t stream)
{
    clear_error();
    const char *who = "route_grad";
    if (!op) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: null argument", who);
    if (int st = check_route(who, op->value_type, op->score, op->experts, op->cols, op->copies, op->scale)) return st;
    if (int st = check_origin(op->origin)) return st;
    if (int st = check_matrix(who, "L", op->L, op->experts, op->cols, op->ldl, true)) return st;
    if (int st = check_matrix(who, "ids", op->ids, op->copies, op->cols, op->ldi, true)) return st;
    if (int st = check_matrix(who, "dweights", op->dweights, op->copies, op->cols, op->lddw, true)) return st;
    if (int st = check_matrix(who, "dL", op->dL, op->experts, op->cols, op->lddl, true)) return st;
    if (int st = require_device(nullptr)) return st;
    if (op->cols == 0) return JLUST_STATUS_SUCCESS;
    RouteGradArgs a;
    a.cols = op->cols;
    a.experts = (int)op->experts;
    a.copies = (int)op->copies;
    a.origin = op->origin;
    a.score = op->score;
    a.renormalize = op->renormalize;
    a.L = op->L;
    a.ldl = op->ldl;
    a.ids = op->ids;
    a.ldi = op->ldi;
    a.dw = op->dweights;
    a.lddw = op->lddw;
    a.dL = op->dL;
    a.lddl = op->lddl;
    a.scale = op->scale;
    return with_type(op->value_type, [&](auto t) {
        using T = decltype(t);
        const int64_t chunks = (a.experts * (int64_t)sizeof(T) + 15) / 16;
        auto launch = [&](auto kernel, int lanes) {
            hipLaunchKernelGGL(kernel, dim3(column_blocks(a.cols, 256 / lanes)), dim3(256), 0, (hipStream_t)stream, a);
            return check_launch("route_grad_kernel");
        };
        if (chunks <= 16) return launch(route_grad_kernel<T, 16, 1>, 16);
        if (chunks <= 32) return launch(route_grad_kernel<T, 16, 2>, 16);
        if (chunks <= 64) return launch(route_grad_kernel<T, 16, 4>, 16);
        if (chunks <= 256) return launch(route_grad_kernel<T, 64, 4>, 64);
        return launch(route_grad_kernel<T, 64, 0>, 64);
    });
}

namespace jlust {
int preload_route()
{
    JLUST_PRELOAD_KERNEL((route_kernel<float, double, 64, 4>));
    return JLUST_STATUS_SUCCESS;
}
}  // namespace jlust
