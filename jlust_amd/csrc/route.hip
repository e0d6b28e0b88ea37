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

#include <cfloat>
#include <cmath>
#include <type_traits>

namespace jlust {
namespace {

constexpr int64_t MAX_EXPERTS = 4095, MAX_COPIES = 64, MAX_ROUTE_GROUPS = 64;
constexpr int64_t ROUTE_FEW = 2560;            // columns, up to which a wave takes one

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

// Whether this is the first of a column's lanes where `is` holds; the lanes of the wave
// before it in its column.
__device__ __forceinline__ bool first_of(bool is, uint64_t before) { return is && (__ballot(is) & before) == 0; }

template <int LANES>
__device__ __forceinline__ uint64_t lanes_before()
{
    const int lane = threadIdx.x & 63;
    return ((1ull << lane) - 1) & ~((1ull << (lane & ~(LANES - 1))) - 1);
}

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// exp(l - top), 1 where both are the same infinity.  Made in any case, as the scores
// below are, and dropped where it does not count: a branch a score took three times the
// instructions of the scores.
template <typename A>
__device__ __forceinline__ A exp_below(A l, A top)
{
    const A v = exp_of(l - top);
    return l == top ? A(1) : v;
}

// The chosen experts' scores up to a factor that they share, from their logits: NP
// each of LANES lanes, the first `parts` of which hold some (-inf: none).  Softmax: exp(l - m) with m the largest.  Sigmoid
// renormalised: times exp(-m) with m the largest, 0 at most, so that scores below the
// type's range keep their ratios; else as it is.
template <int LANES, int NP, typename A>
__device__ __forceinline__ void chosen_scores(int score, bool relative, int parts, const A (&l)[NP], A (&p)[NP])
{
    A m = -INFINITY;
#pragma unroll
    for (int q = 0; q < NP; ++q) m = l[q] > m ? l[q] : m;
    m = lanes_max<LANES>(m);
    if (score == JLUST_SCORE_SIGMOID) m = !relative || m > A(0) ? A(0) : m;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        p[q] = A(0);
        if (q >= parts) continue;
        if (!(l[q] > A(-INFINITY))) p[q] = A(0);
        else if (score == JLUST_SCORE_SOFTMAX) p[q] = exp_below(l[q], m);
        else p[q] = l[q] > A(0) ? A(1) / (A(1) + exp_of(-l[q])) : exp_below(l[q], m) / (A(1) + exp_of(l[q]));
    }
}

// The middle one of three numbers.
__device__ __forceinline__ float middle(float a, float b, float c) { return __builtin_amdgcn_fmed3f(a, b, c); }
__device__ __forceinline__ double middle(double a, double b, double c) { return fmax(fmin(a, b), fmin(fmax(a, b), c)); }

// How far apart two Float32 keys are in 64 bits for sure, over 1 + the larger: a
// sigmoid's is off by 4 u (u = 2^-24: its exponential's argument 0.4, the exponential
// 0.5, the sum 1, the reciprocal 2), a softmax's by 27 u (its argument 1 and its sum's
// 20 adds and 2 more, the rest 4; a lane of more than 16 experts adds up to 124), the sum
// with the bias by u times itself.  Twice that, rounded up.
constexpr float SIGMOID_APART = 16 * 0x1p-24f, SOFTMAX_APART = 64 * 0x1p-24f, SOFTMAX_APART_LONG = 288 * 0x1p-24f;

// What a lane's share of a column is: `count` experts from `first` on; of none `first` is
// 0, which may be read: a branch around every read waits for the read before.
struct RouteShare { int lane, group, first, count; };

constexpr int MAX_CANDIDATES = MAX_COPIES + 16;

// Writes the experts of a column to chosen[0 .. copies), -1 where none is left, and
// softmax's largest logit and sum where the call needs them.  LANES lanes take a column,
// `1 << lane_shift` of them a group, PER experts at most each (0: any number, their keys
// in LDS): a lane's experts and then the lanes' are in the experts' order, so the first
// lane with the best key holds the lowest expert that has it.  K: the keys' type.
// APPROX: Float32 keys, with a bias of scores that belong to Float64, without one the
// logits, whose last bits the rounds do without.  What they leave open, which groups are
// the last kept and the order of the experts, goes by the sigmoids (or logits) in Float64
// of those few that are near enough (`exact`: theirs); true where that does not settle it
// (more than 16 experts as near to the last one chosen, or softmax with a bias, whose
// Float64 sum takes them all).
template <typename T, typename K, bool APPROX, bool BIASED, int LANES, int PER>
__device__ __forceinline__ bool choose(const RouteArgs &a, const RouteShare &w, const T *L, char *lds, int *chosen, double *exact,
                                       double *top_, double *total_)
{
    using A = typename Elem<T>::Acc;
    constexpr bool ROUGH = APPROX && BIASED;
    using S = std::conditional_t<ROUGH, float, double>;                 // the scores' type
    constexpr int HELD = PER ? PER : 1;
    constexpr K NONE = -INFINITY;
    const int of_group = 1 << a.lane_shift;
    const bool softmax = a.score == JLUST_SCORE_SOFTMAX;
    const float apart = !softmax ? SIGMOID_APART : PER ? SOFTMAX_APART : SOFTMAX_APART_LONG;
    const A *bias = (const A *)a.bias;
    const uint64_t before = lanes_before<LANES>();
    bool unsure = false;
    K held[HELD];
    // f(j, key) of this lane's keys, which it may change.
    auto each = [&](auto &&f) {
        if constexpr (PER > 0) {
#pragma unroll
            for (int j = 0; j < PER; ++j) f(j, held[j]);
        } else {
            K *keys = (K *)lds + w.lane;
            for (int j = 0; j < a.per; ++j) {
                K k = keys[j * 64];
                f(j, k);
                keys[j * 64] = k;
            }
        }
    };
    if (PER > 0 && a.whole) {
        T raw[HELD];
        load_vec<HELD>(L + w.first, raw);
#pragma unroll
        for (int j = 0; j < PER; ++j) held[j] = w.count && A(raw[j]) > A(-INFINITY) ? K(A(raw[j])) : NONE;
    } else {
        each([&](int j, K &k) {
            const A l = A(L[w.first + (j < w.count ? j : 0)]);
            k = j < w.count && l > A(-INFINITY) ? K(l) : NONE;
        });
    }
    // Softmax's sum is needed where scores are compared or left as they are.
    S top = -INFINITY, total = 1;
    if (softmax && (BIASED || !a.renormalize)) {
        K m = NONE;
        each([&](int, K &k) { m = k > m ? k : m; });
        m = lanes_max<LANES>(m);
        top = S(m);
        if (BIASED) {
            S sum = 0;
            each([&](int, K &k) {
                const S v = exp_below(S(k), top);
                sum += k > NONE ? v : S(0);
            });
            total = lanes_sum<LANES>(sum);
        } else {
            A sum = A(0);
            each([&](int, K &k) {
                const A v = exp_below(A(k), A(m));
                sum += k > NONE ? v : A(0);
            });
            total = S(lanes_sum<LANES>(sum));
        }
    }
    *top_ = (double)top;
    *total_ = (double)total;
    auto part_of = [&](S l, S m, S all) {
        if constexpr (ROUGH) {
            const S v = __expf(l - m);
            return (l == m ? S(1) : v) / all;
        } else {
            return exp_below(l, m) / all;
        }
    };
    auto sigmoid = [&](S l) {
        if constexpr (ROUGH) return __builtin_amdgcn_rcpf(1 + __expf(-l));
        else return 1 / (1 + exp(-l));
    };
    if constexpr (BIASED) {
        auto key_all = [&](auto &&score) {
            auto keyed = [&](K &k, A b) {
                K v = K(score(S(k)) + S(b));
                v = k > NONE ? v : NONE;
                k = Larger()(v, NONE);             // of NaN, NONE
            };
            if (PER > 0 && a.whole) {
                A add[HELD];
                load_vec<HELD>(bias + w.first, add);
#pragma unroll
                for (int j = 0; j < PER; ++j) keyed(held[j], add[j]);
            } else {
                each([&](int j, K &k) { keyed(k, bias[w.first + (j < w.count ? j : 0)]); });
            }
        };
        if (softmax) key_all([&](S l) { return part_of(l, top, total); });
        else key_all(sigmoid);
    }
    if (a.keep < a.groups) {
        K v1 = NONE, v2 = NONE;
        each([&](int, K &k) {
            v2 = middle(v1, v2, k);
            v1 = Larger()(v1, k);
        });
        using R = std::conditional_t<ROUGH, K, S>;    // sums are compared in 64 bits
        R rank;
        K least;                                   // the last key that its rank goes by
        float undone = 0;                          // what a rank's two keys have of each other's sign
        const int first_in_wave = threadIdx.x & 63 & ~(LANES - 1);
        const uint64_t column = (LANES < 64 ? (1ull << (LANES & 63)) - 1 : ~0ull) << first_in_wave;
        // The best of all the lanes' firsts, and of what is left of them and their seconds.
        auto best_two = [&](auto &x, auto &y) {
            const auto m = over_lanes<LANES>(x, Larger(), of_group);
            const uint64_t mine = __ballot(x == m) >> (threadIdx.x & 63 & ~(of_group - 1));
            const bool holds = (__ffsll((unsigned long long)mine) - 1) == (w.lane & (of_group - 1));
            y = over_lanes<LANES>(holds ? y : x, Larger(), of_group);
            x = m;
        };
        // The lanes of the first group that is `in` and whose rank is the best.
        auto wins = [&](bool in, auto r, auto m) {
            const uint64_t mask = __ballot(in && r == m) & column;
            return mask != 0 && (__ffsll((unsigned long long)mask) - 1 - first_in_wave) >> a.lane_shift == w.group;
        };
        if (a.best == 1) {
            least = over_lanes<LANES>(v1, Larger(), of_group);
            rank = R(least);
        } else {
            best_two(v1, v2);
            const K m = v1, rest = v2;
            least = rest > NONE ? rest : m;
            S x = S(m), y = S(rest);
            if (!BIASED) {
                const S most = softmax ? S(lanes_max<LANES>(m)) : S(0);
                x = m > NONE ? softmax ? part_of(x, most, S(1)) : sigmoid(x) : x;
                y = rest > NONE ? softmax ? part_of(y, most, S(1)) : sigmoid(y) : y;
            }
            const S sum = x + (rest > NONE ? y : S(0));
            // A Float32 sum of a group with a candidate may be less than the type holds; as
            // its lowest value it is near all others past that, for 64 bits to settle.
            rank = !(m > NONE) ? S(-INFINITY) : ROUGH ? Larger()(sum, S(-FLT_MAX)) : sum;
            if constexpr (ROUGH) undone = rest > NONE && y < 0 && x > 0 ? -2 * y : 0;
        }
        // Which groups have a candidate goes by their keys: a Float64 sum may be -infinity.
        bool kept = false, waits = least > NONE;
        R last = -INFINITY;
        for (int r = 0; r < a.keep; ++r) {
            last = lanes_max<LANES>(waits ? rank : R(-INFINITY));
            if (wins(waits, rank, last)) {
                kept = true;
                waits = false;
            }
        }
        if constexpr (ROUGH) {
            const K next = lanes_max<LANES>(waits ? rank : NONE);
            // Keys of two signs make a sum smaller than they are: their error is not.
            if (__ballot(undone > 0)) undone = lanes_max<LANES>(undone);
            const float near = a.best * apart * (1 + fabsf(last) + undone);
            const bool open = next > NONE && !(last - next > near);
            if (softmax) {
                unsure = open;
            } else if (__ballot(open)) {
                // Kept for sure: what is past the best one left out.  Of those as near
                // as that to the last one kept the best in 64 bits fill the places.
                const bool sure = rank > next + near, maybe = open && !sure && rank > NONE && !(rank < last - near);
                double d1 = -INFINITY, d2 = -INFINITY;
                for (int base = 0; base < a.per; base += 32) {
                    uint32_t some = 0;
                    each([&](int j, K &k) {
                        if (j >= base && j < base + 32 && k > NONE && !(k < least - apart * (1 + fabsf(least)))) some |= 1u << (j - base);
                    });
                    if (!maybe) some = 0;
                    while (__ballot(some != 0)) {
                        if (some) {
                            const int e = w.first + base + __ffs(some) - 1;
                            some &= some - 1;
                            const double v = 1 / (1 + exp(-(double)A(L[e]))) + (double)bias[e];
                            d2 = v > d1 ? d1 : v > d2 ? v : d2;
                            d1 = v > d1 ? v : d1;
                        }
                    }
                }
                best_two(d1, d2);
                double wide = !maybe ? -INFINITY : a.best == 2 && d2 > -INFINITY ? d1 + d2 : d1;
                const bool leads = (w.lane & (of_group - 1)) == 0;
                const int places = a.keep - __popcll(__ballot(sure && leads) & column);
                if (open) kept = sure;
                for (int r = 0; r < a.keep; ++r) {
                    const double m = lanes_max<LANES>(wide);
                    if (wins(wide > -INFINITY, wide, m) && r < places) {
                        kept = true;
                        wide = -INFINITY;
                    }
                }
            }
        }
        each([&](int, K &k) { k = kept ? k : NONE; });
    }
    const int slots = APPROX ? MAX_CANDIDATES : a.copies;
    for (int i = w.lane; i < slots; i += LANES) chosen[i] = -1;
    wave_sync();
    int found = 0;
    bool close = false;                            // keys so near that their order may be another
    if constexpr (sizeof(K) == 4) {
        // Keys by whole numbers in their order, the expert's place in the last bits, where
        // the larger is the earlier: a lane's are all different, and the next one after m is
        // where m - 1 - k is the least, which for a key already taken wraps around to more
        // than for any other: a subtraction and half a minimum a key and round.  16-bit
        // logits leave the last 13 bits free, which hold the expert's number: equal ones are
        // in order over all lanes.
        constexpr bool FREE = !APPROX;
        constexpr uint32_t PLACE = FREE ? 4095 : PER ? PER - 1 : 127, GONE = 0, LIVE = 0x00800000;        // of -infinity, less
        static_assert(MAX_EXPERTS <= 4095, "a number in 12 bits");
        const float near_by = apart + 4 * (PLACE + 1) * 0x1p-24f;      // and what the bits took from two keys
        uint32_t packed[HELD];
        auto pass = [&](auto &&f) {
            if constexpr (PER > 0) {
#pragma unroll
                for (int j = 0; j < PER; ++j) f(packed[j]);
            } else {
                const uint32_t *keys = (const uint32_t *)lds + w.lane;
                for (int j = 0; j < a.per; ++j) f(keys[j * 64]);
            }
        };
        each([&](int j, K &k) {
            const int bits = __builtin_bit_cast(int, ROUGH ? k : k + K(0));        // -0 is 0, as near as it gets
            const uint32_t p = (uint32_t)((bits ^ (bits >> 31 | INT32_MIN)) & ~PLACE) + (PLACE - j - (FREE ? w.first : 0));
            if constexpr (PER > 0) packed[j] = p;
            else k = __builtin_bit_cast(float, p);
        });
        uint32_t best = GONE;
        pass([&](uint32_t k) { best = k > best ? k : best; });
        auto value = [&](uint32_t m) {
            const int bits = (int)(m & ~PLACE);
            return __builtin_bit_cast(float, bits ^ (~(bits >> 31) | INT32_MIN));
        };
        auto near = [&](uint32_t last, uint32_t m) {
            if constexpr (ROUGH) {
                const float v = value(last);
                return m >= LIVE && !(v - value(m) > near_by * (1 + fabsf(v)));
            } else {
                return APPROX && m >= LIVE && (m | PLACE) == (last | PLACE);
            }
        };
        auto take = [&](int r, uint32_t m) {
            chosen[r] = (FREE ? 0 : w.first) + (int)(PLACE - (m & PLACE));
            uint32_t least = UINT32_MAX;
            pass([&](uint32_t k) { least = m - 1 - k < least ? m - 1 - k : least; });
            best = m - 1 - least;
            best = best < m ? best : GONE;
        };
        uint32_t m = lanes_max<LANES>(best), last = GONE;
        for (int r = 0; r < a.copies; ++r) {
            found += m >= LIVE;
            if (first_of(best == m && m >= LIVE, before)) take(r, m);
            last = m;
            m = lanes_max<LANES>(best);
            close |= near(last, m);
        }
        // Past the last one asked for: those as near to it.
        if (APPROX && __ballot(close) && !(ROUGH && softmax))
            for (int r = a.copies;; ++r) {
                const bool more = near(last, m);
                if (__ballot(more) == 0) break;
                if (r == slots) {
                    unsure |= more;
                    break;
                }
                found += more;
                if (first_of(best == m && more, before)) take(r, m);
                m = lanes_max<LANES>(best);
            }
    } else {
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
            if (first_of(best == m && m > NONE, before)) {
                chosen[r] = w.first + at;
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
    }
    if constexpr (APPROX) {
        if (ROUGH && softmax) return unsure || close;
        // The experts' order in 64 bits: one's place is how many come before it.
        if (__ballot(close)) {
            wave_sync();
#pragma unroll 1
            for (int i = w.lane; i < found; i += LANES)
                exact[i] = ROUGH ? 1 / (1 + exp(-(double)A(L[chosen[i]]))) + (double)bias[chosen[i]] : (double)A(L[chosen[i]]);
            wave_sync();
            int *order = (int *)(exact + MAX_CANDIDATES);
#pragma unroll 1
            for (int i = w.lane; i < found; i += LANES) {
                const double key = exact[i];
                const int e = chosen[i];
                int ahead = 0;
                for (int j = 0; j < found; ++j) ahead += exact[j] > key || (exact[j] == key && chosen[j] < e);
                order[ahead] = e;
            }
            wave_sync();
#pragma unroll 1
            for (int i = w.lane; i < found; i += LANES) chosen[i] = order[i];
        }
    }
    return unsure;
}

// BIASED: keys are scores plus biases, Float64, else the logits.  But for Float64 logits,
// and 16-bit ones without a bias, they are Float32 first, and Float64 for a column that
// those do not settle.
template <typename T, bool BIASED, int LANES, int PER>
__global__ __launch_bounds__(PER ? 256 : 64, PER == 0 ? 1 : LANES == 64 ? 3 : 4) void route_kernel(const RouteArgs a)
{
    using A = typename Elem<T>::Acc;
    constexpr int NT = PER ? 256 : 64, COLS = NT / LANES, NP = MAX_COPIES / LANES;
    __shared__ int s_chosen[COLS][MAX_CANDIDATES];
    constexpr bool APPROX = BIASED ? sizeof(T) < 8 : sizeof(T) == 4;
    __shared__ double s_exact[APPROX ? COLS : 1][MAX_CANDIDATES * 3 / 2];
    extern __shared__ double s_keys[];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES, of_group = 1 << a.lane_shift;
    const int group = lane >> a.lane_shift, place = (lane & (of_group - 1)) * a.per;
    const bool softmax = a.score == JLUST_SCORE_SOFTMAX;
    const int64_t c0 = (int64_t)blockIdx.x * COLS;
    const int64_t c = c0 + sub;
    const T *L = (const T *)a.L + (c < a.cols ? c : a.cols - 1) * a.ldl;
    int count = a.size - place < a.per ? a.size - place : a.per;
    if (group >= a.groups || c >= a.cols || count < 0) count = 0;
    const RouteShare w{lane, group, count ? group * a.size + place : 0, count};
    double top, total;
    if constexpr (!APPROX) {
        choose<T, A, false, BIASED, LANES, PER>(a, w, L, (char *)s_keys, s_chosen[sub], nullptr, &top, &total);
    } else {
        const bool unsure = choose<T, float, true, BIASED, LANES, PER>(a, w, L, (char *)s_keys, s_chosen[sub], s_exact[sub], &top, &total);
        uint64_t open = __ballot(unsure && lane == 0);
        // A wave takes each such column: its registers hold Float64 keys of four lanes.
        while (open) {
            const int at = __ffsll((unsigned long long)open) - 1, theirs = (threadIdx.x & ~63) / LANES + at / LANES;
            open &= open - 1;
            constexpr int WIDE = LANES == 64 ? PER : PER > 4 ? PER / 4 : 1;
            RouteArgs b = a;
            b.lane_shift += LANES == 64 ? 0 : 2;
            b.per = (a.size + (1 << b.lane_shift) - 1) >> b.lane_shift;
            b.whole = b.per == WIDE && a.size % b.per == 0;
            const int mine = threadIdx.x & 63, g = mine >> b.lane_shift, from = (mine & ((1 << b.lane_shift) - 1)) * b.per;
            int some = a.size - from < b.per ? a.size - from : b.per;
            if (g >= a.groups || some < 0) some = 0;
            double m, all;
            wave_sync();
            choose<T, double, false, BIASED, 64, WIDE>(b, RouteShare{mine, g, some ? g * a.size + from : 0, some}, (const T *)a.L + (c0 + theirs) * a.ldl,
                                               (char *)s_keys, s_chosen[theirs], nullptr, &m, &all);
            if (sub == theirs) {
                top = m;
                total = all;
            }
        }
    }
    wave_sync();
    A l[NP], p[NP];
    int e[NP];
    const int parts = (a.copies + LANES - 1) / LANES;
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
        chosen_scores<LANES>(a.score, a.renormalize, parts, l, p);
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) sum += p[q];
    sum = a.renormalize ? lanes_sum<LANES>(sum) : A(1);
    if (c >= a.cols) return;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        const int i = lane + q * LANES;
        if (q >= parts || i >= a.copies) continue;
        a.ids[c * a.ldi + i] = e[q] + a.origin;
        ((A *)a.weights)[c * a.ldw + i] = e[q] >= 0 ? A(a.scale * (double)(p[q] / sum)) : A(0);
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
    if constexpr (sizeof(T) == 2) {
        const A v = __expf(l - top);
        return l == top ? A(1) : v;
    } else {
        return exp_below(l, top);
    }
}

// With t = scale dw and p the weights' shares of the chosen: softmax renormalised
// p (t - sum p t), sigmoid renormalised the same times 1 - s, sigmoid t s (1 - s) at the
// chosen and 0 elsewhere; softmax as it is s_e (t_e - sum s t) everywhere.  LANES lanes
// take a column, CPL chunks of 16 bytes each in registers, so logits are read once (CPL
// 0: any number, read again).  What goes to the chosen passes through a row of LDS; asking
// of every element which of the chosen it is took 23.1 us for 13,433 Float32 columns of
// 298 with 14 chosen, 12.5 so (160 bfloat16 experts, 6 chosen: 7.9 and 6.7).
template <typename T, bool WHOLE, int LANES, int CPL>
__global__ __launch_bounds__(256) void route_grad_kernel(const RouteGradArgs a)
{
    constexpr int CH = 16 / sizeof(T), HELD = CPL ? CPL : 1;
    using A = typename Elem<T>::Acc;
    constexpr int COLS = 256 / LANES, NP = MAX_COPIES / LANES;
    __shared__ int s_expert[COLS][MAX_COPIES];
    __shared__ A s_part[COLS][MAX_COPIES];
    __shared__ __align__(16) A s_row[CPL ? COLS : 1][CPL ? LANES * CPL * CH : 1];      // the parts at their experts
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const bool softmax = a.score == JLUST_SCORE_SOFTMAX, dense = softmax && !a.renormalize;
    const int64_t c0 = (int64_t)blockIdx.x * COLS;
    const int64_t c = c0 + sub;
    const bool live = c < a.cols;
    const T *L = (const T *)a.L + c * a.ldl;
    A top = -INFINITY, total = A(0), s[HELD][CH];
    if (CPL > 0 && dense) {
        uint32x4 raw[HELD];
#pragma unroll
        for (int i = 0; i < CPL; ++i)
            raw[i] = read_at<WHOLE>((const T *)a.L + (live ? c : a.cols - 1) * a.ldl, (lane + LANES * i) * CH, a.experts);
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            values<T>(raw[i], s[i]);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const bool some = (lane + LANES * i) * CH + (WHOLE ? 0 : j) < a.experts && s[i][j] > A(-INFINITY);
                s[i][j] = some ? s[i][j] : A(-INFINITY);
                top = s[i][j] > top ? s[i][j] : top;
            }
        }
        top = lanes_max<LANES>(top);
#pragma unroll
        for (int i = 0; i < CPL; ++i)
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const A v = score_below<T>(s[i][j], top);
                s[i][j] = s[i][j] > A(-INFINITY) ? v : A(0);
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
    const int parts = (a.copies + LANES - 1) / LANES;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        const int i = lane + q * LANES;
        at[q] = -1;
        l[q] = -INFINITY;
        t[q] = A(0);
        if (q < parts && live && i < a.copies) {
            const int64_t e = (int64_t)a.ids[c * a.ldi + i] - a.origin;
            if (e >= 0 && e < a.experts) {
                at[q] = (int)e;
                const A v = A(L[e]);
                l[q] = v > A(-INFINITY) ? v : A(-INFINITY);        // of NaN too the score is 0
                t[q] = A(a.scale * (double)((const A *)a.dw)[c * a.lddw + i]);
            }
        }
    }
    A sum = A(0), dot = A(0);
    if (dense) {
#pragma unroll
        for (int q = 0; q < NP; ++q) p[q] = q < parts && l[q] > A(-INFINITY) ? exp_below(l[q], top) / total : A(0);
    } else {
        chosen_scores<LANES>(a.score, a.renormalize, parts, l, p);
        if (a.renormalize) {
#pragma unroll
            for (int q = 0; q < NP; ++q) sum += p[q];
            sum = lanes_sum<LANES>(sum);
#pragma unroll
            for (int q = 0; q < NP; ++q) p[q] = q < parts && p[q] > A(0) ? p[q] / sum : A(0);
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
        if (q >= parts || i >= a.copies) continue;
        A g = dense ? t[q] : p[q] * (t[q] - dot);
        if (!softmax) g *= A(1) / (A(1) + exp_of(l[q]));
        s_expert[sub][i] = at[q];
        s_part[sub][i] = at[q] >= 0 ? g : A(0);
    }
    if constexpr (CPL > 0) {
        A none[CH] = {};
#pragma unroll
        for (int i = 0; i < CPL; ++i) __builtin_memcpy(&s_row[sub][(lane + LANES * i) * CH], none, sizeof(none));
    }
    wave_sync();
    if constexpr (CPL > 0) {
        // An expert that is named twice gets both parts, the same sum from either.
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            if (q >= parts || at[q] < 0) continue;
            A g = A(0);
            for (int k = 0; k < a.copies; ++k) g += s_expert[sub][k] == at[q] ? s_part[sub][k] : A(0);
            s_row[sub][at[q]] = g;
        }
        wave_sync();
        const A inv = total > A(0) ? A(1) / total : A(0);
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            const int at = (lane + LANES * i) * CH;
            A g[CH];
            __builtin_memcpy(g, &s_row[sub][at], sizeof(g));
            if (dense) {
#pragma unroll
                for (int j = 0; j < CH; ++j) g[j] = s[i][j] * inv * (g[j] - dot);
            }
            if (live) write_at<WHOLE>((T *)a.dL + c * a.lddl, at, a.experts, g);
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

// launch(a, blocks) for the columns of `a`, `each` a workgroup: a workgroup that walked
// over several would hold what it asks of its arguments in registers over the walk
// (16,384 columns of 256 experts in 8 groups: 18.0 us and 13.6), so past the columns of
// 2^21 workgroups another launch follows.
template <typename T, typename Args, typename F>
int by_launches(Args a, int64_t each, F &&launch)
{
    using A = typename Elem<T>::Acc;
    const int64_t most = ((int64_t)1 << 21) * each, cols = a.cols;
    for (int64_t c = 0; c < cols; c += most) {
        a.cols = cols - c < most ? cols - c : most;
        if (int st = launch(a, (unsigned)((a.cols + each - 1) / each))) return st;
        a.L = (const T *)a.L + most * a.ldl;
        a.ids += most * a.ldi;
        if constexpr (std::is_same_v<Args, RouteArgs>) {
            a.weights = (A *)a.weights + most * a.ldw;
        } else {
            a.dw = (const A *)a.dw + most * a.lddw;
            a.dL = (T *)a.dL + most * a.lddl;
        }
    }
    return JLUST_STATUS_SUCCESS;
}

template <typename T, bool BIASED, int LANES, int PER>
int launch_route(RouteArgs a, hipStream_t s)
{
    constexpr int NT = PER ? 256 : 64;
    a.whole = a.per == PER && a.size % (PER ? PER : 1) == 0;
    return by_launches<T>(a, NT / LANES, [&](const RouteArgs &some, unsigned blocks) {
        hipLaunchKernelGGL((route_kernel<T, BIASED, LANES, PER>), dim3(blocks), dim3(NT),
                           PER ? 0 : (BIASED || sizeof(T) >= 4 ? sizeof(double) : sizeof(float)) * 64 * a.per, s, some);
        return check_launch("route_kernel");
    });
}

// 16 lanes a column where it fits them and the columns fill the CUs (a round of the
// best key then serves four columns), else a wave (us by a wave and by 16 lanes, sigmoids
// with a bias: 256 experts in 8 groups 7.0 and 7.6 for 2,048 columns, 9.2 and 7.8 for 4,096,
// 23.1 and 12.4 for 16,384; 64 experts 5.1 and 5.4, 5.7 and 5.2, 12.8 and 6.4).
template <typename T, bool BIASED>
int route(RouteArgs a, hipStream_t s)
{
    if (a.cols > ROUTE_FEW && route_lanes(16, &a) && a.per <= 16) {
        if (a.per <= 1) return launch_route<T, BIASED, 16, 1>(a, s);
        if (a.per <= 2) return launch_route<T, BIASED, 16, 2>(a, s);
        if (a.per <= 4) return launch_route<T, BIASED, 16, 4>(a, s);
        if (a.per <= 8) return launch_route<T, BIASED, 16, 8>(a, s);
        return launch_route<T, BIASED, 16, 16>(a, s);
    }
    route_lanes(64, &a);
    if (a.per <= 1) return launch_route<T, BIASED, 64, 1>(a, s);
    if (a.per <= 2) return launch_route<T, BIASED, 64, 2>(a, s);
    if (a.per <= 4) return launch_route<T, BIASED, 64, 4>(a, s);
    if (a.per <= 8) return launch_route<T, BIASED, 64, 8>(a, s);
    if (a.per <= 16) return launch_route<T, BIASED, 64, 16>(a, s);
    return launch_route<T, BIASED, 64, 0>(a, s);
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
        return a.bias ? route<T, true>(a, (hipStream_t)stream) : route<T, false>(a, (hipStream_t)stream);
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
            return by_launches<T>(a, 256 / lanes, [&](const RouteGradArgs &some, unsigned blocks) {
                hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, some);
                return check_launch("route_grad_kernel");
            });
        };
        auto go = [&](auto whole) {
            constexpr bool W = decltype(whole)::value;
            if (chunks <= 16) return launch(route_grad_kernel<T, W, 16, 1>, 16);
            if (chunks <= 32) return launch(route_grad_kernel<T, W, 16, 2>, 16);
            if (chunks <= 64) return launch(route_grad_kernel<T, W, 16, 4>, 16);
            if (chunks <= 256) return launch(route_grad_kernel<T, W, 64, 4>, 64);
            return launch(route_grad_kernel<T, W, 64, 0>, 64);
        };
        return a.experts % (16 / sizeof(T)) == 0 ? go(std::true_type()) : go(std::false_type());
    });
}

namespace jlust {
int preload_route()
{
    JLUST_PRELOAD_KERNEL((route_kernel<float, true, 64, 4>));
    return JLUST_STATUS_SUCCESS;
}
}  // namespace jlust
