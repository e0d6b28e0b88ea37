// linear.hip -- a layer's dense products, Y = act.(W*X .+ b) .+ R, with one W or
// one per group of columns, and their gradients; the plan that sorts the columns
// by group.  The products run in tile_kernel.hpp; here are their arguments, the
// gradient's first pass over dY, and the small sums.
#include <initializer_list>

#include "tile_product.hpp"
#include "wave.hpp"

namespace jlust {
namespace {

// ---------------------------------------------------------------- group plans

constexpr int64_t MAX_GROUPS = 4095;           // 4 waves' counters of a workgroup fit 64 KB of LDS
constexpr int PLAN_WAVES = 4;                  // of a workgroup of the plan kernels on many columns
constexpr int PLAN_ROUNDS = 4;                 // of 64 ids a wave holds in registers
constexpr int SMALL_WAVES = 16, SMALL_ROUNDS = 4;
constexpr int64_t SMALL_COLUMNS = SMALL_WAVES * SMALL_ROUNDS * 64, SMALL_GROUPS = 1000;
constexpr int64_t SCAN_COUNTS = 1 << 16;       // that one workgroup scans

// The bin of column p: its group, `groups` if it names none.
__device__ __forceinline__ int bin_of(const void *ids, int ids64, int64_t p, int origin, int groups)
{
    const int64_t id = (ids64 ? ((const int64_t *)ids)[p] : (int64_t)((const int32_t *)ids)[p]) - origin;
    return id >= 0 && id < groups ? (int)id : groups;
}

// The lanes of the wave that hold the same bin as this one (bits: those of a
// bin); lanes without one pass active = false and get 0.
__device__ __forceinline__ uint64_t same_bin(int bin, bool active, int bits)
{
    uint64_t mask = __ballot(active);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot(bin >> b & 1);
        mask &= bin >> b & 1 ? set : ~set;
    }
    return active ? mask : 0;
}

// A wave's ids, 64 a round, all read before the first is used (a round of its own
// reads took 0.7 us): the bins of [p0, p1), -1 past the end.
template <int ROUNDS>
__device__ __forceinline__ void read_bins(const void *ids, int ids64, int64_t p0, int64_t p1, int origin, int groups,
                                          int (&bin)[ROUNDS])
{
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t p = p0 + r * 64 + lane_id();
        bin[r] = p < p1 ? bin_of(ids, ids64, p, origin, groups) : -1;
    }
}

// Counts them, or (PLACE) writes every column at its bin's next place: a column's
// place among its own 64 by the lanes before it, so equal bins keep their order.
template <bool PLACE, int ROUNDS>
__device__ __forceinline__ void walk_bins(const int (&bins)[ROUNDS], int64_t p0, int bits, int32_t *cnt, int32_t *perm,
                                          int32_t *src, int copies)
{
    const int lane = lane_id();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool active = bins[r] >= 0;
        if (__ballot(active) == 0) break;
        const int bin = active ? bins[r] : 0;
        const uint64_t mask = same_bin(bin, active, bits);
        const int before = __popcll(mask & ((1ull << lane) - 1));
        const int at = active ? cnt[bin] : 0;
        wave_sync();
        if (active && before == 0) cnt[bin] = at + __popcll(mask);
        wave_sync();
        if (PLACE && active) {
            const int64_t p = p0 + r * 64 + lane;
            perm[at + before] = (int32_t)p;
            if (src) src[at + before] = (int32_t)(p / copies);
        }
    }
}

// The whole plan in one workgroup: a few columns cost a launch, not six.
__global__ __launch_bounds__(SMALL_WAVES * 64) void group_plan_small_kernel(int64_t n, int groups, int copies, int origin,
                                                                            const void *ids, int ids64, int bits,
                                                                            int32_t *offsets, int32_t *perm, int32_t *src)
{
    extern __shared__ int32_t cnt[];               // [waves][groups + 1]
    __shared__ int32_t waves[SMALL_WAVES + 1];
    const int wave = threadIdx.x >> 6, bins = groups + 1;
    for (int i = threadIdx.x; i < SMALL_WAVES * bins; i += SMALL_WAVES * 64) cnt[i] = 0;
    __syncthreads();
    const int64_t per = ((n + SMALL_WAVES - 1) / SMALL_WAVES + 63) / 64 * 64;
    const int64_t p0 = per * wave < n ? per * wave : n, p1 = p0 + per < n ? p0 + per : n;
    int bin[SMALL_ROUNDS];
    read_bins(ids, ids64, p0, p1, origin, groups, bin);
    walk_bins<false>(bin, p0, bits, cnt + wave * bins, nullptr, nullptr, 1);
    __syncthreads();
    // bins <= 1,024: one a thread.
    const int b = threadIdx.x, lane = lane_id();
    int32_t total = 0;
    if (b < bins)
        for (int w = 0; w < SMALL_WAVES; ++w) total += cnt[w * bins + b];
    int32_t incl = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int32_t t = __shfl_up(incl, d, 64);
        if (lane >= d) incl += t;
    }
    if (lane == 63) waves[wave] = incl;
    __syncthreads();
    if (b < bins) {
        int32_t run = incl - total;
        for (int w = 0; w < wave; ++w) run += waves[w];
        offsets[b] = run;
        for (int w = 0; w < SMALL_WAVES; ++w) {
            const int32_t c = cnt[w * bins + b];
            cnt[w * bins + b] = run;
            run += c;
        }
    }
    __syncthreads();
    walk_bins<true>(bin, p0, bits, cnt + wave * bins, perm, src, copies);
}

// Many columns: counts[bin][run] of a wave's runs of columns, which a scan turns
// into each run's first place in every bin.  More groups have longer runs, so that
// the counts stay below the ids.
template <bool PLACE>
__global__ __launch_bounds__(PLAN_WAVES * 64) void group_plan_kernel(int64_t n, int groups, int copies, int origin,
                                                                     const void *ids, int ids64, int bits, int64_t runs, int per,
                                                                     int32_t *counts, int32_t *offsets, int32_t *perm,
                                                                     int32_t *src)
{
    extern __shared__ int32_t cnt[];
    const int wave = threadIdx.x >> 6, lane = lane_id(), bins = groups + 1;
    const int64_t run = (int64_t)blockIdx.x * PLAN_WAVES + wave;
    int32_t *mine = cnt + wave * bins;
    for (int b = lane; b < bins; b += 64) mine[b] = PLACE && run < runs ? counts[b * runs + run] : 0;
    __syncthreads();
    const int64_t p0 = run * per < n ? run * per : n, p1 = p0 + per < n ? p0 + per : n;
    if (PLACE && run == 0)
        for (int b = lane; b < bins; b += 64) offsets[b] = counts[b * runs];
    for (int64_t p = p0; p < p1; p += PLAN_ROUNDS * 64) {
        int bin[PLAN_ROUNDS];
        read_bins(ids, ids64, p, p1, origin, groups, bin);
        walk_bins<PLACE>(bin, p, bits, mine, perm, src, copies);
    }
    __syncthreads();
    if (!PLACE && run < runs)
        for (int b = lane; b < bins; b += 64) counts[b * runs + run] = mine[b];
}

// Exclusive scan of n counts in one workgroup, 4 a thread and round.
__global__ __launch_bounds__(1024) void group_scan_kernel(int n, int32_t *counts)
{
    __shared__ int32_t s_wave[16];
    const int wave = threadIdx.x >> 6, lane = lane_id();
    int32_t base = 0;
    for (int i0 = 0; i0 < n; i0 += 4096) {
        const int i = i0 + (int)threadIdx.x * 4;
        int32_t v[4], sum = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = i + e < n ? counts[i + e] : 0;
            sum += v[e];
        }
        int32_t incl = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int32_t t = __shfl_up(incl, d, 64);
            if (lane >= d) incl += t;
        }
        __syncthreads();
        if (lane == 63) s_wave[wave] = incl;
        __syncthreads();
        int32_t run = base + incl - sum;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            if (w < wave) run += s_wave[w];
            base += s_wave[w];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i + e < n) counts[i + e] = run;
            run += v[e];
        }
    }
}

int check_groups(const char *who, int64_t n, int64_t groups, int64_t copies)
{
    if (n < 0 || n >= (int64_t)1 << 31)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %lld columns are not within [0, 2^31)", who, (long long)n);
    if (groups < 1 || groups > MAX_GROUPS)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %lld groups are not within [1, %lld]", who, (long long)groups,
                    (long long)MAX_GROUPS);
    if (copies < 1 || copies >= (int64_t)1 << 31 || n % copies)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %lld columns are not %lld copies of some", who, (long long)n,
                    (long long)copies);
    return JLUST_STATUS_SUCCESS;
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

// ------------------------------------------------------- the gradient's first pass

// Runs of rows that one workgroup takes; 256 threads are 32 vectors along m by
// 8 rows.
template <typename T>
struct Prepass {
    static constexpr int V = 16 / sizeof(T), COLS = 32 * V;
};

// G = dY .* act'(Z) in the order of the groups (row p of G is column perm[p]),
// rounded to T, its rows ldg apart (a whole number of 16 bytes, zeros at their ends),
// and the sums of its unrounded rows over a run of `per` columns: sums[run][m].  dY
// and Z are read once; G and dbias would each read them again.
// The rounding is one to the type of dY, W and X, which the 16-bit matrix steps take:
// the results' error goes from 0.0017 to 0.0023 in bfloat16.  G as the sum of two
// 16-bit values would take both products twice (8,192 columns 2048 -> 8192: dX 248 us
// and 486, dW 230 and 460, of 566 in all); Float32 operands, which a caller who needs
// more can pass, take 4,257.
template <typename T>
__global__ __launch_bounds__(256) void grad_prepass_kernel(int64_t n, int64_t m, const T *__restrict__ dY, int64_t lddy,
                                                           const T *__restrict__ Z, int64_t ldz, int act, T *__restrict__ G,
                                                           int64_t ldg, const int32_t *__restrict__ offsets,
                                                           const int32_t *__restrict__ perm, int groups, int per, int blocks_m,
                                                           typename Elem<T>::Acc *__restrict__ sums)
{
    using A = typename Elem<T>::Acc;
    constexpr int V = Prepass<T>::V, COLS = Prepass<T>::COLS;
    __shared__ A s_sum[8][COLS + 1];
    const int64_t run = blockIdx.x / blocks_m;
    const int64_t m0 = (int64_t)(blockIdx.x % blocks_m) * COLS;
    GroupRun r;
    if (offsets) {
        if (!find_run(offsets, groups, n, run, per, &r) || r.group == groups) return;
    } else {
        r.begin = run * per;
        r.end = r.begin + per < n ? r.begin + per : n;
    }
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = m0 + (int64_t)tx * V, left = m - c;
    A acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = A(0);
    if (left > 0)
        for (int64_t p = r.begin + ty; p < r.end; p += 8) {
            const int64_t col = perm ? (int64_t)perm[p] : p;
            T y[V], z[V];
            const uint32x4 vy = left >= V ? load_chunk(dY + col * lddy + c) : load_chunk_part(dY + col * lddy + c, left);
            __builtin_memcpy(y, &vy, 16);
            if (Z) {
                const uint32x4 vz = left >= V ? load_chunk(Z + col * ldz + c) : load_chunk_part(Z + col * ldz + c, left);
                __builtin_memcpy(z, &vz, 16);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                A g = A(y[e]);
                if (Z) g *= activate_slope<sizeof(T) == 2>(act, A(z[e]));
                acc[e] += g;
                y[e] = T(g);
            }
            if (G) store_vec<V>(G + p * ldg + c, y);           // zeros past m
        }
    if (!sums) return;
#pragma unroll
    for (int e = 0; e < V; ++e) s_sum[ty][tx * V + e] = acc[e];
    __syncthreads();
    for (int i = threadIdx.x; i < COLS; i += 256) {
        A s = A(0);
#pragma unroll
        for (int q = 0; q < 8; ++q) s += s_sum[q][i];
        if (m0 + i < m) sums[run * m + m0 + i] = s;
    }
}

// A launch takes fewer than 2^32 threads (of more it runs their number modulo 2^32,
// without an error): at most 2^21 workgroups, which walk over the items in turn.
unsigned blocks_for(int64_t items, int64_t each)
{
    const int64_t blocks = (items + each - 1) / each;
    return (unsigned)(blocks < 1 << 21 ? blocks : 1 << 21);
}

// Rows src[idx[p]] (or src[p]) of `len` values for p < rows (or offsets[groups]) of
// each of the blockIdx.y matrices, `stride` apart, 16-byte aligned and `ld` apart,
// zeros at their ends: what the copies of tile_kernel.hpp take.
template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(int64_t rows, int64_t len, const T *__restrict__ src, int64_t lds_,
                                                        int64_t stride, const int32_t *__restrict__ idx,
                                                        const int32_t *__restrict__ limit, T *__restrict__ out, int64_t ld)
{
    constexpr int V = 16 / sizeof(T);
    const int64_t end = limit && *limit < rows ? *limit : rows;
    // 32 chunks along a row by 8 rows.
    for (int64_t p = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); p < end; p += (int64_t)gridDim.x * 8) {
        const T *from = src + blockIdx.y * stride + (idx ? (int64_t)idx[p] : p) * lds_;
        T *to = out + (blockIdx.y * rows + p) * ld;
        for (int64_t c = (int64_t)(threadIdx.x & 31) * V; c < ld; c += 32 * V) {
            const int64_t left = len - c;
            const T *q = from + c;
            const uint32x4 v = left >= V ? load_chunk(q) : load_chunk_part(q, left);
            __builtin_memcpy(to + c, &v, 16);
        }
    }
}

template <typename T>
int pack_rows(int64_t rows, int64_t len, const void *src, int64_t lds, int64_t matrices, int64_t stride, const int32_t *idx,
              const int32_t *limit, void *out, int64_t ld, hipStream_t s)
{
    if (rows == 0 || ld == 0) return JLUST_STATUS_SUCCESS;
    hipLaunchKernelGGL((pack_rows_kernel<T>), dim3(blocks_for(rows, 8), (unsigned)matrices), dim3(256), 0, s, rows, len,
                       (const T *)src, lds, stride, idx, limit, (T *)out, ld);
    return check_launch("pack_rows_kernel");
}

// The matrices that groups' packed weights take: one where the groups share it.
int64_t packed_matrices(int64_t groups, int64_t w_stride) { return groups && w_stride ? groups : 1; }

template <typename T>
int64_t padded(int64_t len)
{
    constexpr int64_t V = 16 / sizeof(T);
    return (len + V - 1) / V * V;
}

// Whether rows of `len` values can be copied to LDS as they lie.
template <typename T>
bool lies_well(const void *p, int64_t len, int64_t ld, int64_t stride)
{
    return (((uintptr_t)p | (uintptr_t)(len * sizeof(T)) | (uintptr_t)(ld * sizeof(T)) | (uintptr_t)(stride * sizeof(T))) & 15) == 0;
}

// Whether operands of `values` values are better packed first: the product through
// registers runs at 550 Tflop/s where rows along its sides lie badly and 800 where rows
// along k do, at 1,000 from copies (8,191 columns 2047 -> 8191: 482 and 334 us against
// 257), Float32's at 108 against 127 (8,191 columns 2047 -> 2047: 636 us and 558; 4,600
// columns 1001 -> 1001: 126 and 131).  Packing reads and writes them at 3 TB/s.
// Float32 with k of 256 and less runs through registers all the same.
template <typename T>
bool worth_packing(int64_t m, int64_t n, int64_t k, int64_t values, bool sides)
{
    if (sizeof(T) > 4 || values == 0 || (sizeof(T) == 4 && k <= 256)) return false;
    const double gain = sizeof(T) == 4 ? 1 / 108.0 - 1 / 127.0 : sides ? 1 / 550.0 - 1 / 1000.0 : 1 / 800.0 - 1 / 1000.0;
    return 2e-6 * m * n * k * gain > 3 + values * (sizeof(T) * 0.65e-6);
}

// dbias of a group: the sums of its runs, in order; 32 m by LANES runs at a time (8
// where groups have few: 13 us by 32 and 5 by 8 for 32 groups of 8 runs).
template <typename T, int LANES>
__global__ __launch_bounds__(32 * LANES) void grad_bias_kernel(int64_t n, int64_t m, const int32_t *__restrict__ offsets, int per,
                                                         const typename Elem<T>::Acc *__restrict__ sums, T *__restrict__ dbias,
                                                         int64_t stride)
{
    using A = typename Elem<T>::Acc;
    __shared__ A s_sum[LANES][33];
    __shared__ int64_t s_first;
    const int group = blockIdx.y, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    int64_t first = 0, count = (n + per - 1) / per;
    if (offsets) {
        if (threadIdx.x < 64) {                    // the runs of the groups before
            int64_t before = 0;
            for (int g = lane_id(); g < group; g += 64) before += (offsets[g + 1] - offsets[g] + per - 1) / per;
            for (int d = 32; d; d >>= 1) before += __shfl_xor(before, d, 64);
            if (threadIdx.x == 0) s_first = before;
        }
        __syncthreads();
        first = s_first;
        count = (offsets[group + 1] - offsets[group] + per - 1) / per;
    }
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < m; c0 += (int64_t)gridDim.x * 32) {
        const int64_t c = c0 + tx;
        A s = A(0);
        if (c < m) {
#pragma unroll 8
            for (int64_t i = ty; i < count; i += LANES) s += sums[(first + i) * m + c];
        }
        __syncthreads();
        s_sum[ty][tx] = s;
        __syncthreads();
        if (ty == 0 && c < m) {
            A t = A(0);
#pragma unroll
            for (int q = 0; q < LANES; ++q) t += s_sum[q][tx];
            dbias[group * stride + c] = T(t);
        }
    }
}

// dX's column t: the sum of its copies' columns of the product.
template <typename T>
__global__ __launch_bounds__(256) void sum_copies_kernel(int64_t cols, int64_t d, int copies,
                                                         const typename Elem<T>::Acc *__restrict__ src, T *__restrict__ dX,
                                                         int64_t ldx)
{
    using A = typename Elem<T>::Acc;
    constexpr int V = 4;
    const int64_t per = (d + V - 1) / V;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < cols * per; at += (int64_t)gridDim.x * 256) {
        const int64_t t = at / per, c = (at - t * per) * V;
        const A *p = src + t * copies * d + c;
        if (c + V <= d) {
            A s[V] = {0, 0, 0, 0};
            T o[V];
            for (int q = 0; q < copies; ++q, p += d) {
                A v[V];
                load_vec<V>(p, v);
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] += v[e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = T(s[e]);
            store_vec<V>(dX + t * ldx + c, o);
            continue;
        }
        for (int e = 0; c + e < d; ++e) {
            A v = A(0);
            for (int q = 0; q < copies; ++q) v += p[q * d + e];
            dX[t * ldx + c + e] = T(v);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void fill_zero_kernel(int64_t rows, int64_t d, T *__restrict__ out, int64_t ld)
{
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < rows * d; at += (int64_t)gridDim.x * 256)
        out[at / d * ld + at % d] = T(0);
}

template <typename T>
int fill_zero(int64_t rows, int64_t d, void *out, int64_t ld, hipStream_t s)
{
    if (rows * d == 0) return JLUST_STATUS_SUCCESS;
    hipLaunchKernelGGL((fill_zero_kernel<T>), dim3(blocks_for(rows * d, 256)), dim3(256), 0, s, rows, d, (T *)out, ld);
    return check_launch("fill_zero_kernel");
}

// ---------------------------------------------------------------------- checks

struct Operand { const char *name; const void *p; int64_t rows, cols, ld; bool needed; };

int check_operands(const char *who, std::initializer_list<Operand> ops)
{
    for (const Operand &o : ops) {
        const bool empty = o.rows == 0 || o.cols == 0;
        if (!o.p) {
            if (o.needed && !empty) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %s is null", who, o.name);
            continue;
        }
        if (o.cols > 1 && o.ld < o.rows)
            return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %s has leading dimension %lld, its columns %lld rows", who,
                        o.name, (long long)o.ld, (long long)o.rows);
    }
    return JLUST_STATUS_SUCCESS;
}

// The matrices of a result's groups must not share memory: each lies behind the one
// before, or all of them within one's leading dimension.
int check_apart(const char *who, const char *name, const void *p, int64_t rows, int64_t cols, int64_t ld, int64_t groups,
                int64_t stride)
{
    if (!p || groups < 2 || rows == 0 || cols == 0) return JLUST_STATUS_SUCCESS;
    const int64_t by = stride < 0 ? -stride : stride;
    const bool behind = by >= (cols > 1 ? (cols - 1) * ld : 0) + rows, within = by >= rows && ld >= (groups - 1) * by + rows;
    if (behind || within) return JLUST_STATUS_SUCCESS;
    return fail(JLUST_STATUS_NONCANONICAL_STORAGE, "%s: the groups' matrices of %s overlap (%lld x %lld, leading dimension %lld, "
                "%lld elements from one to the next)", who, name, (long long)rows, (long long)cols, (long long)ld, (long long)stride);
}

int check_common(const char *who, int32_t value_type, int32_t act, int32_t w_layout, int64_t out, int64_t inp, int64_t cols,
                 int64_t groups, int64_t copies, const int32_t *plan)
{
    if (value_type < JLUST_VALUE_F64 || value_type > JLUST_VALUE_BF16)
        return fail(JLUST_STATUS_UNSUPPORTED_VALUE_TYPE, "%s: unknown value type %d", who, value_type);
    if (act != JLUST_FN_IDENTITY && act != JLUST_FN_RELU && act != JLUST_FN_GELU && act != JLUST_FN_SILU)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: function kind %d is no activation of this call", who, act);
    if (w_layout != 0 && w_layout != 1) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: w_layout is %d", who, w_layout);
    if (out < 0 || inp < 0 || cols < 0) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: negative extent", who);
    if (out >= (int64_t)1 << 31 || inp >= (int64_t)1 << 31 || cols >= (int64_t)1 << 31)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: an extent of 2^31 or more", who);
    if (groups) {
        if (int st = check_groups(who, cols, groups, copies)) return st;
        if (!plan && cols) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: groups without a plan", who);
    } else if (copies > 1) {
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: copies without groups", who);
    }
    return JLUST_STATUS_SUCCESS;
}

struct PlanParts { const int32_t *offsets, *perm, *src; };

PlanParts plan_parts(const int32_t *plan, int64_t n, int64_t groups, int64_t copies)
{
    if (!groups) return {nullptr, nullptr, nullptr};
    const int32_t *perm = plan + groups + 1;
    return {plan, perm, copies > 1 ? perm + n : perm};
}

template <typename F>
int by_type(int32_t value_type, F &&f)
{
    switch (value_type) {
    case JLUST_VALUE_F64: return f(double());
    case JLUST_VALUE_F32: return f(float());
    case JLUST_VALUE_F16: return f((_Float16)0);
    default: return f((__bf16)0.0f);
    }
}

// --------------------------------------------------------------------- forward

// What is planned, for the info entries.
jlust_product_info info_of(const TileArgs &a, int shape, bool w, bool x, bool g, size_t scratch_bytes)
{
    const TileForm f = tile_form(shape);
    return {f.m, f.n, f.copies, a.split, (w ? JLUST_PACKED_W : 0) | (x ? JLUST_PACKED_X : 0) | (g ? JLUST_PACKED_DY : 0),
            (int64_t)scratch_bytes};
}

template <typename T>
int linear(const jlust_linear &op, jlust_stream_t stream, jlust_product_info *info = nullptr)
{
    const PlanParts pl = plan_parts(op.plan, op.cols, op.groups, op.copies);
    TileArgs a;
    a.m = op.out;
    a.n = op.cols;
    a.k = op.inp;
    a.P = op.W;
    a.ldp = op.ldw;
    a.gp = op.w_stride;
    a.Q = op.X;
    a.ldq = op.ldx;
    a.qrow = pl.src;
    a.crow = pl.perm;
    a.offsets = pl.offsets;
    a.groups = (int)op.groups;
    a.C = op.Y;
    a.ldc = op.ldy;
    a.bias = op.bias;
    a.gb = op.bias_stride;
    a.R = op.R;
    a.ldr = op.ldr;
    a.Z = op.Z;
    a.ldz = op.ldz;
    a.act = op.act;
    const bool pkc = op.w_layout == 1;
    const int64_t batch = op.groups ? op.groups : 1, w_rows = pkc ? op.out : op.inp, w_len = pkc ? op.inp : op.out;
    const int64_t x_rows = op.cols / (op.groups ? op.copies : 1), ldw = padded<T>(w_len), ldx = padded<T>(op.inp);
    const bool bad_w = !lies_well<T>(op.W, w_len, op.ldw, op.groups ? op.w_stride : 0), bad_x = !lies_well<T>(op.X, op.inp, op.ldx, 0);
    const int64_t matrices = packed_matrices(op.groups, op.w_stride);
    const int64_t w_values = bad_w ? matrices * w_rows * ldw : 0, x_values = bad_x ? x_rows * ldx : 0;
    size_t pack = 0;
    if (op.cols > 48 * batch && worth_packing<T>(op.out, op.cols, op.inp, w_values + x_values, bad_w && !pkc)) {
        if (bad_w) {
            a.P = nullptr;
            a.ldp = ldw;
            a.gp = matrices > 1 ? w_rows * ldw : 0;
            a.p_pad = true;
        }
        if (bad_x) {
            a.Q = nullptr;
            a.ldq = ldx;
            a.q_pad = true;
        }
        pack = align256(sizeof(T) * w_values) + align256(sizeof(T) * x_values);
    }
    int shape = 0;
    size_t bytes = 0;
    if (int st = plan_tile_product<T>(&a, pkc, true, &shape, &bytes)) return st;
    if (info) {
        *info = info_of(a, shape, a.p_pad, a.q_pad, false, pack + bytes);
        return JLUST_STATUS_SUCCESS;
    }
    hipStream_t s = (hipStream_t)stream;
    if (pack + bytes) {
        void *ws = nullptr;
        if (int st = scratch(stream, pack + bytes, &ws)) return st;
        char *at = (char *)ws;
        if (a.p_pad) {
            if (int st = pack_rows<T>(w_rows, w_len, op.W, op.ldw, matrices, op.w_stride, nullptr, nullptr, at, ldw, s)) return st;
            a.P = at;
            at += align256(sizeof(T) * w_values);
        }
        if (a.q_pad) {
            if (int st = pack_rows<T>(x_rows, op.inp, op.X, op.ldx, 1, 0, nullptr, nullptr, at, ldx, s)) return st;
            a.Q = at;
            at += align256(sizeof(T) * x_values);
        }
        a.part = at;
    }
    return launch_tile_product<T>(a, pkc, true, shape, s);
}

// ------------------------------------------------------------------- gradients

template <typename T>
int linear_grad(const jlust_linear_grad &op, jlust_stream_t stream, jlust_product_info *info = nullptr)
{
    using A = typename Elem<T>::Acc;
    hipStream_t s = (hipStream_t)stream;
    const PlanParts pl = plan_parts(op.plan, op.cols, op.groups, op.copies);
    const bool slope = op.act != JLUST_FN_IDENTITY;
    const int64_t n = op.cols, out = op.out, inp = op.inp, batch = op.groups ? op.groups : 1;
    const bool wide = op.dX && op.groups && op.copies > 1;

    // What is packed.  G is made where there is a slope, and where dW's columns are
    // sorted by group: its sums then walk rows in order (found through the plan, their
    // copies waited for the indexes: 262 us of 573 in the gradients of 32 experts).
    // X is sorted with it.  Else what lies badly, where it pays.
    const bool x_kc = op.w_layout == 0;
    const int64_t w_rows = x_kc ? inp : out, w_len = x_kc ? out : inp, matrices = packed_matrices(op.groups, op.w_stride);
    const int64_t ldg_made = padded<T>(out), ldx_made = padded<T>(inp), ldw_made = padded<T>(w_len);
    bool make_g = (slope && (op.dX || op.dW)) || (op.groups && op.dW), make_x = op.groups && op.dW, make_w = false;
    {
        const bool bad_g = !lies_well<T>(op.dY, out, op.lddy, 0), bad_x = !lies_well<T>(op.X, inp, op.ldx, 0);
        const bool bad_w = !lies_well<T>(op.W, w_len, op.ldw, op.groups ? op.w_stride : 0);
        const int64_t g_values = bad_g && !make_g ? n * ldg_made : 0;
        const int64_t w_values = bad_w ? matrices * w_rows * ldw_made : 0, x_values = bad_x && !make_x ? n * ldx_made : 0;
        if (op.dX && n > 48 * batch && worth_packing<T>(inp, n, out, g_values + w_values, bad_w && !x_kc)) {
            make_g |= g_values > 0;
            make_w = bad_w;
        }
        if (op.dW && worth_packing<T>(inp, n, out, (make_g ? 0 : g_values) + x_values, true)) {
            make_g |= g_values > 0;
            make_x |= bad_x;
        }
    }
    make_g = make_g && n > 0;
    make_x = make_x && n > 0;

    // G's columns are the groups' in order where it is made, dY's own where not.
    const T *G = (const T *)op.dY;
    int64_t ldg = op.lddy;
    const int32_t *grow = pl.perm;
    if (make_g) {
        G = nullptr;
        ldg = ldg_made;
        grow = nullptr;
    }

    TileArgs x;
    int shape_x = 0;
    size_t part_x = 0;
    if (op.dX) {
        x.m = inp;
        x.n = n;
        x.k = out;
        x.P = make_w ? nullptr : op.W;             // the plan goes by alignment: what is made has any
        x.ldp = make_w ? ldw_made : op.ldw;
        x.gp = make_w ? (matrices > 1 ? w_rows * ldw_made : 0) : op.w_stride;
        x.p_pad = make_w;
        x.Q = G;
        x.ldq = ldg;
        x.q_pad = make_g;
        x.qrow = grow;
        x.crow = pl.perm;
        x.offsets = pl.offsets;
        x.groups = (int)op.groups;
        x.C = op.dX;
        x.ldc = wide ? inp : op.lddx;
        x.c_wide = wide;
        if (int st = plan_tile_product<T>(&x, x_kc, true, &shape_x, &part_x)) return st;
    }
    TileArgs w;
    int shape_w = 0;
    size_t part_w = 0;
    if (op.dW) {
        w.m = op.w_layout ? inp : out;
        w.n = op.w_layout ? out : inp;
        w.k = n;
        (op.w_layout ? w.P : w.Q) = make_x ? nullptr : op.X;
        (op.w_layout ? w.ldp : w.ldq) = make_x ? ldx_made : op.ldx;
        (op.w_layout ? w.p_pad : w.q_pad) = make_x;
        (op.w_layout ? w.Q : w.P) = G;
        (op.w_layout ? w.ldq : w.ldp) = ldg;
        (op.w_layout ? w.q_pad : w.p_pad) = make_g;
        w.offsets = pl.offsets;
        w.groups = (int)op.groups;
        w.C = op.dW;
        w.ldc = op.lddw;
        w.gc = op.dw_stride;
        if (int st = plan_tile_product<T>(&w, false, false, &shape_w, &part_w)) return st;
    }

    const int64_t blocks_m = (out + Prepass<T>::COLS - 1) / Prepass<T>::COLS;
    int64_t per = (n * blocks_m + 2047) / 2048;                // about 2,048 workgroups
    per = per < 64 ? 64 : (per + 7) / 8 * 8;
    const int64_t runs = (n + per - 1) / per + (op.groups ? (op.groups < n ? op.groups : n) : 0);
    if ((make_g || op.dbias) && runs * blocks_m >= 1 << 24)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "linear_grad: dY of %lld x %lld (%lld groups) is more than one launch takes",
                    (long long)out, (long long)n, (long long)op.groups);
    const size_t g_bytes = make_g ? align256(sizeof(T) * n * ldg) : 0;
    const size_t x_bytes = make_x ? align256(sizeof(T) * n * ldx_made) : 0;
    const size_t w_bytes = make_w ? align256(sizeof(T) * matrices * w_rows * ldw_made) : 0, made = g_bytes + x_bytes + w_bytes;
    const size_t wide_bytes = wide ? align256(sizeof(A) * n * inp) : 0;
    const size_t part = align256(part_x > part_w ? part_x : part_w);
    const size_t sum_bytes = op.dbias ? sizeof(A) * runs * out : 0;
    if (info) {
        info[0] = op.dX ? info_of(x, shape_x, make_w, false, make_g, made + wide_bytes + part + sum_bytes) : jlust_product_info{};
        info[1] = op.dW ? info_of(w, shape_w, false, make_x, make_g, made + wide_bytes + part + sum_bytes) : jlust_product_info{};
        return JLUST_STATUS_SUCCESS;
    }
    void *ws = nullptr;
    if (made + wide_bytes + part + sum_bytes)
        if (int st = scratch(stream, made + wide_bytes + part + sum_bytes, &ws)) return st;
    char *at = (char *)ws;
    T *g_buf = make_g ? (T *)at : nullptr, *x_buf = (T *)(at + g_bytes), *w_buf = (T *)(at + g_bytes + x_bytes);
    A *wide_buf = (A *)(at + made);
    x.part = w.part = at + made + wide_bytes;
    A *sums = op.dbias ? (A *)(at + made + wide_bytes + part) : nullptr;
    if (make_g) {
        x.Q = g_buf;
        (op.w_layout ? w.Q : w.P) = g_buf;
    }
    if (make_x) {
        if (int st = pack_rows<T>(n, inp, op.X, op.ldx, 1, 0, pl.src, pl.offsets ? pl.offsets + op.groups : nullptr, x_buf,
                                  ldx_made, s))
            return st;
        (op.w_layout ? w.P : w.Q) = x_buf;
    }
    if (make_w) {
        if (int st = pack_rows<T>(w_rows, w_len, op.W, op.ldw, matrices, op.w_stride, nullptr, nullptr, w_buf, ldw_made, s))
            return st;
        x.P = w_buf;
    }

    if (make_g || op.dbias) {
        if (n > 0) {
            hipLaunchKernelGGL((grad_prepass_kernel<T>), dim3((unsigned)(runs * blocks_m)), dim3(256), 0, s, n, out,
                               (const T *)op.dY, op.lddy, slope ? (const T *)op.Z : nullptr, op.ldz, op.act, g_buf, ldg,
                               pl.offsets, pl.perm, (int)op.groups, (int)per, (int)blocks_m, sums);
            if (int st = check_launch("grad_prepass_kernel")) return st;
        }
        if (op.dbias) {
            const dim3 grid(blocks_for(out, 32), (unsigned)(op.groups ? op.groups : 1));
            const int32_t *offsets = n ? pl.offsets : nullptr;
            if (runs <= 32 * (op.groups ? op.groups : 1))
                hipLaunchKernelGGL((grad_bias_kernel<T, 8>), grid, dim3(256), 0, s, n, out, offsets, (int)per, sums,
                                   (T *)op.dbias, op.dbias_stride);
            else
                hipLaunchKernelGGL((grad_bias_kernel<T, 32>), grid, dim3(1024), 0, s, n, out, offsets, (int)per, sums,
                                   (T *)op.dbias, op.dbias_stride);
            if (int st = check_launch("grad_bias_kernel")) return st;
        }
    }
    if (op.dX && n > 0 && inp > 0) {
        if (wide) x.C = wide_buf;
        if (int st = launch_tile_product<T>(x, x_kc, true, shape_x, s)) return st;
        if (wide) {
            const int64_t cols = n / op.copies, items = cols * ((inp + 3) / 4);
            hipLaunchKernelGGL((sum_copies_kernel<T>), dim3(blocks_for(items, 256)), dim3(256), 0, s, cols, inp,
                               (int)op.copies, wide_buf, (T *)op.dX, op.lddx);
            if (int st = check_launch("sum_copies_kernel")) return st;
        }
    }
    if (op.dW && inp > 0) {
        if (n == 0) {
            const int64_t rows = op.w_layout ? out : inp, d = op.w_layout ? inp : out;
            for (int64_t g = 0; g < (op.groups ? op.groups : 1); ++g)
                if (int st = fill_zero<T>(rows, d, (T *)op.dW + g * op.dw_stride, op.lddw, s)) return st;
        } else {
            if (int st = launch_tile_product<T>(w, false, false, shape_w, s)) return st;
        }
    }
    return JLUST_STATUS_SUCCESS;
}

}  // namespace
}  // namespace jlust

using namespace jlust;

extern "C" int jlust_hip_group_plan_ints(int64_t n, int64_t groups, int64_t copies, int64_t *ints)
{
    clear_error();
    if (int st = check_groups("group_plan", n, groups, copies)) return st;
    if (!ints) return fail(JLUST_STATUS_INVALID_ARGUMENT, "group_plan: null result");
    *ints = groups + 1 + n * (copies > 1 ? 2 : 1);
    return JLUST_STATUS_SUCCESS;
}

extern "C" int jlust_hip_group_plan_build(int64_t n, int64_t groups, int64_t copies, int32_t origin, const void *ids,
                                          int ids64, int32_t *plan, jlust_stream_t stream)
{
    clear_error();
    if (int st = check_groups("group_plan", n, groups, copies)) return st;
    if (int st = check_origin(origin)) return st;
    if (bad_ptr(ids, n) || !plan) return fail(JLUST_STATUS_INVALID_ARGUMENT, "group_plan: null device pointer");
    if (int st = require_device(nullptr)) return st;
    hipStream_t s = (hipStream_t)stream;
    int bits = 1;
    while ((groups >> bits) != 0) ++bits;
    int32_t *perm = plan + groups + 1, *src = copies > 1 ? perm + n : nullptr;
    if (n <= SMALL_COLUMNS && groups <= SMALL_GROUPS) {
        hipLaunchKernelGGL(group_plan_small_kernel, dim3(1), dim3(SMALL_WAVES * 64),
                           SMALL_WAVES * (groups + 1) * sizeof(int32_t), s, n, (int)groups, (int)copies, (int)origin, ids,
                           ids64, bits, plan, perm, src);
        return check_launch("group_plan_small_kernel");
    }
    int64_t per = (groups + 256) / 256 * 256;
    int64_t runs = (n + per - 1) / per;
    if (runs < 1) runs = 1;
    const int64_t counts_n = (groups + 1) * runs;
    const size_t first = (exclusive_scan_scratch_bytes(counts_n) + 255) / 256 * 256;
    void *ws = nullptr;
    if (int st = scratch(stream, first + sizeof(int32_t) * counts_n, &ws)) return st;
    int32_t *counts = (int32_t *)((char *)ws + first);
    const dim3 grid((unsigned)((runs + PLAN_WAVES - 1) / PLAN_WAVES)), block(PLAN_WAVES * 64);
    const size_t lds = PLAN_WAVES * (groups + 1) * sizeof(int32_t);
    hipLaunchKernelGGL((group_plan_kernel<false>), grid, block, lds, s, n, (int)groups, (int)copies, (int)origin, ids, ids64,
                       bits, runs, (int)per, counts, plan, perm, src);
    if (int st = check_launch("group_plan_kernel")) return st;
    if (counts_n <= SCAN_COUNTS) {
        hipLaunchKernelGGL(group_scan_kernel, dim3(1), dim3(1024), 0, s, (int)counts_n, counts);
        if (int st = check_launch("group_scan_kernel")) return st;
    } else if (int st = exclusive_scan_i32(counts, counts, counts_n, stream)) {
        return st;
    }
    hipLaunchKernelGGL((group_plan_kernel<true>), grid, block, lds, s, n, (int)groups, (int)copies, (int)origin, ids, ids64,
                       bits, runs, (int)per, counts, plan, perm, src);
    return check_launch("group_plan_kernel");
}

namespace {

int check_linear(const jlust_linear *op)
{
    clear_error();
    if (!op) return fail(JLUST_STATUS_INVALID_ARGUMENT, "linear: null argument");
    const char *who = "linear";
    if (int st = check_common(who, op->value_type, op->act, op->w_layout, op->out, op->inp, op->cols, op->groups, op->copies,
                              op->plan))
        return st;
    const int64_t xcols = op->groups ? op->cols / op->copies : op->cols;
    const int64_t wr = op->w_layout ? op->inp : op->out, wc = op->w_layout ? op->out : op->inp;
    return check_operands(who, {{"W", op->W, wr, wc, op->ldw, true},
                                {"X", op->X, op->inp, xcols, op->ldx, true},
                                {"Y", op->Y, op->out, op->cols, op->ldy, true},
                                {"R", op->R, op->out, op->cols, op->ldr, false},
                                {"Z", op->Z, op->out, op->cols, op->ldz, false}});
}

int check_linear_grad(const jlust_linear_grad *op)
{
    clear_error();
    if (!op) return fail(JLUST_STATUS_INVALID_ARGUMENT, "linear_grad: null argument");
    const char *who = "linear_grad";
    if (int st = check_common(who, op->value_type, op->act, op->w_layout, op->out, op->inp, op->cols, op->groups, op->copies,
                              op->plan))
        return st;
    const int64_t xcols = op->groups ? op->cols / op->copies : op->cols;
    const int64_t wr = op->w_layout ? op->inp : op->out, wc = op->w_layout ? op->out : op->inp;
    if (int st = check_apart(who, "dW", op->dW, wr, wc, op->lddw, op->groups, op->dw_stride)) return st;
    if (int st = check_apart(who, "dbias", op->dbias, op->out, 1, op->out, op->groups, op->dbias_stride)) return st;
    // W is read for dX alone (it may be laid out otherwise beside a dW), X for dW alone.
    return check_operands(who, {{"W", op->dX ? op->W : nullptr, wr, wc, op->ldw, op->dX != nullptr},
                                {"X", op->dW ? op->X : nullptr, op->inp, xcols, op->ldx, op->dW != nullptr},
                                {"dY", op->dY, op->out, op->cols, op->lddy, true},
                                {"Z", op->Z, op->out, op->cols, op->ldz, op->act != JLUST_FN_IDENTITY},
                                {"dX", op->dX, op->inp, xcols, op->lddx, false},
                                {"dW", op->dW, wr, wc, op->lddw, false}});
}

}  // namespace

extern "C" int jlust_hip_linear(const jlust_linear *op, jlust_stream_t stream)
{
    if (int st = check_linear(op)) return st;
    if (int st = require_device(nullptr)) return st;
    if (op->out == 0 || op->cols == 0) return JLUST_STATUS_SUCCESS;
    return by_type(op->value_type, [&](auto t) { return linear<decltype(t)>(*op, stream); });
}

extern "C" int jlust_hip_linear_grad(const jlust_linear_grad *op, jlust_stream_t stream)
{
    if (int st = check_linear_grad(op)) return st;
    if (int st = require_device(nullptr)) return st;
    if (op->out == 0) {
        if (!op->dX) return JLUST_STATUS_SUCCESS;
        return by_type(op->value_type, [&](auto t) {
            const int64_t xcols = op->groups ? op->cols / op->copies : op->cols;
            return fill_zero<decltype(t)>(xcols, op->inp, op->dX, op->lddx, (hipStream_t)stream);
        });
    }
    return by_type(op->value_type, [&](auto t) { return linear_grad<decltype(t)>(*op, stream); });
}

extern "C" int jlust_hip_linear_info(const jlust_linear *op, jlust_product_info *info)
{
    if (int st = check_linear(op)) return st;
    if (!info) return fail(JLUST_STATUS_INVALID_ARGUMENT, "linear_info: null result");
    *info = jlust_product_info{};
    if (op->out == 0 || op->cols == 0) return JLUST_STATUS_SUCCESS;
    return by_type(op->value_type, [&](auto t) { return linear<decltype(t)>(*op, nullptr, info); });
}

extern "C" int jlust_hip_linear_grad_info(const jlust_linear_grad *op, jlust_product_info *info)
{
    if (int st = check_linear_grad(op)) return st;
    if (!info) return fail(JLUST_STATUS_INVALID_ARGUMENT, "linear_grad_info: null result");
    info[0] = info[1] = jlust_product_info{};
    if (op->out == 0) return JLUST_STATUS_SUCCESS;
    return by_type(op->value_type, [&](auto t) { return linear_grad<decltype(t)>(*op, nullptr, info); });
}

namespace jlust {
int preload_linear()
{
    JLUST_PRELOAD_KERNEL(group_plan_small_kernel);
    return JLUST_STATUS_SUCCESS;
}
}  // namespace jlust
