// tile_product.hpp -- the dense products' common form,
//
//   C[n][m] = sum_k P(m, k) Q(n, k)         (row n of C is contiguous in m)
//
// with an epilogue (bias, activation, residual, kept pre-activation) or, with
// the k range split over workgroups, partial sums for split_reduce.  A
// column-major matrix is the row-major array of its columns, so with n a column
// of Y, m a row of W and k a row of X this is Y = W*X; the gradients are the
// same sum over other axes (linear.hip).  The kernels are in tile_kernel.hpp.
#pragma once

#include "activation.hpp"
#include "common.hpp"

namespace jlust {

// One product.  P and Q are each contiguous along k ("kc": element (r, k) at
// base[r * ld + k]) or along their own side ("sc": base[k * ld + r]).
struct TileArgs {
    int64_t m = 0, n = 0, k = 0;
    const void *P = nullptr, *Q = nullptr;
    int64_t ldp = 0, ldq = 0;
    int64_t gp = 0;                     // elements between the P of two groups
    bool p_pad = false, q_pad = false;  // rows lie in buffers of their own, zeros after them to the next 16 bytes
    const int32_t *qrow = nullptr;      // kc: the row of Q that n stands for (null: n itself)
    const int32_t *crow = nullptr;      // the row of C, R and Z that n stands for
    void *C = nullptr;
    int64_t ldc = 0, gc = 0;
    int c_wide = 0;                     // C holds the sums' type, not T
    const void *bias = nullptr;         // m values, gb elements between groups
    int64_t gb = 0;
    const void *R = nullptr;            // added after the activation
    int64_t ldr = 0;
    void *Z = nullptr;                  // gets the sum with its bias, before the activation
    int64_t ldz = 0;
    int act = JLUST_FN_IDENTITY;
    // Groups.  A product with kc Q: the rows [offsets[g], offsets[g+1]) of n
    // take group g's P, those from offsets[groups] on belong to none (their sum
    // is 0, without a bias).  A product of two sc operands: group g's C sums
    // over the k of [offsets[g], offsets[g+1]).
    const int32_t *offsets = nullptr;
    int groups = 0;
    // Products of 8-bit integers, whose C, bias, R and Z hold another type: what a row
    // of P and a row of Q are times of.
    const float *ps = nullptr;          // m values, gs elements between groups
    int64_t gs = 0;
    const float *qs = nullptr;          // by the rows of Q
    bool streamed = false;              // whole chunks of 16 bytes of C go past the caches
    void *part = nullptr;               // partial sums [split][C's rows][m]
    int split = 1;
    int tiles_m = 0, tiles_n = 0;
};

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef double doublex4 __attribute__((ext_vector_type(4)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem { using Acc = float; using Acc4 = floatx4; };
template <> struct Elem<int8_t> { using Acc = int; using Acc4 = intx4; };
template <> struct Elem<double> { using Acc = double; using Acc4 = doublex4; };

// ------------------------------------------------------------ loads, stores

// V values at p, which may lie at any element: the hardware takes vector
// accesses at 2-byte and 4-byte alignment.
template <int V, typename T>
__device__ __forceinline__ void load_vec(const T *p, T *v)
{
    __builtin_memcpy(v, p, V * sizeof(T));
}

template <int V, typename T>
__device__ __forceinline__ void store_vec(T *p, const T *v)
{
    __builtin_memcpy(p, v, V * sizeof(T));
}

// 16 bytes past the caches.  Results that the eight L2s of 4 MB do not hold would only
// push out what is still read (16,384 bfloat16 columns of 4,096: 71.4 us by plain stores
// and 63.9; backward, 200,003 Float32 columns of 100: 51.6 and 49.2; products' results
// of 16 bits gain nothing: 8,192 columns 2048 -> 8192, 305 and 307 us; of 8 bits, 220 and
// 210, 32 experts' 120 and 109).
constexpr int64_t STREAMED = 32 << 20;         // bytes of a result from which it is stored so
typedef uint32_t uint32x4_any __attribute__((ext_vector_type(4), aligned(2), may_alias));

template <typename T>
__device__ __forceinline__ void stream_chunk(T *p, const T *v)
{
    uint32x4 u;
    __builtin_memcpy(&u, v, 16);
    __builtin_nontemporal_store((uint32x4_any)u, reinterpret_cast<uint32x4_any *>(p));
}

template <typename T>
__device__ __forceinline__ uint32x4 load_chunk(const T *p)
{
    uint32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// The first `count` elements of a chunk, zeros after them.
template <typename T>
__device__ __forceinline__ uint32x4 load_chunk_part(const T *p, int64_t count)
{
    constexpr int CH = 16 / sizeof(T);
    T e[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) e[j] = j < count ? p[j] : T(0);
    uint32x4 v;
    __builtin_memcpy(&v, e, 16);
    return v;
}

// The group of the tile'th run of at most `per` rows when every group's rows
// [offsets[g], offsets[g+1]) are cut into such runs, group after group, and
// those from offsets[groups] to n as group `groups`.  False past the last.
// Every lane of a wave calls it with the same arguments.
struct GroupRun { int group; int64_t begin, end, group_end; };

__device__ __forceinline__ bool find_run(const int32_t *__restrict__ offsets, int groups, int64_t n, int64_t tile,
                                         int per, GroupRun *out)
{
    const int lane = lane_id();
    int64_t base = 0;
    for (int g0 = 0; g0 <= groups; g0 += 64) {
        const int g = g0 + lane;
        int32_t lo = 0, hi = 0;
        if (g <= groups) {
            lo = offsets[g];
            hi = g < groups ? offsets[g + 1] : (int32_t)n;
        }
        const int32_t tiles = (hi - lo + per - 1) / per;
        int32_t incl = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int32_t t = __shfl_up(incl, d, 64);
            if (lane >= d) incl += t;
        }
        const int32_t total = __shfl(incl, 63, 64);
        if (tile < base + total) {
            const uint64_t mask = __ballot(tile < base + incl);
            const int l = __ffsll((unsigned long long)mask) - 1;
            const int64_t first = base + __shfl(incl - tiles, l, 64);
            const int64_t b = __shfl(lo, l, 64), e = __shfl(hi, l, 64);
            out->group = g0 + l;
            out->group_end = e;
            out->begin = b + (tile - first) * per;
            out->end = out->begin + per < e ? out->begin + per : e;
            return true;
        }
        base += total;
    }
    return false;
}

// Chooses the tile shape and the split of k and sets them in `a`; *part_bytes of
// partial sums are to be at a->part when it is launched.  INVALID_ARGUMENT where one
// launch does not take all the tiles.
template <typename T>
int plan_tile_product(TileArgs *a, bool pkc, bool qkc, int *shape, size_t *part_bytes, double *estimate = nullptr);
template <typename T>
int launch_tile_product(const TileArgs &a, bool pkc, bool qkc, int shape, hipStream_t s);
// The same of 8-bit operands along k, C holding O.
template <typename O>
int launch_tile_product8(const TileArgs &a, int shape, hipStream_t s);

// What a shape is: its tile, and whether its operands are copied to LDS.
struct TileForm { int m, n, copies; };
TileForm tile_form(int shape);

}  // namespace jlust
