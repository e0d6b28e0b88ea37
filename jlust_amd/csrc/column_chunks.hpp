// column_chunks.hpp -- columns of a matrix by chunks of 16 bytes: their reads and
// writes, packed and as the sums' type, and sums over the lanes that hold a column.
#pragma once

#include "tile_product.hpp"

namespace jlust {

// The sums of K values over the LANES lanes of a column, in every one of them.
template <int LANES, int K, typename A>
__device__ __forceinline__ void column_sum(A (&v)[K], A *lds)
{
#pragma unroll
    for (int d = (LANES < 64 ? LANES : 64) / 2; d; d >>= 1)
#pragma unroll
        for (int q = 0; q < K; ++q) v[q] += __shfl_xor(v[q], d, 64);
    if constexpr (LANES > 64) {
        constexpr int W = LANES / 64;
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int q = 0; q < K; ++q) lds[wave * K + q] = v[q];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < K; ++q) {
            A s = A(0);
#pragma unroll
            for (int w = 0; w < W; ++w) s += lds[w * K + q];
            v[q] = s;
        }
    }
}

// A chunk as it lies in memory, and its values.  Past the column's end: zeros, or
// where `over` what follows, the next column, which is not summed.  (Half's 8 values
// read one by one hold the wave up, 60,000 columns of 333: 28.1 and 26.8 us, backward
// 45.9 and 40.3; Float32's 4 do not, 9,001 of 2,049: 27.1 and 27.8, 57.5 and 59.8.)
template <typename T>
__device__ __forceinline__ uint32x4 read_raw(const T *p, int64_t left, bool over = false)
{
    constexpr int CH = 16 / sizeof(T);
    const uint32x4 zero = {0, 0, 0, 0};
    return left >= CH || (over && left > 0) ? load_chunk(p) : left > 0 ? load_chunk_part(p, left) : zero;
}

// The chunk at `at` of a column of d values; WHOLE: d is a whole number of chunks, and
// what lies past it is the first chunk, read and dropped: no branch around a partial
// chunk's reads comes between a wave's reads (the gradient of 16,384 columns' routing to
// 160 experts: 9.3 us and 8.0).
template <bool WHOLE, typename T>
__device__ __forceinline__ uint32x4 read_at(const T *column, int64_t at, int64_t d, bool over = false)
{
    if constexpr (WHOLE) {
        const bool in = at < d;
        const uint32x4 v = load_chunk(column + (in ? at : 0)), zero = {0, 0, 0, 0};
        return in ? v : zero;
    } else {
        return read_raw(column + at, d - at, over);
    }
}

template <typename T, typename A>
__device__ __forceinline__ void values(uint32x4 v, A (&f)[16 / sizeof(T)])
{
    constexpr int CH = 16 / sizeof(T);
    T e[CH];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int j = 0; j < CH; ++j) f[j] = A(e[j]);
}

// Its values again: without this the compiler keeps those of an earlier pass, two
// or four times the registers of the packed chunk.
template <typename T, typename A>
__device__ __forceinline__ void values_again(uint32x4 &v, A (&f)[16 / sizeof(T)])
{
    asm("" : "+v"(v));
    values<T>(v, f);
}

template <typename T, typename A>
__device__ __forceinline__ void read_chunk(const T *p, int64_t left, A (&f)[16 / sizeof(T)])
{
    values<T>(read_raw(p, left), f);
}

template <typename T, typename A>
__device__ __forceinline__ void write_chunk(T *p, int64_t left, const A (&f)[16 / sizeof(T)], bool streamed = false)
{
    constexpr int CH = 16 / sizeof(T);
    T e[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) e[j] = T(f[j]);
    if (left >= CH) {
        if (streamed) stream_chunk(p, e);
        else store_vec<CH>(p, e);
    } else {
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (j < left) p[j] = e[j];
    }
}

// As write_chunk of the chunk at `at` of d values.
template <bool WHOLE, typename T, typename A>
__device__ __forceinline__ void write_at(T *column, int64_t at, int64_t d, const A (&f)[16 / sizeof(T)], bool streamed = false)
{
    constexpr int CH = 16 / sizeof(T);
    if constexpr (WHOLE) {
        if (at < d) write_chunk(column + at, CH, f, streamed);
    } else {
        write_chunk(column + at, d - at, f, streamed);
    }
}

// n / d by a product, for n below 2^31: m = floor(2^(31 + s) / d) + 1 is below 2^32 and
// within 2^s / 2^(31 + s) of it with s = ceil(log2 d).
struct Divider {
    int64_t d;
    uint32_t m, shift;
    bool fits;                                     // all n are below 2^31
    Divider(int64_t d_, int64_t n) : d(d_), m(0), shift(0), fits(n < (int64_t)1 << 31 && d_ < (int64_t)1 << 31)
    {
        if (!fits) return;
        while (((int64_t)1 << shift) < d) ++shift;
        m = (uint32_t)(((uint64_t)1 << (31 + shift)) / d + 1);
        shift += 31;
    }
    __device__ __forceinline__ int64_t of(int64_t n) const
    {
        return fits ? (int64_t)((uint64_t)(uint32_t)n * m >> shift) : n / d;
    }
};

// A launch takes fewer than 2^32 threads: at most 2^21 workgroups, which walk over the
// items in turn.
inline unsigned column_blocks(int64_t items, int64_t each, int64_t most = 1 << 21)
{
    const int64_t blocks = (items + each - 1) / each;
    return (unsigned)(blocks < most ? blocks : most);
}

// A rows x cols operand of a call (null: `needed` refuses it where it holds something).
inline int check_matrix(const char *who, const char *name, const void *p, int64_t rows, int64_t cols, int64_t ld, bool needed)
{
    if (!p) {
        if (needed && rows && cols) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %s is null", who, name);
        return JLUST_STATUS_SUCCESS;
    }
    if (cols > 1 && ld < rows)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %s has leading dimension %lld, its columns %lld rows", who, name,
                    (long long)ld, (long long)rows);
    return JLUST_STATUS_SUCCESS;
}

inline int check_extents(const char *who, int32_t value_type, int64_t d, int64_t cols)
{
    if (value_type < JLUST_VALUE_F64 || value_type > JLUST_VALUE_BF16)
        return fail(JLUST_STATUS_UNSUPPORTED_VALUE_TYPE, "%s: unknown value type %d", who, value_type);
    if (d < 0 || cols < 0) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: negative extent", who);
    if (d >= (int64_t)1 << 31 || cols >= (int64_t)1 << 31)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: an extent of 2^31 or more", who);
    return JLUST_STATUS_SUCCESS;
}

// f(a value of the type).
template <typename F>
int with_type(int32_t value_type, F &&f)
{
    switch (value_type) {
    case JLUST_VALUE_F64: return f(double());
    case JLUST_VALUE_F32: return f(float());
    case JLUST_VALUE_F16: return f((_Float16)0);
    default: return f((__bf16)0.0f);
    }
}

}  // namespace jlust
