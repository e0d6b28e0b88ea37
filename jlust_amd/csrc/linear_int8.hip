// linear_int8.hip -- the dense products of 8-bit integers, and the columns' scales and
// integers that they take.
#include "column_chunks.hpp"
#include "lanes.hpp"
#include "tile_kernel.hpp"

#include <cmath>

namespace jlust {

template int plan_tile_product<int8_t>(TileArgs *, bool, bool, int *, size_t *, double *);

namespace {

template <typename O, int BM, int BN, int WM, int WN>
int launch_registers(const TileArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL((tile_product_kernel<int8_t, true, true, BM, BN, WM, WN, O>), dim3((unsigned)work_groups(a, false)),
                       dim3(WM * WN * 64), 0, s, a);
    return check_launch("tile_product_kernel");
}

template <typename O, int BM, int BN, int WM, int WN, int BK, int NB>
int launch_copied(const TileArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL((tile_copy_kernel<int8_t, true, true, BM, BN, WM, WN, BK, NB, O>), dim3((unsigned)work_groups(a, false)),
                       dim3(WM * WN * 64), 0, s, a);
    return check_launch("tile_copy_kernel");
}

}  // namespace

template <typename O>
int launch_tile_product8(const TileArgs &args, int shape, hipStream_t s)
{
    TileArgs a = args;
    if (a.split == 1) a.part = nullptr;
    int st;
    switch (shape) {
    case FEW_16:
        hipLaunchKernelGGL((few_columns_kernel<int8_t, true, 1, O>), dim3((unsigned)work_groups(a, false)), dim3(Few<1>::WAVES * 64), 0,
                           s, a);
        st = check_launch("few_columns_kernel");
        break;
    case REG_32: st = launch_registers<O, 128, 32, 4, 1>(a, s); break;
    case COPY_256: st = launch_copied<O, 256, 256, 2, 4, 128, 2>(a, s); break;
    case COPY_TALL: st = launch_copied<O, 256, 128, 2, 2, 64, 3>(a, s); break;
    case COPY_128: st = launch_copied<O, 128, 128, 2, 2, 128, 2>(a, s); break;
    default: st = launch_registers<O, 64, 64, 2, 2>(a, s); break;
    }
    if (st || a.split == 1) return st;
    const int64_t items = a.n * ((a.m + 3) / 4);
    const bool shares = a.split > 16;
    const dim3 grid((unsigned)((items + (shares ? 15 : 255)) / (shares ? 16 : 256)));
    if (shares) hipLaunchKernelGGL((split_reduce_kernel<int8_t, false, 16, O>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((split_reduce_kernel<int8_t, false, 1, O>), grid, dim3(256), 0, s, a);
    return check_launch("split_reduce_kernel");
}

template int launch_tile_product8<float>(const TileArgs &, int, hipStream_t);
template int launch_tile_product8<_Float16>(const TileArgs &, int, hipStream_t);
template int launch_tile_product8<__bf16>(const TileArgs &, int, hipStream_t);

// ------------------------------------------------------------------ quantising

namespace {

typedef uint16_t ushortx2 __attribute__((ext_vector_type(2)));

// The largest |x| of a chunk and `top` by their bits, which NaN and infinity end: bits of
// values without their sign are in the values' order, 16-bit ones two to a register.
template <typename T>
__device__ __forceinline__ uint32_t chunk_top(uint32x4 v, uint32_t top)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = v[i];
        if constexpr (sizeof(T) == 2) {
            const ushortx2 m = __builtin_elementwise_max(__builtin_bit_cast(ushortx2, u & 0x7FFF7FFFu), __builtin_bit_cast(ushortx2, top));
            top = __builtin_bit_cast(uint32_t, m);
        } else {
            top = (u & 0x7FFFFFFFu) > top ? u & 0x7FFFFFFFu : top;
        }
    }
    return top;
}

// The value that the largest bits of a column's lanes stand for.
template <typename T, int LANES>
__device__ __forceinline__ float column_top(uint32_t v, uint32_t *lds)
{
    if constexpr (sizeof(T) == 2) v = (v >> 16) > (v & 0xFFFF) ? v >> 16 : v & 0xFFFF;
    v = over_lanes<(LANES < 64 ? LANES : 64)>(v, Larger());
    if constexpr (LANES > 64) {
        constexpr int W = LANES / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) v = lds[w] > v ? lds[w] : v;
    }
    if constexpr (sizeof(T) == 2) return (float)__builtin_bit_cast(T, (uint16_t)v);
    else return __builtin_bit_cast(float, v);
}

// A column's scale s.  `up`: x and s are both times it, where 1/s would pass the type's
// range or s is so small that x/s may pass 127; 0: the column becomes zeros.
struct Scale { float s, by, inv, up; };

__device__ __forceinline__ Scale scale_from(float top)
{
    if (!(top < INFINITY)) return {__builtin_nanf(""), 0.0f, 0.0f, 0.0f};
    const float s = (float)((double)top / 127.0);
    if (s == 0) return {0.0f, 0.0f, 0.0f, 0.0f};
    const float up = s < 0x1p-100f ? 0x1p64f : 1.0f, by = s * up;
    return {s, by, 1.0f / by, up};
}

// CH values of a column over s to the nearest whole numbers, halves to the even one.
// x inv + 1.5 2^23 has n, about x/s, in its low bits; inv is off by a little, so the
// nearest is found again from x - n s, which is exact (a multiple of half s's last place,
// at most about s/2): an odd n is left at s/2, an even one past it.
template <typename T>
__device__ __forceinline__ void quantize_chunk(uint32x4 v, const Scale &c, int8_t (&q)[16 / sizeof(T)])
{
    constexpr int CH = 16 / sizeof(T);
    constexpr float MAGIC = 12582912.0f;
    if (c.up == 0) v = uint32x4{0, 0, 0, 0};
    float x[CH];
    values<T>(v, x);
    if (c.up != 1) {
#pragma unroll
        for (int j = 0; j < CH; ++j) x[j] *= c.up;
    }
    int n[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const float r = fmaf(x[j], c.inv, MAGIC), t = fmaf(MAGIC - r, c.by, x[j]);
        const int bits = __builtin_bit_cast(int, r);
        const float most = __builtin_bit_cast(float, __builtin_bit_cast(int, 0.5f * c.by) - (bits & 1));
        n[j] = bits + (t > most) - (t < -most);
    }
    if (c.up != 1) {
        constexpr int ZERO = 0x4B400000;           // MAGIC's bits
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int m = c.up == 0 ? 0 : n[j] - ZERO;
            n[j] = m > 127 ? 127 : m < -127 ? -127 : m;
        }
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) q[j] = (int8_t)n[j];
}

template <int CH>
__device__ __forceinline__ void store_bytes(int8_t *p, int64_t left, const int8_t (&q)[CH])
{
    if (left >= CH) {
        store_vec<CH>(p, q);
    } else {
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (j < left) p[j] = q[j];
    }
}

// A column stays in the registers of LANES lanes, VPL chunks each, between its read and
// its write.  A wave with two columns, the second read before the first is worked on,
// took 15.2 us for 8,192 of 2,048 bfloat16; as many waves as columns take 11.8.
template <typename T, bool WHOLE, int LANES, int VPL>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void quantize_kernel(int64_t d, int64_t cols, const T *__restrict__ X,
                                                                             int64_t ldx, int8_t *__restrict__ Q, int64_t ldq,
                                                                             float *__restrict__ scales)
{
    constexpr int CH = 16 / sizeof(T), NT = LANES > 256 ? LANES : 256, COLS = NT / LANES;
    __shared__ uint32_t s_top[NT / 64];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    for (int64_t c0 = (int64_t)blockIdx.x * COLS; c0 < cols; c0 += (int64_t)gridDim.x * COLS) {
        // A chunk over the end of all but the last column is read whole; what follows the
        // column is taken out again.
        const int64_t c = c0 + sub;
        const bool over = sizeof(T) == 2 && c + 1 < cols && d >= CH;
        const T *column = X + (c < cols ? c : cols - 1) * ldx;
        uint32x4 x[VPL];
#pragma unroll
        for (int i = 0; i < VPL; ++i) x[i] = read_at<WHOLE>(column, (int64_t)(lane + LANES * i) * CH, d, over);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t left = d - (int64_t)(lane + LANES * i) * CH;
            if (!WHOLE && sizeof(T) == 2 && left > 0 && left < CH) {
                T e[CH];
                __builtin_memcpy(e, &x[i], 16);
#pragma unroll
                for (int j = 0; j < CH; ++j) e[j] = j < left ? e[j] : T(0);
                __builtin_memcpy(&x[i], e, 16);
            }
            top = chunk_top<T>(x[i], top);
        }
        const Scale s = scale_from(column_top<T, LANES>(top, s_top));
        if (c >= cols) continue;
        if (lane == 0) scales[c] = s.s;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t at = (int64_t)(lane + LANES * i) * CH;
            if (at >= d) continue;
            int8_t q[CH];
            quantize_chunk<T>(x[i], s, q);
            store_bytes(Q + c * ldq + at, WHOLE ? CH : d - at, q);
        }
    }
}

// Columns of any length: the second pass reads them again.
template <typename T>
__global__ __launch_bounds__(1024) void quantize_long_kernel(int64_t d, int64_t cols, const T *__restrict__ X, int64_t ldx,
                                                             int8_t *__restrict__ Q, int64_t ldq, float *__restrict__ scales)
{
    constexpr int CH = 16 / sizeof(T);
    __shared__ uint32_t s_top[16];
    for (int64_t c = blockIdx.x; c < cols; c += gridDim.x) {
        uint32_t top = 0;
        for (int64_t at = (int64_t)threadIdx.x * CH; at < d; at += 1024 * CH)
            top = chunk_top<T>(read_raw(X + c * ldx + at, d - at), top);
        const Scale s = scale_from(column_top<T, 1024>(top, s_top));
        if (threadIdx.x == 0) scales[c] = s.s;
        for (int64_t at = (int64_t)threadIdx.x * CH; at < d; at += 1024 * CH) {
            int8_t q[CH];
            quantize_chunk<T>(read_raw(X + c * ldx + at, d - at), s, q);
            store_bytes(Q + c * ldq + at, d - at, q);
        }
    }
}

template <typename T>
int quantize(int64_t d, int64_t cols, const void *X, int64_t ldx, int8_t *Q, int64_t ldq, float *scales, hipStream_t s)
{
    const int64_t chunks = (d * (int64_t)sizeof(T) + 15) / 16;
    auto launch = [&](auto kernel, int lanes) {
        const int nt = lanes > 256 ? lanes : 256;
        hipLaunchKernelGGL(kernel, dim3(column_blocks(cols, nt / lanes, 1 << 14)), dim3(nt), 0, s, d, cols, (const T *)X, ldx, Q, ldq, scales);
    };
    // Few columns wait for one of them: it goes over more lanes (bfloat16 columns of 2,048 by
    // 64 lanes and by 256: 512 of them 3.50 and 2.76 us, 1,024 3.66 and 3.58, 2,048 4.23 and 4.67).
    const bool few = cols <= 1024;
    auto go = [&](auto whole) {
        constexpr bool W = decltype(whole)::value;
        if (chunks <= 16) launch(quantize_kernel<T, W, 16, 1>, 16);
        else if (chunks <= 64) launch(quantize_kernel<T, W, 64, 1>, 64);
        else if (chunks <= 128 && !few) launch(quantize_kernel<T, W, 64, 2>, 64);
        else if (chunks <= 256 && !few) launch(quantize_kernel<T, W, 64, 4>, 64);
        else if (chunks <= 256) launch(quantize_kernel<T, W, 256, 1>, 256);
        else if (chunks <= 512) launch(quantize_kernel<T, W, 256, 2>, 256);
        else if (chunks <= 1024) launch(quantize_kernel<T, W, 256, 4>, 256);
        else if (chunks <= 2048) launch(quantize_kernel<T, W, 512, 4>, 512);
        else launch(quantize_long_kernel<T>, 1024);
    };
    if (d > 0 && d % (16 / sizeof(T)) == 0) go(std::true_type());
    else go(std::false_type());
    return check_launch("quantize_kernel");
}

}  // namespace
}  // namespace jlust

using namespace jlust;

extern "C" int jlust_hip_quantize_columns(int32_t value_type, int64_t d, int64_t cols, const void *X, int64_t ldx, int8_t *Q,
                                          int64_t ldq, float *scales, jlust_stream_t stream)
{
    clear_error();
    const char *who = "quantize";
    if (int st = check_extents(who, value_type, d, cols)) return st;
    if (value_type == JLUST_VALUE_F64)
        return fail(JLUST_STATUS_UNSUPPORTED_VALUE_TYPE, "%s: columns are Float32, Float16 or BFloat16", who);
    if (int st = check_matrix(who, "X", X, d, cols, ldx, true)) return st;
    if (int st = check_matrix(who, "Q", Q, d, cols, ldq, true)) return st;
    if (bad_ptr(scales, cols)) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: scales are null", who);
    if (int st = require_device(nullptr)) return st;
    if (cols == 0) return JLUST_STATUS_SUCCESS;
    hipStream_t s = (hipStream_t)stream;
    switch (value_type) {
    case JLUST_VALUE_F32: return quantize<float>(d, cols, X, ldx, Q, ldq, scales, s);
    case JLUST_VALUE_F16: return quantize<_Float16>(d, cols, X, ldx, Q, ldq, scales, s);
    default: return quantize<__bf16>(d, cols, X, ldx, Q, ldq, scales, s);
    }
}

namespace jlust {
int preload_linear_int8()
{
    JLUST_PRELOAD_KERNEL((quantize_kernel<float, true, 64, 1>));
    return JLUST_STATUS_SUCCESS;
}
}  // namespace jlust
