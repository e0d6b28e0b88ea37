// layer_norm.hip -- layer norm of the columns of a matrix, and its gradients.
//
//   mean = sum(x)/d    var = sum((x - mean)^2)/d    rstd = 1/sqrt(var + eps)
//   y = (x - mean) rstd weight + bias
//   h = (x - mean) rstd, g = dy weight:
//   dx = rstd (g - sum(g)/d - h sum(g h)/d),   dweight = sum dy h,   dbias = sum dy
//
// Both directions are bound by memory.  A column stays in the registers of LANES
// lanes between its one read and its one write (two-pass variance, so a large
// mean costs no digits); the backward kernel also keeps its share of dweight and
// dbias in registers over all the columns it takes, so X and dY are read once for
// all three results.  Columns too long for that are read again from L2.
#include "tile_product.hpp"

namespace jlust {
namespace {

constexpr int64_t LN_BLOCKS = 2048;            // workgroups that walk over the columns, forward

template <typename A>
__device__ __forceinline__ A inv_sqrt(A v)
{
    return A(1) / sqrt(v);
}

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

// 16 bytes past the caches.  Results that the eight L2s of 4 MB do not hold would only
// push out what is still read (16,384 bfloat16 columns of 4,096: 71.4 us by plain stores
// and 63.9; backward, 200,003 Float32 columns of 100: 51.6 and 49.2; products' results
// gain nothing: 8,192 columns 2048 -> 8192, 305 and 307 us).
constexpr int64_t STREAMED = 32 << 20;         // bytes of a result from which it is stored so
typedef uint32_t uint32x4_any __attribute__((ext_vector_type(4), aligned(2), may_alias));

template <typename T>
__device__ __forceinline__ void stream_chunk(T *p, const T *v)
{
    uint32x4 u;
    __builtin_memcpy(&u, v, 16);
    __builtin_nontemporal_store((uint32x4_any)u, reinterpret_cast<uint32x4_any *>(p));
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

// Lane l of a column's LANES holds its chunks l, l + LANES, ..., packed as they are
// read: the few registers leave room for the waves that hide the reads.  weight and
// bias stay in registers over the columns that a workgroup takes.
template <typename T, int LANES, int VPL>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void layer_norm_kernel(
    int64_t d, int64_t cols, const T *X, int64_t ldx, const T *__restrict__ weight, const T *__restrict__ bias,
    typename Elem<T>::Acc eps, T *Y, int64_t ldy, typename Elem<T>::Acc *__restrict__ stats, int64_t lds_, bool streamed)
{
    using A = typename Elem<T>::Acc;
    constexpr int CH = 16 / sizeof(T), NT = LANES > 256 ? LANES : 256, COLS = NT / LANES;
    __shared__ A s_red[NT / 64];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const A len = A(d);                            // divided by: a constant column's mean is exact
    uint32x4 w[VPL], b[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int64_t at = (int64_t)(lane + LANES * i) * CH;
        w[i] = read_raw(weight + at, weight ? d - at : 0);
        b[i] = read_raw(bias + at, bias ? d - at : 0);
    }
    for (int64_t c0 = (int64_t)blockIdx.x * COLS; c0 < cols; c0 += (int64_t)gridDim.x * COLS) {
        const int64_t c = c0 + sub;
        const bool live = c < cols, over = sizeof(T) == 2 && c + 1 < cols && d >= CH;
        uint32x4 x[VPL];
        A f[CH], sum[1] = {A(0)};
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t at = (int64_t)(lane + LANES * i) * CH;
            x[i] = read_raw(X + c * ldx + at, live ? d - at : 0, over);
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t left = live ? d - (int64_t)(lane + LANES * i) * CH : 0;
            values<T>(x[i], f);
#pragma unroll
            for (int j = 0; j < CH; ++j)
                if (j < left) sum[0] += f[j];
        }
        column_sum<LANES>(sum, s_red);
        const A mean = sum[0] / len;
        A sq[1] = {A(0)};
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t left = d - (int64_t)(lane + LANES * i) * CH;
            values_again<T>(x[i], f);
#pragma unroll
            for (int j = 0; j < CH; ++j)
                if (j < left) sq[0] += (f[j] - mean) * (f[j] - mean);
        }
        column_sum<LANES>(sq, s_red);
        const A rstd = inv_sqrt(sq[0] / len + eps);
        if (!live) continue;
        if (stats && lane == 0) {
            stats[c * lds_] = mean;
            stats[c * lds_ + 1] = rstd;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t at = (int64_t)(lane + LANES * i) * CH, left = d - at;
            if (left <= 0) continue;
            A v[CH];
            values_again<T>(x[i], f);
#pragma unroll
            for (int j = 0; j < CH; ++j) f[j] = (f[j] - mean) * rstd;
            if (weight) {
                values_again<T>(w[i], v);
#pragma unroll
                for (int j = 0; j < CH; ++j) f[j] *= v[j];
            }
            if (bias) {
                values_again<T>(b[i], v);
#pragma unroll
                for (int j = 0; j < CH; ++j) f[j] += v[j];
            }
            write_chunk(Y + c * ldy + at, left, f, streamed);
        }
    }
}

// Columns of any length: each pass reads them again.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(
    int64_t d, int64_t cols, const T *X, int64_t ldx, const T *__restrict__ weight, const T *__restrict__ bias,
    typename Elem<T>::Acc eps, T *Y, int64_t ldy, typename Elem<T>::Acc *__restrict__ stats, int64_t lds_)
{
    using A = typename Elem<T>::Acc;
    constexpr int CH = 16 / sizeof(T);
    __shared__ A s_red[16];
    const A len = A(d);
    for (int64_t c = blockIdx.x; c < cols; c += gridDim.x) {
        A sum[1] = {A(0)}, f[CH];
        for (int64_t at = (int64_t)threadIdx.x * CH; at < d; at += 1024 * CH) {
            read_chunk(X + c * ldx + at, d - at, f);
#pragma unroll
            for (int j = 0; j < CH; ++j) sum[0] += f[j];
        }
        column_sum<1024>(sum, s_red);
        const A mean = sum[0] / len;
        A sq[1] = {A(0)};
        for (int64_t at = (int64_t)threadIdx.x * CH; at < d; at += 1024 * CH) {
            read_chunk(X + c * ldx + at, d - at, f);
#pragma unroll
            for (int j = 0; j < CH; ++j)
                if (j < d - at) sq[0] += (f[j] - mean) * (f[j] - mean);
        }
        column_sum<1024>(sq, s_red);
        const A rstd = inv_sqrt(sq[0] / len + eps);
        if (stats && threadIdx.x == 0) {
            stats[c * lds_] = mean;
            stats[c * lds_ + 1] = rstd;
        }
        for (int64_t at = (int64_t)threadIdx.x * CH; at < d; at += 1024 * CH) {
            A w[CH];
            read_chunk(X + c * ldx + at, d - at, f);
#pragma unroll
            for (int j = 0; j < CH; ++j) f[j] = (f[j] - mean) * rstd;
            if (weight) {
                read_chunk(weight + at, d - at, w);
#pragma unroll
                for (int j = 0; j < CH; ++j) f[j] *= w[j];
            }
            if (bias) {
                read_chunk(bias + at, d - at, w);
#pragma unroll
                for (int j = 0; j < CH; ++j) f[j] += w[j];
            }
            write_chunk(Y + c * ldy + at, d - at, f);
        }
    }
}

// ------------------------------------------------------------------- gradients

// parts[workgroup][0] and [1] (of d values each) get the workgroup's share of
// dweight and dbias.
template <typename T, int LANES, int VPL>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void layer_norm_grad_kernel(
    int64_t d, int64_t cols, const T *__restrict__ X, int64_t ldx, const T *dY, int64_t lddy,
    const typename Elem<T>::Acc *__restrict__ stats, int64_t lds_, const T *__restrict__ weight, T *dX, int64_t lddx,
    typename Elem<T>::Acc *__restrict__ parts, bool streamed)
{
    using A = typename Elem<T>::Acc;
    constexpr int CH = 16 / sizeof(T), NT = LANES > 256 ? LANES : 256, COLS = NT / LANES, SPAN = LANES * VPL * CH;
    __shared__ A s_red[2 * (NT / 64)];
    __shared__ A s_part[COLS > 1 ? COLS * SPAN : 1];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const A len = A(d);
    A dw[VPL][CH], db[VPL][CH];
#pragma unroll
    for (int i = 0; i < VPL; ++i)
#pragma unroll
        for (int j = 0; j < CH; ++j) dw[i][j] = db[i][j] = A(0);
    uint32x4 w[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int64_t at = (int64_t)(lane + LANES * i) * CH;
        w[i] = read_raw(weight + at, weight ? d - at : 0);
    }
    for (int64_t c0 = (int64_t)blockIdx.x * COLS; c0 < cols; c0 += (int64_t)gridDim.x * COLS) {
        const int64_t c = c0 + sub;
        const bool live = c < cols, over = sizeof(T) == 2 && c + 1 < cols && d >= CH;
        const A mean = live ? stats[c * lds_] : A(0), rstd = live ? stats[c * lds_ + 1] : A(0);
        uint32x4 x[VPL], y[VPL];
        A sum[2] = {A(0), A(0)};
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t at = (int64_t)(lane + LANES * i) * CH, left = live ? d - at : 0;
            x[i] = read_raw(X + c * ldx + at, left, over);
            y[i] = read_raw(dY + c * lddy + at, left, over);
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t left = live ? d - (int64_t)(lane + LANES * i) * CH : 0;
            A h[CH], g[CH], v[CH];
            values<T>(x[i], h);
            values<T>(y[i], g);
            if (weight) values_again<T>(w[i], v);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                if (j >= left) continue;
                h[j] = (h[j] - mean) * rstd;
                dw[i][j] += g[j] * h[j];
                db[i][j] += g[j];
                if (weight) g[j] *= v[j];
                sum[0] += g[j];
                sum[1] += g[j] * h[j];
            }
        }
        if (!dX) continue;
        column_sum<LANES>(sum, s_red);
        if (!live) continue;
        const A m0 = sum[0] / len, m1 = sum[1] / len;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int64_t at = (int64_t)(lane + LANES * i) * CH, left = d - at;
            if (left <= 0) continue;
            A h[CH], g[CH], v[CH];
            values_again<T>(x[i], h);
            values_again<T>(y[i], g);
            if (weight) values_again<T>(w[i], v);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                if (weight) g[j] *= v[j];
                g[j] = rstd * (g[j] - m0 - (h[j] - mean) * rstd * m1);
            }
            write_chunk(dX + c * lddx + at, left, g, streamed);
        }
    }
    if (!parts) return;
    A *p = parts + (int64_t)blockIdx.x * 2 * d;
#pragma unroll
    for (int q = 0; q < 2; ++q, p += d) {
        if constexpr (COLS == 1) {
#pragma unroll
            for (int i = 0; i < VPL; ++i)
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    const int64_t at = (int64_t)(lane + LANES * i) * CH + j;
                    if (at < d) p[at] = q ? db[i][j] : dw[i][j];
                }
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < VPL; ++i)
#pragma unroll
                for (int j = 0; j < CH; ++j) s_part[sub * SPAN + (lane + LANES * i) * CH + j] = q ? db[i][j] : dw[i][j];
            __syncthreads();
            for (int at = threadIdx.x; at < SPAN && at < d; at += NT) {
                A s = A(0);
#pragma unroll
                for (int u = 0; u < COLS; ++u) s += s_part[u * SPAN + at];
                p[at] = s;
            }
        }
    }
}

// dX of columns of any length.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_grad_long_kernel(
    int64_t d, int64_t cols, const T *__restrict__ X, int64_t ldx, const T *dY, int64_t lddy,
    const typename Elem<T>::Acc *__restrict__ stats, int64_t lds_, const T *__restrict__ weight, T *dX, int64_t lddx)
{
    using A = typename Elem<T>::Acc;
    constexpr int CH = 16 / sizeof(T);
    __shared__ A s_red[32];
    const A len = A(d);
    for (int64_t c = blockIdx.x; c < cols; c += gridDim.x) {
        const A mean = stats[c * lds_], rstd = stats[c * lds_ + 1];
        A sum[2] = {A(0), A(0)}, h[CH], g[CH], w[CH];
        for (int64_t at = (int64_t)threadIdx.x * CH; at < d; at += 1024 * CH) {
            read_chunk(X + c * ldx + at, d - at, h);
            read_chunk(dY + c * lddy + at, d - at, g);
            if (weight) read_chunk(weight + at, d - at, w);
#pragma unroll
            for (int j = 0; j < CH; ++j)
                if (j < d - at) {
                    const A t = weight ? g[j] * w[j] : g[j];
                    sum[0] += t;
                    sum[1] += t * ((h[j] - mean) * rstd);
                }
        }
        column_sum<1024>(sum, s_red);
        const A a = sum[0] / len, b = sum[1] / len;
        for (int64_t at = (int64_t)threadIdx.x * CH; at < d; at += 1024 * CH) {
            read_chunk(X + c * ldx + at, d - at, h);
            read_chunk(dY + c * lddy + at, d - at, g);
            if (weight) read_chunk(weight + at, d - at, w);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const A t = weight ? g[j] * w[j] : g[j];
                g[j] = rstd * (t - a - (h[j] - mean) * rstd * b);
            }
            write_chunk(dX + c * lddx + at, d - at, g);
        }
    }
}

// Their dweight and dbias: a workgroup takes `per` columns of 256 chunks' rows.
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_weight_kernel(
    int64_t d, int64_t cols, const T *__restrict__ X, int64_t ldx, const T *__restrict__ dY, int64_t lddy,
    const typename Elem<T>::Acc *__restrict__ stats, int64_t lds_, int64_t per, typename Elem<T>::Acc *__restrict__ parts)
{
    using A = typename Elem<T>::Acc;
    constexpr int CH = 16 / sizeof(T);
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * CH, left = d - at;
    if (left <= 0) return;
    A dw[CH], db[CH], x[CH], g[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) dw[j] = db[j] = A(0);
    const int64_t c0 = (int64_t)blockIdx.y * per, c1 = c0 + per < cols ? c0 + per : cols;
    for (int64_t c = c0; c < c1; ++c) {
        const A mean = stats[c * lds_], rstd = stats[c * lds_ + 1];
        read_chunk(X + c * ldx + at, left, x);
        read_chunk(dY + c * lddy + at, left, g);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            dw[j] += g[j] * ((x[j] - mean) * rstd);
            db[j] += g[j];
        }
    }
    A *p = parts + (int64_t)blockIdx.y * 2 * d + at;
#pragma unroll
    for (int j = 0; j < CH; ++j)
        if (j < left) {
            p[j] = dw[j];
            p[d + j] = db[j];
        }
}

// The sums of `count` workgroups' shares, in order: 32 values by 32 shares.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_parts_kernel(int64_t d, int64_t count,
                                                                const typename Elem<T>::Acc *__restrict__ parts,
                                                                T *__restrict__ dweight, T *__restrict__ dbias)
{
    using A = typename Elem<T>::Acc;
    __shared__ A s_sum[32][33];
    T *out = blockIdx.y ? dbias : dweight;
    if (!out) return;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    // In turn where a launch would not take 32 threads for each of d (2^32 in all).
    for (int64_t at0 = (int64_t)blockIdx.x * 32; at0 < d; at0 += (int64_t)gridDim.x * 32) {
        const int64_t at = at0 + tx;
        const A *p = parts + blockIdx.y * d + at;
        A s = A(0);
        if (at < d) {
#pragma unroll 8
            for (int64_t i = ty; i < count; i += 32) s += p[i * 2 * d];
        }
        __syncthreads();
        s_sum[ty][tx] = s;
        __syncthreads();
        if (ty == 0 && at < d) {
            A t = A(0);
#pragma unroll
            for (int q = 0; q < 32; ++q) t += s_sum[q][tx];
            out[at] = T(t);
        }
    }
}

// f(std::integral_constant lanes, ... chunks a lane) for a column of d values;
// false if it is too long for the registers.
template <int L, int V> struct Span { static constexpr int lanes = L, vpl = V; };

template <bool GRAD, typename T, typename F>
bool by_span(int64_t d, F &&f)
{
    const int64_t chunks = (d * (int64_t)sizeof(T) + 15) / 16;
    if (chunks <= 16) f(Span<16, 1>());
    else if (chunks <= 32) f(Span<32, 1>());
    else if (chunks <= 64) f(Span<64, 1>());
    else if (chunks <= 128) f(Span<64, 2>());
    else if (chunks <= 256) f(Span<64, 4>());
    else if (chunks <= 512) f(Span<GRAD ? 256 : 64, GRAD ? 2 : 8>());
    else if (chunks <= 1024) f(Span<256, 4>());
    else if (chunks <= 2048) f(Span<512, 4>());
    else return false;
    return true;
}

template <typename T>
int layer_norm(int64_t d, int64_t cols, const void *X, int64_t ldx, const void *weight, const void *bias, double eps, void *Y,
               int64_t ldy, void *stats, int64_t lds, hipStream_t s)
{
    using A = typename Elem<T>::Acc;
    const bool held = by_span<false, T>(d, [&](auto span) {
        constexpr int L = decltype(span)::lanes, V = decltype(span)::vpl, NT = L > 256 ? L : 256;
        const int64_t blocks = (cols + NT / L - 1) / (NT / L);
        hipLaunchKernelGGL((layer_norm_kernel<T, L, V>), dim3((unsigned)(blocks < LN_BLOCKS ? blocks : LN_BLOCKS)), dim3(NT), 0, s, d, cols,
                           (const T *)X, ldx, (const T *)weight, (const T *)bias, (A)eps, (T *)Y, ldy, (A *)stats, lds,
                           d * cols * (int64_t)sizeof(T) > STREAMED);
    });
    if (!held)
        hipLaunchKernelGGL((layer_norm_long_kernel<T>), dim3((unsigned)(cols < 8192 ? cols : 8192)), dim3(1024), 0, s, d, cols,
                           (const T *)X, ldx, (const T *)weight, (const T *)bias, (A)eps, (T *)Y, ldy, (A *)stats, lds);
    return check_launch("layer_norm_kernel");
}

template <typename T>
int layer_norm_grad(int64_t d, int64_t cols, const void *X, int64_t ldx, const void *dY, int64_t lddy, const void *stats,
                    int64_t lds, const void *weight, void *dX, int64_t lddx, void *dweight, void *dbias, jlust_stream_t stream)
{
    using A = typename Elem<T>::Acc;
    hipStream_t s = (hipStream_t)stream;
    const bool sums = dweight || dbias;
    int64_t count = 0;                             // workgroups with a share of the sums
    void *ws = nullptr;
    int st = JLUST_STATUS_SUCCESS;
    auto parts = [&](int64_t n) {
        count = n;
        if (sums && n) st = scratch(stream, sizeof(A) * 2 * d * n, &ws);
        return st;
    };
    const bool held = by_span<true, T>(d, [&](auto span) {
        constexpr int L = decltype(span)::lanes, V = decltype(span)::vpl, NT = L > 256 ? L : 256;
        int64_t blocks = (cols + NT / L - 1) / (NT / L);
        // As many as the CUs hold: each adds a share of 2 d sums to write and read
        // (9,001 x 2,047 half: 43 us with 512, 51 with 1,024, 62 with 2,048; 200,003 x
        // 100 Float32: 75, 51, 58).
        const int64_t most = V * 16 / (int64_t)sizeof(T) >= 32 ? 512 : 1024;
        if (blocks > most) blocks = most;
        if (parts(blocks) || !blocks) return;
        hipLaunchKernelGGL((layer_norm_grad_kernel<T, L, V>), dim3((unsigned)blocks), dim3(NT), 0, s, d, cols, (const T *)X, ldx,
                           (const T *)dY, lddy, (const A *)stats, lds, (const T *)weight, (T *)dX, lddx, (A *)ws,
                           d * cols * (int64_t)sizeof(T) > STREAMED);
        st = check_launch("layer_norm_grad_kernel");
    });
    if (!held && cols) {
        if (sums) {                                // before dX, which may be dY
            const int64_t span = 256 * 16 / (int64_t)sizeof(T), blocks_d = (d + span - 1) / span;
            int64_t per = (cols * blocks_d + 1023) / 1024;
            if (per < 16) per = 16;
            if (!parts((cols + per - 1) / per)) {
                hipLaunchKernelGGL((layer_norm_weight_kernel<T>), dim3((unsigned)blocks_d, (unsigned)count), dim3(256), 0, s, d,
                                   cols, (const T *)X, ldx, (const T *)dY, lddy, (const A *)stats, lds, per, (A *)ws);
                st = check_launch("layer_norm_weight_kernel");
            }
        }
        if (!st && dX) {
            hipLaunchKernelGGL((layer_norm_grad_long_kernel<T>), dim3((unsigned)(cols < 8192 ? cols : 8192)), dim3(1024), 0, s, d,
                               cols, (const T *)X, ldx, (const T *)dY, lddy, (const A *)stats, lds, (const T *)weight, (T *)dX,
                               lddx);
            st = check_launch("layer_norm_grad_long_kernel");
        }
    }
    if (st || !sums) return st;
    hipLaunchKernelGGL((layer_norm_parts_kernel<T>), dim3((unsigned)(d < 1 << 26 ? (d + 31) / 32 : 1 << 21), 2), dim3(1024), 0, s, d, count,
                       (const A *)ws, (T *)dweight, (T *)dbias);
    return check_launch("layer_norm_parts_kernel");
}

int check(const char *who, int32_t value_type, int64_t d, int64_t cols, int64_t lds, const void *stats)
{
    if (value_type < JLUST_VALUE_F64 || value_type > JLUST_VALUE_BF16)
        return fail(JLUST_STATUS_UNSUPPORTED_VALUE_TYPE, "%s: unknown value type %d", who, value_type);
    if (d < 0 || cols < 0) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: negative extent", who);
    if (d >= (int64_t)1 << 31 || cols >= (int64_t)1 << 31)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: an extent of 2^31 or more", who);
    if (stats && cols > 1 && lds < 2)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: stats have leading dimension %lld", who, (long long)lds);
    return JLUST_STATUS_SUCCESS;
}

int check_ld(const char *who, const char *name, const void *p, int64_t d, int64_t cols, int64_t ld, bool needed)
{
    if (!p) {
        if (needed && d && cols) return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %s is null", who, name);
        return JLUST_STATUS_SUCCESS;
    }
    if (cols > 1 && ld < d)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %s has leading dimension %lld, its columns %lld rows", who, name,
                    (long long)ld, (long long)d);
    return JLUST_STATUS_SUCCESS;
}

}  // namespace
}  // namespace jlust

using namespace jlust;

extern "C" int jlust_hip_layer_norm(int32_t value_type, int64_t d, int64_t cols, const void *X, int64_t ldx,
                                    const void *weight, const void *bias, double eps, void *Y, int64_t ldy, void *stats,
                                    int64_t lds, jlust_stream_t stream)
{
    clear_error();
    const char *who = "layer_norm";
    if (int st = check(who, value_type, d, cols, lds, stats)) return st;
    if (int st = check_ld(who, "X", X, d, cols, ldx, true)) return st;
    if (int st = check_ld(who, "Y", Y, d, cols, ldy, true)) return st;
    if (!(eps >= 0)) return fail(JLUST_STATUS_INVALID_ARGUMENT, "layer_norm: eps is negative or NaN");
    if (int st = require_device(nullptr)) return st;
    if (d == 0 || cols == 0) return JLUST_STATUS_SUCCESS;
    hipStream_t s = (hipStream_t)stream;
    switch (value_type) {
    case JLUST_VALUE_F64: return layer_norm<double>(d, cols, X, ldx, weight, bias, eps, Y, ldy, stats, lds, s);
    case JLUST_VALUE_F32: return layer_norm<float>(d, cols, X, ldx, weight, bias, eps, Y, ldy, stats, lds, s);
    case JLUST_VALUE_F16: return layer_norm<_Float16>(d, cols, X, ldx, weight, bias, eps, Y, ldy, stats, lds, s);
    default: return layer_norm<__bf16>(d, cols, X, ldx, weight, bias, eps, Y, ldy, stats, lds, s);
    }
}

extern "C" int jlust_hip_layer_norm_grad(int32_t value_type, int64_t d, int64_t cols, const void *X, int64_t ldx,
                                         const void *dY, int64_t lddy, const void *stats, int64_t lds, const void *weight,
                                         void *dX, int64_t lddx, void *dweight, void *dbias, jlust_stream_t stream)
{
    clear_error();
    const char *who = "layer_norm_grad";
    if (int st = check(who, value_type, d, cols, lds, stats)) return st;
    if (int st = check_ld(who, "X", X, d, cols, ldx, true)) return st;
    if (int st = check_ld(who, "dY", dY, d, cols, lddy, true)) return st;
    if (int st = check_ld(who, "dX", dX, d, cols, lddx, false)) return st;
    if (!stats && d && cols) return fail(JLUST_STATUS_INVALID_ARGUMENT, "layer_norm_grad: stats are null");
    if (int st = require_device(nullptr)) return st;
    if (d == 0) return JLUST_STATUS_SUCCESS;
    switch (value_type) {
    case JLUST_VALUE_F64:
        return layer_norm_grad<double>(d, cols, X, ldx, dY, lddy, stats, lds, weight, dX, lddx, dweight, dbias, stream);
    case JLUST_VALUE_F32:
        return layer_norm_grad<float>(d, cols, X, ldx, dY, lddy, stats, lds, weight, dX, lddx, dweight, dbias, stream);
    case JLUST_VALUE_F16:
        return layer_norm_grad<_Float16>(d, cols, X, ldx, dY, lddy, stats, lds, weight, dX, lddx, dweight, dbias, stream);
    default:
        return layer_norm_grad<__bf16>(d, cols, X, ldx, dY, lddy, stats, lds, weight, dX, lddx, dweight, dbias, stream);
    }
}

namespace jlust {
int preload_layer_norm()
{
    JLUST_PRELOAD_KERNEL((layer_norm_kernel<float, 64, 1>));
    return JLUST_STATUS_SUCCESS;
}
}  // namespace jlust
