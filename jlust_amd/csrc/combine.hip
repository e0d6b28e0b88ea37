// combine.hip -- the weighted sum of the columns that belong together, and its
// gradients: column t of Y is the sum over c of weights[c, t] X[:, copies t + c].
//
//   dX[:, copies t + c] = weights[c, t] dY[:, t],   dweights[c, t] = <X[:, copies t + c], dY[:, t]>
//
// Both are bound by memory: every operand is read once, in chunks of 16 bytes.
#include "column_chunks.hpp"

namespace jlust {
namespace {

// A thread makes a chunk of a column of Y.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void combine_kernel(int64_t d, int64_t cols, Divider chunks, int copies, const T *__restrict__ X, int64_t ldx,
                                                      const typename Elem<T>::Acc *__restrict__ weights, int64_t ldw, const T *R,
                                                      int64_t ldr, T *Y, int64_t ldy, bool streamed)
{
    using A = typename Elem<T>::Acc;
    constexpr int CH = 16 / sizeof(T), AHEAD = 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks.d * cols; i += (int64_t)gridDim.x * 256) {
        const int64_t t = chunks.of(i), at = (i - t * chunks.d) * CH, left = WHOLE ? CH : d - at;
        const T *x = X + t * copies * ldx + at;
        const A *w = weights + t * ldw;
        A sum[CH], f[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) sum[j] = A(0);
        const uint32x4 r = read_raw(R + t * ldr + at, R ? left : 0);
        for (int k = 0; k < copies; k += AHEAD) {
            uint32x4 v[AHEAD];
            A by[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                by[q] = k + q < copies ? w[k + q] : A(0);
                v[q] = read_raw(x + (k + q) * ldx, by[q] != A(0) ? left : 0);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                values<T>(v[q], f);
#pragma unroll
                for (int j = 0; j < CH; ++j) sum[j] += by[q] * f[j];
            }
        }
        values<T>(r, f);
#pragma unroll
        for (int j = 0; j < CH; ++j) sum[j] += f[j];
        write_chunk(Y + t * ldy + at, left, sum, streamed);
    }
}

// LANES lanes take column t of dY, COPIES of its columns of X at a time.
template <typename T, int LANES, int COPIES>
__global__ __launch_bounds__(256) void combine_grad_kernel(int64_t d, int64_t cols, int copies, const T *X, int64_t ldx,
                                                           const typename Elem<T>::Acc *__restrict__ weights, int64_t ldw,
                                                           const T *__restrict__ dY, int64_t lddy, T *dX, int64_t lddx,
                                                           typename Elem<T>::Acc *__restrict__ dweights, int64_t lddw, bool streamed)
{
    using A = typename Elem<T>::Acc;
    constexpr int CH = 16 / sizeof(T), COLS = 256 / LANES;
    __shared__ A s_red[COPIES * 4];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    for (int64_t c0 = (int64_t)blockIdx.x * COLS; c0 < cols; c0 += (int64_t)gridDim.x * COLS) {
        const int64_t t = c0 + sub;
        const bool live = t < cols;
        for (int k = 0; k < copies; k += COPIES) {
            A by[COPIES], dot[COPIES];
#pragma unroll
            for (int q = 0; q < COPIES; ++q) {
                by[q] = dX && live && k + q < copies ? weights[t * ldw + k + q] : A(0);     // a call without dX has none
                dot[q] = A(0);
            }
            for (int64_t at = (int64_t)lane * CH; live && at < d; at += LANES * CH) {
                const int64_t left = d - at;
                uint32x4 v[COPIES];
                A g[CH], f[CH];
#pragma unroll
                for (int q = 0; q < COPIES; ++q)
                    v[q] = read_raw(X + (t * copies + k + q) * ldx + at, dweights && k + q < copies ? left : 0);
                read_chunk(dY + t * lddy + at, left, g);
#pragma unroll
                for (int q = 0; q < COPIES; ++q) {
                    values<T>(v[q], f);
#pragma unroll
                    for (int j = 0; j < CH; ++j) dot[q] += f[j] * g[j];
                    if (!dX || k + q >= copies) continue;
#pragma unroll
                    for (int j = 0; j < CH; ++j) f[j] = by[q] * g[j];
                    write_chunk(dX + (t * copies + k + q) * lddx + at, left, f, streamed);
                }
            }
            if (!dweights) continue;
            column_sum<LANES>(dot, s_red);
            if (live && lane == 0)
#pragma unroll
                for (int q = 0; q < COPIES; ++q)
                    if (k + q < copies) dweights[t * lddw + k + q] = dot[q];
        }
    }
}

template <typename T, int LANES>
int launch_grad(int64_t d, int64_t cols, int copies, const void *X, int64_t ldx, const void *weights, int64_t ldw, const void *dY,
                int64_t lddy, void *dX, int64_t lddx, void *dweights, int64_t lddw, hipStream_t s)
{
    using A = typename Elem<T>::Acc;
    const unsigned blocks = column_blocks(cols, 256 / LANES);
    const bool streamed = d * cols * copies * (int64_t)sizeof(T) > STREAMED;
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, s, d, cols, copies, (const T *)X, ldx, (const A *)weights, ldw,
                           (const T *)dY, lddy, (T *)dX, lddx, (A *)dweights, lddw, streamed);
    };
    if (copies == 1) launch(combine_grad_kernel<T, LANES, 1>);
    else if (copies == 2) launch(combine_grad_kernel<T, LANES, 2>);
    else launch(combine_grad_kernel<T, LANES, 4>);
    return check_launch("combine_grad_kernel");
}

int check_copies(const char *who, int64_t cols, int64_t copies)
{
    if (copies < 1 || copies * cols >= (int64_t)1 << 31 || copies >= (int64_t)1 << 31)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "%s: %lld copies of %lld columns are not within [1, 2^31)", who,
                    (long long)copies, (long long)cols);
    return JLUST_STATUS_SUCCESS;
}

}  // namespace
}  // namespace jlust

using namespace jlust;

extern "C" int jlust_hip_combine(int32_t value_type, int64_t d, int64_t cols, int64_t copies, const void *X, int64_t ldx,
                                 const void *weights, int64_t ldw, const void *R, int64_t ldr, void *Y, int64_t ldy,
                                 jlust_stream_t stream)
{
    clear_error();
    const char *who = "combine";
    if (int st = check_extents(who, value_type, d, cols)) return st;
    if (int st = check_copies(who, cols, copies)) return st;
    if (int st = check_matrix(who, "X", X, d, cols * copies, ldx, true)) return st;
    if (int st = check_matrix(who, "weights", weights, copies, cols, ldw, d > 0)) return st;
    if (int st = check_matrix(who, "R", R, d, cols, ldr, false)) return st;
    if (int st = check_matrix(who, "Y", Y, d, cols, ldy, true)) return st;
    if (int st = require_device(nullptr)) return st;
    if (d == 0 || cols == 0) return JLUST_STATUS_SUCCESS;
    return with_type(value_type, [&](auto z) {
        using T = decltype(z);
        using A = typename Elem<T>::Acc;
        constexpr int64_t CH = 16 / sizeof(T);
        const int64_t chunks = (d + CH - 1) / CH;
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(column_blocks(chunks * cols, 256)), dim3(256), 0, (hipStream_t)stream, d, cols,
                               Divider(chunks, chunks * cols), (int)copies, (const T *)X, ldx, (const A *)weights, ldw,
                               (const T *)R, ldr, (T *)Y, ldy, d * cols * (int64_t)sizeof(T) > STREAMED);
        };
        if (d % CH == 0) launch(combine_kernel<T, true>);
        else launch(combine_kernel<T, false>);
        return check_launch("combine_kernel");
    });
}

extern "C" int jlust_hip_combine_grad(int32_t value_type, int64_t d, int64_t cols, int64_t copies, const void *X, int64_t ldx,
                                      const void *weights, int64_t ldw, const void *dY, int64_t lddy, void *dX, int64_t lddx,
                                      void *dweights, int64_t lddw, jlust_stream_t stream)
{
    clear_error();
    const char *who = "combine_grad";
    if (int st = check_extents(who, value_type, d, cols)) return st;
    if (int st = check_copies(who, cols, copies)) return st;
    // X is read for dweights alone, the weights for dX alone.
    if (int st = check_matrix(who, "X", dweights ? X : nullptr, d, cols * copies, ldx, dweights != nullptr)) return st;
    if (int st = check_matrix(who, "weights", dX ? weights : nullptr, copies, cols, ldw, dX != nullptr)) return st;
    if (int st = check_matrix(who, "dY", dY, d, cols, lddy, true)) return st;
    if (int st = check_matrix(who, "dX", dX, d, cols * copies, lddx, false)) return st;
    if (int st = check_matrix(who, "dweights", dweights, copies, cols, lddw, false)) return st;
    if (int st = require_device(nullptr)) return st;
    if (cols == 0 || (!dX && !dweights)) return JLUST_STATUS_SUCCESS;
    hipStream_t s = (hipStream_t)stream;
    return with_type(value_type, [&](auto z) {
        using T = decltype(z);
        const int64_t chunks = (d * (int64_t)sizeof(T) + 15) / 16;
        auto go = [&](auto f) { return f(d, cols, (int)copies, X, ldx, weights, ldw, dY, lddy, dX, lddx, dweights, lddw, s); };
        // Few lanes for short columns, a workgroup's for long ones and where columns are few
        // (us by 16, 32, 64 and 256 lanes: 100,000 columns of 16 chunks, two copies, 21, 24, 38,
        // 120; 100,000 of 25 chunks 42, 33, 39, 126; 40,000 of 64 chunks, four copies, 73, 69, 66,
        // 112; 20,000 of 128 chunks 33, 33, 32, 35; 64 of them, eight copies, 16, 10, 6.7, 5.5;
        // 8,000 of 512 chunks 267, 251, 241, 211; 64 of them 55, 30, 17, 7.6).
        if (chunks <= 16) return go(launch_grad<T, 16>);
        if (chunks <= 32) return go(launch_grad<T, 32>);
        if (chunks <= 64 || (chunks < 192 && cols > 1024)) return go(launch_grad<T, 64>);
        return go(launch_grad<T, 256>);
    });
}

namespace jlust {
int preload_combine()
{
    JLUST_PRELOAD_KERNEL((combine_kernel<float, true>));
    return JLUST_STATUS_SUCCESS;
}
}  // namespace jlust
