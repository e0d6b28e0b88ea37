// dropout.hip -- Y = X .* mask .* scale (.+ R) with a mask that is made where it is
// used: field i % 8, of 16 bits, of Philox4x32-10 (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter {i / 8, j, offset}
// under the key `seed` says whether element (i, j) is kept.  The mask goes by the
// element's place alone, so the backward pass makes it again.
#include "column_chunks.hpp"

#include <cmath>

namespace jlust {
namespace {

// 8 fields of 16 bits: of word w the low half is field 2 w, the high half 2 w + 1.
__device__ __forceinline__ uint32x4 philox(uint32x4 c, uint32_t k0, uint32_t k1)
{
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
        c = uint32x4{(uint32_t)(b >> 32) ^ c[1] ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c[3] ^ k1, (uint32_t)a};
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}

// A thread makes 8 elements of a column, one counter's.  Stores go through the caches: a
// thread's 32 bytes of Float32 in two of them, past the caches, are written by half lines
// (100 x 200,003: 41.5 us and 32.7; 16-bit 70.9 and 71.2 of 4,096 x 16,384 with R).
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void dropout_kernel(int64_t d, int64_t cols, Divider eights, const T *X, int64_t ldx, const T *R, int64_t ldr, T *Y,
                                                      int64_t ldy, uint32_t dropped, typename Elem<T>::Acc scale, uint64_t seed,
                                                      uint64_t offset, const int64_t *__restrict__ state)
{
    using A = typename Elem<T>::Acc;
    constexpr int CH = 16 / sizeof(T), PARTS = 8 / CH;
    if (state) {
        seed = (uint64_t)state[0];
        offset = (uint64_t)state[1];
    }
    for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < eights.d * cols; n += (int64_t)gridDim.x * 256) {
        const int64_t j = eights.of(n), e = n - j * eights.d, i = e * 8;
        uint32x4 x[PARTS], r[PARTS];
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
            x[q] = read_at<WHOLE>(X + j * ldx, i + q * CH, d);
            r[q] = uint32x4{0, 0, 0, 0};
        }
        if (R)
#pragma unroll
            for (int q = 0; q < PARTS; ++q) r[q] = read_at<WHOLE>(R + j * ldr, i + q * CH, d);
        const uint32x4 u = philox(uint32x4{(uint32_t)e, (uint32_t)j, (uint32_t)offset, (uint32_t)(offset >> 32)}, (uint32_t)seed,
                                  (uint32_t)(seed >> 32));
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
            A f[CH], g[CH];
            values<T>(x[q], f);
            values<T>(r[q], g);
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                const int at = q * CH + k;
                const uint32_t field = u[at / 2] >> (at & 1) * 16 & 0xFFFF;
                f[k] = (field >= dropped ? f[k] * scale : A(0)) + g[k];
            }
            write_at<WHOLE>(Y + j * ldy, i + q * CH, d, f);
        }
    }
}

}  // namespace
}  // namespace jlust

using namespace jlust;

extern "C" int jlust_hip_dropout(int32_t value_type, int64_t d, int64_t cols, const void *X, int64_t ldx, const void *R, int64_t ldr,
                                 void *Y, int64_t ldy, double p, uint64_t seed, uint64_t offset, const int64_t *state,
                                 jlust_stream_t stream)
{
    clear_error();
    const char *who = "dropout";
    if (int st = check_extents(who, value_type, d, cols)) return st;
    if (int st = check_matrix(who, "X", X, d, cols, ldx, true)) return st;
    if (int st = check_matrix(who, "R", R, d, cols, ldr, false)) return st;
    if (int st = check_matrix(who, "Y", Y, d, cols, ldy, true)) return st;
    if (!(p >= 0 && p <= 1)) return fail(JLUST_STATUS_INVALID_ARGUMENT, "dropout: p = %g is no probability", p);
    if (int st = require_device(nullptr)) return st;
    if (d == 0 || cols == 0) return JLUST_STATUS_SUCCESS;
    const uint32_t dropped = (uint32_t)std::lround(p * 65536);
    const double scale = dropped < 65536 ? 65536.0 / (65536 - dropped) : 0.0;
    return with_type(value_type, [&](auto z) {
        using T = decltype(z);
        using A = typename Elem<T>::Acc;
        const int64_t eights = (d + 7) / 8;
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(column_blocks(eights * cols, 256)), dim3(256), 0, (hipStream_t)stream, d, cols,
                               Divider(eights, eights * cols), (const T *)X, ldx, (const T *)R, ldr, (T *)Y, ldy, dropped, (A)scale,
                               seed, offset, state);
        };
        if (d % (16 / sizeof(T)) == 0) launch(dropout_kernel<T, true>);
        else launch(dropout_kernel<T, false>);
        return check_launch("dropout_kernel");
    });
}

namespace jlust {
int preload_dropout()
{
    JLUST_PRELOAD_KERNEL((dropout_kernel<float, true>));
    return JLUST_STATUS_SUCCESS;
}
}  // namespace jlust
