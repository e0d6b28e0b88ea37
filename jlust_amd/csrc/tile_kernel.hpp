// tile_kernel.hpp -- the matrix-core kernel of tile_product.hpp.
#pragma once

#include "tile_product.hpp"
#include "wave.hpp"

#include <type_traits>

namespace jlust {

typedef uint32_t uint32x2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int intx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// One operand's tile of R rows by 128 bytes of k: global memory to registers to
// LDS.  kc: LDS row r holds its 8 chunks of 16 bytes at chunk ^ (r & 7), so the
// 16 rows that a wave reads at one k lie in different banks.  sc: LDS row k
// holds R elements; 16-bit ones have their 32-byte segments permuted by k, see
// `segment`.
template <typename T, bool KC, int R, int NT>
struct Stage {
    static constexpr int CH = 16 / sizeof(T);
    static constexpr int BK = 128 / sizeof(T);
    static constexpr int CHUNKS = R * 8;                       // R * 128 bytes
    static constexpr int CNT = (CHUNKS + NT - 1) / NT;
    static constexpr int PER = KC ? 8 : R / CH;                // chunks of one LDS row
    static constexpr int STEP = NT / PER;                      // LDS rows between a thread's chunks
    static constexpr bool WHOLE = CHUNKS % NT == 0;
    static_assert(NT % PER == 0, "a thread keeps its place in a row");

    const T *p[KC ? CNT : 1];
    int64_t ld;
    int64_t avail;                       // sc: elements from this thread's first one to the edge
    int64_t over;                        // sc: rows of k below this one may be read past the edge
    uint32x4 v[CNT];

    __device__ __forceinline__ static bool mine(int i) { return WHOLE || (int)threadIdx.x + i * NT < CHUNKS; }
    __device__ __forceinline__ static int place() { return threadIdx.x % PER; }
    __device__ __forceinline__ static int lds_row(int i) { return threadIdx.x / PER + i * STEP; }

    // Where the 32-byte segment of an LDS row lies: a transposed read takes 4
    // rows by 16 columns a lane group, and rows k, k+1, k+2, k+3, k+8, ... + 11
    // of one column at once; R * 2 bytes a row put them on the same banks.
    __device__ __forceinline__ static int segment(int seg, int k)
    {
        constexpr int MASK = R / 16 >= 8 ? 7 : R / 16 - 1;
        return seg ^ (((k & 3) | (k >> 1 & 4)) & MASK);
    }

    // `ks`: the operand's extent along k.
    __device__ __forceinline__ void init(const T *b, int64_t ld_, const int32_t *idx, int64_t r0, int64_t rend, int64_t ks)
    {
        ld = ld_;
        if constexpr (KC) {
#pragma unroll
            for (int i = 0; i < CNT; ++i) {
                int64_t r = r0 + lds_row(i);
                r = r < rend ? r : rend - 1;               // rows past the edge are computed and not stored
                if (idx) r = idx[r];
                p[i] = b + r * ld + place() * CH;
            }
        } else {
            const int64_t c = r0 + (int64_t)place() * CH;
            avail = rend - c;
            over = rend >= CH ? ks - 1 : 0;
            p[0] = b + c;
        }
    }

    // Reads the tile of [k0, k0 + BK); what lies past kend is zero.  sc: a chunk
    // over the edge takes the start of the next row with it (those columns are not
    // stored), and only the last row's is read by elements: with both kinds in a wave
    // every chunk waited for the one before (dW of 7168 x 111 over 4,600 columns,
    // Float32: 144 us and 111).
    __device__ __forceinline__ void load(int64_t k0, int64_t kend)
    {
        const uint32x4 zero = {0, 0, 0, 0};
        if constexpr (KC) {
            if (k0 + BK <= kend) {
#pragma unroll
                for (int i = 0; i < CNT; ++i)
                    if (mine(i)) v[i] = load_chunk(p[i] + k0);
            } else {
                const int64_t left = kend - k0 - place() * CH;
#pragma unroll
                for (int i = 0; i < CNT; ++i) {
                    v[i] = zero;
                    if (mine(i) && left > 0) v[i] = left >= CH ? load_chunk(p[i] + k0) : load_chunk_part(p[i] + k0, left);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < CNT; ++i) {
                const int64_t k = k0 + lds_row(i);
                v[i] = zero;
                if (mine(i) && k < kend && avail > 0) {
                    const T *q = p[0] + k * ld;
                    v[i] = avail >= CH || k < over ? load_chunk(q) : load_chunk_part(q, avail);
                }
            }
        }
    }

    __device__ __forceinline__ void store(char *lds) const
    {
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            if (!mine(i)) continue;
            const int r = lds_row(i), c = place();
            int at;
            if constexpr (KC) at = r * 128 + ((c ^ (r & 7)) << 4);
            else if constexpr (sizeof(T) == 2) at = r * R * 2 + (segment(c >> 1, r) << 5) + ((c & 1) << 4);
            else at = r * R * (int)sizeof(T) + (c << 4);
            *reinterpret_cast<uint32x4 *>(lds + at) = v[i];
        }
    }

    // The 16 bytes of row r at chunk c (kc).
    __device__ __forceinline__ static uint32x4 chunk(const char *lds, int r, int c)
    {
        return *reinterpret_cast<const uint32x4 *>(lds + r * 128 + ((c ^ (r & 7)) << 4));
    }

    // 16-bit operands: what lane (li, g) feeds to a 16x16x32 step: row
    // 16*tile + li, k = 32*s + 8*g .. + 7.  8-bit ones along k: 16 of k to a 16x16x64
    // step in the place of 8.
    __device__ __forceinline__ static uint32x4 frag16(const char *lds, int tile, int s)
    {
        const int li = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
        if constexpr (KC) {
            return chunk(lds, 16 * tile + li, g + 4 * s);
        } else {
            uint32x4 out;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = 32 * s + 8 * g + 4 * h + (li >> 2);
                const int at = k * R * 2 + (segment(tile, k) << 5) + ((li & 3) << 3);
                const shortx4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) shortx4 *)(lds + at));
                const uint32x2 u = __builtin_bit_cast(uint32x2, t);
                out[2 * h] = u[0];
                out[2 * h + 1] = u[1];
            }
            return out;
        }
    }

    // 32- and 64-bit operands: the values of 16-row tiles [0, TILES) from row r0
    // for the CH steps of half s of the k range: f[i][j] is lane (lr, g)'s, row
    // r0 + 16 i + lr at k = CH*(g + 4s) + j.
    template <int TILES>
    __device__ __forceinline__ static void frag(const char *lds, int r0, int lr, int g, int s, T (&f)[TILES][CH])
    {
        if constexpr (KC) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const uint32x4 c = chunk(lds, r0 + 16 * i + lr, g + 4 * s);
                __builtin_memcpy(f[i], &c, 16);
            }
        } else {
            const T *q = (const T *)lds + CH * (g + 4 * s) * R + r0 + lr;
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int i = 0; i < TILES; ++i) f[i][j] = q[j * R + 16 * i];
        }
    }
};

__device__ __forceinline__ floatx4 mma(uint32x4 a, uint32x4 b, floatx4 c, __bf16)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mma(uint32x4 a, uint32x4 b, floatx4 c, _Float16)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mma(uint32x4 a, uint32x4 b, floatx16 c, __bf16)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mma(uint32x4 a, uint32x4 b, floatx16 c, _Float16)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
__device__ __forceinline__ intx4 mma(uint32x4 a, uint32x4 b, intx4 c, int8_t)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), c, 0, 0, 0);
}
__device__ __forceinline__ intx16 mma(uint32x4 a, uint32x4 b, intx16 c, int8_t)
{
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mma(float a, float b, floatx4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ doublex4 mma(double a, double b, doublex4 c)
{
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}

// The first `count` (or all) of V values at p, and writing them.
template <int V, typename T>
__device__ __forceinline__ void load_some(const T *p, int64_t count, T *v)
{
    if (count >= V) {
        load_vec<V>(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = e < count ? p[e] : T(0);
    }
}

template <int V, typename T>
__device__ __forceinline__ void store_some(T *p, int64_t count, const T *v)
{
    if (count >= V) {
        store_vec<V>(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < count) p[e] = v[e];
    }
}

// V values of a group's bias from m on, zeros past the edge or without one.
template <int V, typename T>
__device__ __forceinline__ void load_bias(const TileArgs &a, int group, int64_t m, T *b)
{
    const bool some = a.bias && group < a.groups && m < a.m;
    load_some<V>((const T *)a.bias + group * a.gb + m, some ? a.m - m : 0, b);
}

// V sums of row `row` of C, columns mm ..: the epilogue; res: R's there.  finish_sum: of
// sums that have their bias.
template <int V, bool STREAM, typename T, typename A>
__device__ __forceinline__ void finish_sum(const TileArgs &a, const T *res, int64_t row, int64_t mm, A *s)
{
    const int64_t left = a.m - mm;
    T t[V];
    if (a.Z) {
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] = T(s[e]);
        store_some<V>((T *)a.Z + row * a.ldz + mm, left, t);
    }
    activate_all<sizeof(T) == 2, V>(a.act, s);
    if (a.R) {
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += A(res[e]);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = T(s[e]);
    if constexpr (STREAM && V * sizeof(T) == 16)
        if (a.streamed && left >= V) return stream_chunk((T *)a.C + row * a.ldc + mm, t);
    store_some<V>((T *)a.C + row * a.ldc + mm, left, t);
}

template <int V, typename T, typename A>
__device__ __forceinline__ void finish(const TileArgs &a, const T *bias, const T *res, int64_t row, int64_t mm, A *s)
{
    const int64_t left = a.m - mm;
    if (left <= 0) return;
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] += A(bias[e]);
    if (a.c_wide) {
        store_some<V>((A *)a.C + row * a.ldc + mm, left, s);
        return;
    }
    finish_sum<V, false, T, A>(a, res, row, mm, s);
}

// The scales of a group's V rows of P from m on (0 past the edge and in no group), and
// that of the row of Q that n stands for.
template <int V>
__device__ __forceinline__ void load_scales(const TileArgs &a, int group, int64_t m, float *by)
{
    load_some<V>(a.ps + group * a.gs + m, group < a.groups && m < a.m ? a.m - m : 0, by);
}

__device__ __forceinline__ float scale_of(const TileArgs &a, int group, int64_t n)
{
    return group < a.groups ? a.qs[a.qrow ? a.qrow[n] : n] : 0.0f;
}

// V sums times both scales, one after the other, so that no step leaves Float32's range
// where the result does not (the scales' product may): below the normal range a whole
// number times a scale is exact, and of qs = lo hi a part past 1 comes last.  (8,192
// bfloat16 columns 2048 -> 8192 with gelu 183.2 us by the scales' product and 184.8 so; rows
// with such a qs by a loop of their own cost Float32 results 10 % for want of registers.)
template <int V>
__device__ __forceinline__ void scale_sums(const int *sum, float qs, const float *by, const float *bias, float *f)
{
    const bool small = fabsf(qs) <= 1;
    const float lo = small ? qs : 1.0f, hi = small ? 1.0f : qs;
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = fmaf((float)sum[e] * lo * by[e], hi, bias[e]);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// What a workgroup does: its tile, the piece of k, the group, the rows of n and the
// k range.  Extents are below 2^31, and so are a launch's workgroups.
struct Work { int tm, piece, group, n0, nend, k0, kend; };

// Tile t of tiles_m x tiles_n: bands of 8 along n, m after m inside a band, so that
// neighbours share P and Q tiles.
__device__ __forceinline__ void tile_at(uint32_t t, uint32_t tiles_n, uint32_t tiles_m, int *tm, int *tn)
{
    const uint32_t band = t / (8 * tiles_m), in = t - band * 8 * tiles_m;
    const uint32_t wide = tiles_n - band * 8 < 8 ? tiles_n - band * 8 : 8;
    *tm = in / wide;
    *tn = band * 8 + in % wide;
}

// A launch's work in order: groups, pieces of k, tiles.  Each XCD takes a run of its
// own, the workgroups that run at once on one sharing tiles in its L2.  Groups of
// rows: first the tiles of columns in groups, by their number and not by the bound
// that the launch is sized for (with the empty ones at its end one XCD had nothing
// to do: 32 groups, a quarter of the columns in none, 187 us and 152), then those of
// the columns in none, which only store.  False where there is none.
template <bool KSUM, int BN, int BK>
__device__ __forceinline__ bool find_work(const TileArgs &a, Work *w)
{
    const uint32_t xcd = blockIdx.x % NUM_XCD, i = blockIdx.x / NUM_XCD, tiles_m = a.tiles_m, split = a.split;
    int tn;
    *w = Work{0, 0, 0, 0, (int)a.n, 0, (int)a.k};
    if (!KSUM && a.offsets) {
        // A lane holds every 64th group's rows; up to 63 groups are read once.
        const int lane = lane_id();
        const bool few = a.groups < 64;
        int lo = 0, hi = 0, live = 0;
        for (int g = lane; g <= a.groups; g += 64) {
            lo = a.offsets[g];
            hi = g < a.groups ? a.offsets[g + 1] : (int)a.n;
            if (g < a.groups) live += (hi - lo + BN - 1) / BN;
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) live += __shfl_xor(live, d, 64);
        live = uniform(live);
        const uint32_t tiles = live * tiles_m, total = tiles * split, per = (total + NUM_XCD - 1) / NUM_XCD;
        uint32_t t = xcd * per + i;
        if (i < per) {
            if (t >= total) return false;
            w->piece = t / tiles;
            tile_at(t % tiles, live, tiles_m, &w->tm, &tn);
        } else {
            t = (i - per) * NUM_XCD + xcd;
            w->piece = t % split;
            t /= split;
            w->tm = t % tiles_m;
            tn = live + t / tiles_m;
        }
        if (few) {
            const int runs = (hi - lo + BN - 1) / BN;
            int incl = runs;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int v = __shfl_up(incl, d, 64);
                if (lane >= d) incl += v;
            }
            const uint64_t mask = __ballot(tn < incl);
            if (mask == 0) return false;
            const int g = __ffsll((unsigned long long)mask) - 1;
            w->group = g;
            w->n0 = __shfl(lo + (tn - incl + runs) * BN, g, 64);
            w->nend = __shfl(hi, g, 64);
        } else {
            GroupRun r;
            if (!find_run(a.offsets, a.groups, a.n, tn, BN, &r)) return false;
            w->group = r.group;
            w->n0 = (int)r.begin;
            w->nend = (int)r.group_end;
        }
        if (w->group == a.groups) w->kend = 0;
    } else {
        const uint32_t tiles = tiles_m * (uint32_t)a.tiles_n;
        const uint32_t total = tiles * split * (KSUM && a.offsets ? a.groups : 1), per = (total + NUM_XCD - 1) / NUM_XCD;
        const uint32_t t = xcd * per + i;
        if (i >= per || t >= total) return false;
        tile_at(t % tiles, a.tiles_n, tiles_m, &w->tm, &tn);
        w->piece = t / tiles % split;
        w->n0 = tn * BN;
        if (KSUM && a.offsets) {
            w->group = t / tiles / split;
            w->k0 = a.offsets[w->group];
            w->kend = a.offsets[w->group + 1];
        }
    }
    if (split > 1) {
        const int piece = ((w->kend - w->k0 + a.split - 1) / a.split + BK - 1) / BK * BK;
        const int64_t lo = w->k0 + (int64_t)piece * w->piece, end = w->kend;
        w->k0 = (int)(lo < end ? lo : end);
        w->kend = (int)(lo + piece < end ? lo + piece : end);
    }
    *w = Work{uniform(w->tm), uniform(w->piece), uniform(w->group), uniform(w->n0), uniform(w->nend), uniform(w->k0),
              uniform(w->kend)};
    return true;
}

// The end of a wave's sums, TM along m by 16 * RUNS along n.  The matrix steps
// leave a lane 4 values of a row; 16 rows at a time go through the wave's part of
// the LDS tile (put(run, its place) writes them, chunk c of row r at chunk c ^
// (r & FLIP)), so that a lane ends 16 bytes of C and a row's lanes a whole line.
template <typename A, int TM> struct SumRows {
    static constexpr int USED = TM * (int)sizeof(A) / 16;
    static constexpr int CHUNKS = USED <= 4 ? 4 : USED <= 8 ? 8 : USED <= 16 ? 16 : USED <= 32 ? 32 : 64;
    static constexpr int FLIP = CHUNKS < 16 ? CHUNKS - 1 : 15, BYTES = 16 * CHUNKS * 16;
    __device__ __forceinline__ static int at(int r, int c) { return r * CHUNKS * 16 + ((c ^ (r & FLIP)) << 4); }
};

template <typename T, bool KSUM, int TM, int RUNS, typename Put>
__device__ __forceinline__ void finish_tile(const TileArgs &a, char *lds, int piece, int group, int n0, int nend, int64_t m0, Put &&put)
{
    using A = typename Elem<T>::Acc;
    using SR = SumRows<A, TM>;
    constexpr int CH = 16 / sizeof(T), ACH = 16 / sizeof(A), LANES = TM / CH, ROWS = 64 / LANES, ITER = (16 + ROWS - 1) / ROWS;
    const int lane = threadIdx.x & 63;
    const int r0 = lane < LANES * ROWS ? lane / LANES : 16;
    char *mine = lds + (threadIdx.x >> 6) * SR::BYTES;
    const int64_t m = m0 + lane % LANES * CH, left = a.m - m;
    TileArgs b = a;
    if constexpr (KSUM) b.C = (T *)a.C + group * a.gc;
    if (!a.offsets) b.groups = 1;
    T bias[CH];
    load_bias<CH>(b, group, m, bias);
    const int64_t part_rows = KSUM && a.offsets ? a.n * a.groups : a.n;
    const int64_t part_row = piece * part_rows + (KSUM ? group * a.n : 0);
#pragma unroll
    for (int run = 0; run < RUNS; ++run) {
        // What the rows need from memory, all of it before the first is used.
        int row[ITER];
        T res[ITER][CH];
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            const int r = r0 + it * ROWS, n = n0 + 16 * run + r;
            row[it] = r < 16 && n < nend && left > 0 ? n : -1;
        }
        if (!a.part && a.crow) {
#pragma unroll
            for (int it = 0; it < ITER; ++it) row[it] = row[it] >= 0 ? a.crow[row[it]] : -1;
        }
        if (a.R && !a.part) {
#pragma unroll
            for (int it = 0; it < ITER; ++it) load_some<CH>((const T *)a.R + row[it] * a.ldr + m, row[it] >= 0 ? left : 0, res[it]);
        }
        wave_sync();
        put(run, mine);
        wave_sync();
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            if (row[it] < 0) continue;
            const int r = r0 + it * ROWS;
            A v[CH];
#pragma unroll
            for (int e = 0; e < CH; e += ACH) __builtin_memcpy(v + e, mine + SR::at(r, (lane % LANES * CH + e) / ACH), 16);
            if (a.part) store_some<CH>((A *)a.part + (part_row + row[it]) * a.m + m, left, v);
            else finish<CH, T, A>(b, bias, res[it], row[it], m, v);
        }
    }
}

// The same of 8-bit operands' sums, RUN rows of TW along m at a time (put(run, part of
// m, its place)), a lane ending 8 values.  What the rows need from memory by their
// numbers is read for all of them before the first.
template <typename O, int TM, int RUNS, int RUN, int TW, typename Put>
__device__ __forceinline__ void finish_scaled(const TileArgs &a, char *lds, int piece, int group, int n0, int nend, int64_t m0, Put &&put)
{
    using SR = SumRows<int, TW>;
    constexpr int CH = 8, LANES = TW / CH, ROWS = 64 / LANES, ITER = RUN / ROWS;
    static_assert(RUN % ROWS == 0 && TM % TW == 0, "whole rows");
    const int lane = threadIdx.x & 63, r0 = lane / LANES;
    char *mine = lds + (threadIdx.x >> 6) * SR::BYTES * (RUN / 16);
    TileArgs b = a;
    if (!a.offsets) b.groups = 1;
    int row[RUNS][ITER];
    float qs[RUNS][ITER], by[TM / TW][CH], bias[TM / TW][CH];
#pragma unroll
    for (int run = 0; run < RUNS; ++run)
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            const int n = n0 + RUN * run + r0 + it * ROWS;
            row[run][it] = n < nend ? n : -1;
            qs[run][it] = n < nend && !a.part ? scale_of(b, group, n) : 0.0f;
            if (n < nend && !a.part && a.crow) row[run][it] = a.crow[n];
        }
#pragma unroll
    for (int h = 0; h < TM / TW; ++h) {
        O v[CH];
        load_bias<CH>(b, group, m0 + TW * h + lane % LANES * CH, v);
#pragma unroll
        for (int e = 0; e < CH; ++e) bias[h][e] = (float)v[e];
        load_scales<CH>(b, group, m0 + TW * h + lane % LANES * CH, by[h]);
    }
#pragma unroll
    for (int run = 0; run < RUNS; ++run)
#pragma unroll
        for (int h = 0; h < TM / TW; ++h) {
            const int64_t m = m0 + TW * h + lane % LANES * CH, left = a.m - m;
            O res[ITER][CH];
            if (a.R && !a.part) {
#pragma unroll
                for (int it = 0; it < ITER; ++it)
                    load_some<CH>((const O *)a.R + row[run][it] * a.ldr + m, row[run][it] >= 0 ? left : 0, res[it]);
            }
            wave_sync();
            put(run, h, mine);
            wave_sync();
#pragma unroll
            for (int it = 0; it < ITER; ++it) {
                if (row[run][it] < 0 || left <= 0) continue;
                const int r = r0 + it * ROWS;
                int v[CH];
#pragma unroll
                for (int e = 0; e < CH; e += 4) __builtin_memcpy(v + e, mine + SR::at(r, (lane % LANES * CH + e) / 4), 16);
                if (a.part) {
                    store_some<CH>((int *)a.part + ((int64_t)piece * a.n + row[run][it]) * a.m + m, left, v);
                    continue;
                }
                float f[CH];
                scale_sums<CH>(v, qs[run][it], by[h], bias[h], f);
                finish_sum<CH, true, O, float>(b, res[it], row[run][it], m, f);
            }
        }
}

// A 16-row run of 16 x 16 tiles: lane (li, g) holds rows 4g .. 4g+3 of column li.
template <typename A, int MT, int NTL, int TM, typename A4>
__device__ __forceinline__ void put_rows(const A4 (&acc)[MT][NTL], int j, char *to)
{
    constexpr int ACH = 16 / sizeof(A);
    const int li = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int w = 0; w < 4; w += ACH) {
            A v[ACH];
#pragma unroll
            for (int e = 0; e < ACH; ++e) v[e] = acc[i][j][w + e];
            __builtin_memcpy(to + SumRows<A, TM>::at(li, (16 * i + 4 * g + w) / ACH), v, 16);
        }
}

// A workgroup of WM x WN waves makes BM x BN sums; a wave (BM/WM) x (BN/WN) in
// registers.  One LDS tile of 128 bytes of k per row: while the waves multiply
// it, their loads of the next one are in flight to registers, and two
// workgroups a CU fill each other's waits.
template <typename T, bool PKC, bool QKC, int BM, int BN, int WM, int WN, typename O = T>
__global__ __launch_bounds__(WM *WN * 64, 2) void tile_product_kernel(const TileArgs a)
{
    using A4 = typename Elem<T>::Acc4;
    constexpr int NT = WM * WN * 64, BK = 128 / sizeof(T), CH = 16 / sizeof(T);
    constexpr int TM = BM / WM, TN = BN / WN, MT = TM / 16, NTL = TN / 16;
    constexpr int LM = BM > 64 && BM < 128 ? 128 : BM;  // rows of P in LDS
    constexpr bool KSUM = !PKC && !QKC;                 // groups cut k, not n
    constexpr int TILE = (LM + BN) * 128, SUMS = WM * WN * SumRows<typename Elem<T>::Acc, TM>::BYTES;
    __shared__ __align__(16) char lds[TILE > SUMS ? TILE : SUMS];
    char *lp = lds, *lq = lds + LM * 128;

    Work w;
    if (!find_work<KSUM, BN, BK>(a, &w)) return;
    const int group = w.group, n0 = w.n0, nend = w.nend, k0 = w.k0, kend = w.kend;
    const int64_t m0 = (int64_t)w.tm * BM;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int wm0 = wave % WM * TM, wn0 = wave / WM * TN;
    // The f64 step leaves rows g, g+4, g+8, g+12 in lane (j, g); fed with A's
    // row 4 (i % 4) + i / 4 in place i it leaves 4g .. 4g+3 like the others.
    const int lr = sizeof(T) == 8 ? 4 * (li & 3) + (li >> 2) : li;

    A4 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = A4{0, 0, 0, 0};

    if (k0 < kend) {
        using SP = Stage<T, PKC, LM, NT>;
        using SQ = Stage<T, QKC, BN, NT>;
        SP sp;
        SQ sq;
        const int64_t sg = KSUM ? 0 : group;
        sp.init((const T *)a.P + sg * a.gp, a.ldp, nullptr, m0, a.m, a.k);
        sq.init((const T *)a.Q, a.ldq, a.qrow, n0, nend, a.k);
        sp.load(k0, kend);
        sq.load(k0, kend);
        for (int64_t k = k0; k < kend; k += BK) {
            __syncthreads();
            sp.store(lp);
            sq.store(lq);
            __syncthreads();
            if (k + BK < kend) {
                sp.load(k + BK, kend);
                sq.load(k + BK, kend);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (s && k + BK / 2 >= kend) break;
                if constexpr (sizeof(T) <= 2) {
                    uint32x4 p[MT], q[NTL];
#pragma unroll
                    for (int j = 0; j < NTL; ++j) q[j] = SQ::frag16(lq, wn0 / 16 + j, s);
#pragma unroll
                    for (int i = 0; i < MT; ++i) p[i] = SP::frag16(lp, wm0 / 16 + i, s);
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int j = 0; j < NTL; ++j) acc[i][j] = mma(p[i], q[j], acc[i][j], T());
                } else {
                    T p[MT][CH], q[NTL][CH];
                    SQ::template frag<NTL>(lq, wn0, li, g, s, q);
                    SP::template frag<MT>(lp, wm0, lr, g, s, p);
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int j = 0; j < NTL; ++j) acc[i][j] = mma(p[i][c], q[j][c], acc[i][j]);
                }
            }
        }
    }

    __syncthreads();
    auto put = [&](int j, char *to) { put_rows<typename Elem<T>::Acc, MT, NTL, TM>(acc, j, to); };
    if constexpr (std::is_same_v<T, O>) finish_tile<T, KSUM, TM, NTL>(a, lds, w.piece, group, n0 + wn0, nend, m0 + wm0, put);
    else
        finish_scaled<O, TM, NTL, 16, TM>(a, lds, w.piece, group, n0 + wn0, nend, m0 + wm0, [&](int j, int, char *to) { put(j, to); });
}

// ----------------------------------------------- tiles by copies to LDS

__device__ uint32_t tile_zeros[4];             // what a copy reads for k past the end

// One operand's tile of R rows by BK of k, copied from global memory to LDS
// without a register between: a wave's copy writes 64 chunks of 16 bytes in lane
// order, so the order that the LDS reads want is given by what each lane reads.
// kc rows have their chunks permuted as in Stage (64-byte rows: by r / 4, four of
// them making one pass over the banks), sc rows their segments.
template <typename T, bool KC, int R, int NT, int BK>
struct Copy {
    static constexpr int SZ = sizeof(T), CH = 16 / SZ, RB = BK * SZ;   // a chunk's elements, a kc row's bytes
    static constexpr int PER = KC ? BK / CH : R / CH, CNT = R * BK / CH / NT, BYTES = R * RB, STEP = NT / PER;
    static_assert(R * BK / CH % NT == 0 && NT % PER == 0, "whole copies");
    static_assert(R / 16 >= (SZ == 2 ? 8 : 4), "segments to permute");
    // kc rows may lie anywhere (qrow), so each slot has its address; sc slots lie
    // at 32-bit distances from the step's first row.
    const T *base;
    const T *p[KC ? CNT : 1];
    uint32_t off[KC ? 1 : CNT];
    int64_t ld;

    __device__ __forceinline__ static int lds_row(int i) { return threadIdx.x / PER + i * STEP; }
    __device__ __forceinline__ static int flip(int r)
    {
        return RB == 128 ? (r >> 1 & 7) ^ (r & 1) << 2 : (r >> 2 & 3) ^ (r & 2);
    }
    // Where 16 elements of an sc row lie: a transposed 16-bit read takes 4 rows at
    // two of them at once, a 32-bit read 4 rows 16 bytes of k apart.
    __device__ __forceinline__ static int segment(int seg, int k)
    {
        return SZ == 2 ? seg ^ (k & 3) << 1 : seg ^ (k / CH & 3);
    }
    // The first of the elements along its row that slot i reads.
    __device__ __forceinline__ static int first(int i)
    {
        const int c = threadIdx.x % PER, r = lds_row(i);
        if constexpr (KC) return (c ^ flip(r)) * CH;
        else return segment(c / (16 / CH), r) * 16 + c % (16 / CH) * CH;
    }

    __device__ __forceinline__ void init(const T *b, int64_t ld_, const int32_t *idx, int r0, int rend, int k0)
    {
        ld = ld_;
        base = b;
        if constexpr (KC) {
#pragma unroll
            for (int i = 0; i < CNT; ++i) {
                int r = r0 + lds_row(i);
                r = r < rend ? r : rend - 1;
                if (idx) r = idx[r];
                p[i] = b + (int64_t)r * ld + first(i) + k0;
            }
        } else {
            base += k0 * ld;
#pragma unroll
            for (int i = 0; i < CNT; ++i) {
                int c = r0 + first(i);
                c = c < rend ? c : r0;             // columns past the edge are computed and not stored
                off[i] = c + lds_row(i) * (uint32_t)ld;
            }
        }
    }

    // Starts the copies of [k0, k0 + BK) and steps on.
    template <bool TAIL>
    __device__ __forceinline__ void start(char *lds, int k0, int kend)
    {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const T *q;
            if constexpr (KC) q = p[i];
            else q = base + off[i];
            if constexpr (TAIL) {
                const int k = k0 + (KC ? first(i) : lds_row(i));
                if (k >= kend) q = (const T *)tile_zeros;
            }
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)q,
                                             (__attribute__((address_space(3))) void *)(lds + (i * NT + wave * 64) * 16), 16, 0, 0);
            if constexpr (KC) p[i] += BK;
        }
        if constexpr (!KC) base += BK * ld;
    }

    // Where a lane reads what it feeds to a 32x32x16 step: row 32 tile + lane % 32,
    // k = 8 (lane / 32) .. + 7; the other tiles and steps lie at flips of its bits
    // and at fixed distances.
    __device__ __forceinline__ static int place(int tile)
    {
        const int lane = threadIdx.x & 63, li = lane & 15;
        if constexpr (SZ > 2) {
            // A 16x16x4 step: row 16 tile + li, k = CH g + j.
            const int g = lane >> 4;
            if constexpr (KC) return (16 * tile + li) * RB + ((g ^ flip(li)) << 4);
            return CH * g * R * SZ + (segment(tile, CH * g) * 16 + li) * SZ;
        }
        if constexpr (KC) return (32 * tile + (lane & 31)) * RB + (((lane >> 5) ^ flip(lane & 31)) << 4);
        const int k = 8 * (lane >> 5) + (li >> 2);
        return k * R * 2 + (segment(2 * tile + (lane >> 4 & 1), k) << 5) + ((li & 3) << 3);
    }

    // That of step s of tile `tile` + i (`tile` a multiple of the tiles, a power of
    // two, that it is read for).
    __device__ __forceinline__ static uint32x4 frag(const char *lds, int at, int i, int s)
    {
        if constexpr (KC) {
            return *reinterpret_cast<const uint32x4 *>(lds + (at ^ s << 5) + i * 32 * RB);
        } else {
            uint32x4 out;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const shortx4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) shortx4 *)(lds + (at ^ i << 6) + (16 * s + 4 * h) * R * 2));
                const uint32x2 u = __builtin_bit_cast(uint32x2, t);
                out[2 * h] = u[0];
                out[2 * h + 1] = u[1];
            }
            return out;
        }
    }

    // The same of a 16x16x4 step's: f[j] is its value at k = CH (g + 4 s) + j.
    __device__ __forceinline__ static void frag_wide(const char *lds, int at, int i, int s, T (&f)[CH])
    {
        if constexpr (KC) {
            __builtin_memcpy(f, lds + (at ^ s << 6) + i * 16 * RB, 16);
        } else {
#pragma unroll
            for (int j = 0; j < CH; ++j)
                f[j] = *reinterpret_cast<const T *>(lds + (at ^ i * 16 * SZ) + (4 * CH * s + j) * R * SZ);
        }
    }
};

// Waits until at most N of this wave's copies are under way and its LDS reads are
// done, then for the other waves.  A fence here would wait for all the copies.
template <int N>
__device__ __forceinline__ void copies_done()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 & 3) << 14 | 7 << 4);     // vmcnt(N) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// As tile_product_kernel for operands whose chunks lie whole and aligned, NB
// LDS tiles in turn: while one is multiplied, the copies of the next NB - 1 are
// under way, and a step has one barrier.
template <typename T, bool PKC, bool QKC, int BM, int BN, int WM, int WN, int BK, int NB, typename O = T>
__global__ __launch_bounds__(WM *WN * 64, sizeof(T) == 2 && BM == 128 && BK == 32 ? 3 : 2) void tile_copy_kernel(const TileArgs a)
{
    constexpr bool HALF = sizeof(T) <= 2;
    constexpr int STEP = HALF ? 32 : 16;                // rows and columns of a matrix step
    constexpr int NT = WM * WN * 64, TM = BM / WM, TN = BN / WN, MT = TM / STEP, NTL = TN / STEP;
    constexpr int LM = BM > 64 && BM < 128 ? 128 : BM;  // rows of P in LDS
    constexpr bool KSUM = !PKC && !QKC;
    using A = typename Elem<T>::Acc;
    using Sum = std::conditional_t<sizeof(T) == 1, intx16, std::conditional_t<HALF, floatx16, floatx4>>;
    using CP = Copy<T, PKC, LM, NT, BK>;
    using CQ = Copy<T, QKC, BN, NT, BK>;
    // Arrays of their own: the compiler then knows which copies an LDS read waits for.
    constexpr int TILE = CP::BYTES + CQ::BYTES, SUMS = WM * WN * (sizeof(T) == 1 && TM <= 64 ? 2 : 1) * SumRows<A, TM>::BYTES;
    __shared__ __align__(16) char lds0[TILE > SUMS ? TILE : SUMS];
    __shared__ __align__(16) char lds1[TILE];
    __shared__ __align__(16) char lds2[NB > 2 ? TILE : 16];
    Work w;
    if (!find_work<KSUM, BN, BK>(a, &w)) return;
    const int group = w.group, n0 = w.n0, nend = w.nend, k0 = w.k0, kend = w.kend;
    const int m0 = w.tm * BM;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm0 = wave % WM * TM, wn0 = wave / WM * TN;

    Sum acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = Sum{0};

    if (k0 < kend) {
        CP cp;
        CQ cq;
        cp.init((const T *)a.P + (KSUM ? 0 : group * a.gp), a.ldp, nullptr, m0, a.m, k0);
        cq.init((const T *)a.Q, a.ldq, a.qrow, n0, nend, k0);
        constexpr int EACH = CP::CNT + CQ::CNT;
        auto start = [&](char *to, int k) {
            if (k + BK <= kend) {
                cp.template start<false>(to, k, kend);
                cq.template start<false>(to + CP::BYTES, k, kend);
            } else {
                cp.template start<true>(to, k, kend);
                cq.template start<true>(to + CP::BYTES, k, kend);
            }
        };
        const int at_p = CP::place(wm0 / STEP), at_q = CQ::place(wn0 / STEP);
        auto multiply = [&](const char *from, int left) {
            int pa = at_p, qa = at_q;
            asm("" : "+v"(pa), "+v"(qa));          // its flips are made here, not held in registers over the loop
            if constexpr (HALF) {
#pragma unroll
                for (int s = 0; s < BK * (int)sizeof(T) / 32; ++s) {
                    uint32x4 p[MT], q[NTL];
#pragma unroll
                    for (int j = 0; j < NTL; ++j) q[j] = CQ::frag(from + CP::BYTES, qa, j, s);
#pragma unroll
                    for (int i = 0; i < MT; ++i) p[i] = CP::frag(from, pa, i, s);
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int j = 0; j < NTL; ++j) acc[i][j] = mma(p[i], q[j], acc[i][j], T());
                }
            } else {
                constexpr int CH = 16 / sizeof(T);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (s == 0 || left > BK / 2) {
                    T p[MT][CH], q[NTL][CH];
#pragma unroll
                    for (int j = 0; j < NTL; ++j) CQ::frag_wide(from + CP::BYTES, qa, j, s, q[j]);
#pragma unroll
                    for (int i = 0; i < MT; ++i) CP::frag_wide(from, pa, i, s, p[i]);
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int j = 0; j < NTL; ++j) acc[i][j] = mma(p[i][c], q[j][c], acc[i][j]);
                    }
                }
            }
        };
        // One step: its tile is there once all but the later tiles' copies are.
        auto step = [&](const char *from, char *to, int k) {
            if (NB > 2 && k + BK < kend) copies_done<(NB - 2) * EACH>();
            else copies_done<0>();
            if (k + (NB - 1) * BK < kend) start(to, k + (NB - 1) * BK);
            multiply(from, kend - k);
        };
        // The same where that tile's copies, and the next's, are whole.
        auto copy = [&](char *to, int k) {
            cp.template start<false>(to, k, kend);
            cq.template start<false>(to + CP::BYTES, k, kend);
            __builtin_amdgcn_sched_barrier(0);      // not after the products, where they would be late
        };
        auto steady = [&](const char *from, char *to, int k) {
            copies_done<(NB - 2) * EACH>();
            copy(to, k + (NB - 1) * BK);
            multiply(from, BK);
        };
        char *const last = NB == 2 ? lds1 : lds2;
        int k = k0;
        if (k + (2 * NB - 1) * BK <= kend) {
            copy(lds0, k);
            if constexpr (NB > 2) copy(lds1, k + BK);
            do {
                steady(lds0, last, k);
                steady(lds1, lds0, k + BK);
                if constexpr (NB > 2) steady(lds2, lds1, k + 2 * BK);
                k += NB * BK;
            } while (k + (2 * NB - 1) * BK <= kend);
        } else {
            start(lds0, k);
            if (NB > 2 && k + BK < kend) start(lds1, k + BK);
        }
        // The rounds at the end, and then the steps left over from whole rounds:
        // with exits in a loop's middle the sums would be copied between registers.
        for (; k + (NB - 1) * BK < kend; k += NB * BK) {
            step(lds0, last, k);
            step(lds1, lds0, k + BK);
            if constexpr (NB > 2) step(lds2, lds1, k + 2 * BK);
        }
        if (k < kend) {
            step(lds0, last, k);
            if (NB > 2 && k + BK < kend) step(lds1, lds0, k + BK);
        }
    }
    __syncthreads();
    if constexpr (!std::is_same_v<T, O>) {
        // As below, 32 columns by up to 64 of m a run.
        constexpr int TW = TM < 64 ? TM : 64;
        auto put = [&](int run, int h, char *to) {
            const int lane = threadIdx.x & 63;
#pragma unroll
            for (int i = 0; i < TW / 32; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    A v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[h * (TW / 32) + i][run][4 * q + e];
                    __builtin_memcpy(to + SumRows<A, TW>::at(lane & 31, 8 * i + 2 * q + (lane >> 5)), v, 16);
                }
        };
        finish_scaled<O, TM, NTL, 32, TW>(a, lds0, w.piece, group, n0 + wn0, nend, m0 + wm0, put);
        return;
    }
    auto put = [&](int run, char *to) {
        const int lane = threadIdx.x & 63;
        if constexpr (HALF) {
            // Lane l holds m = 8 q + 4 (l / 32) .. + 3 of column l % 32 in its values 4 q .. + 3.
            if ((lane >> 4 & 1) != (run & 1)) return;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    A v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[i][run / 2][4 * q + e];
                    __builtin_memcpy(to + SumRows<A, TM>::at(lane & 15, 8 * i + 2 * q + (lane >> 5)), v, 16);
                }
        } else {
            put_rows<A, MT, NTL, TM>(acc, run, to);
        }
    };
    if constexpr (std::is_same_v<T, O>) finish_tile<T, KSUM, TM, TN / 16>(a, lds0, w.piece, group, n0 + wn0, nend, m0 + wm0, put);
}

// ------------------------------------------------------------ few columns

// 16-bit products of at most 16 columns a run, where reading P is all the work: a
// workgroup makes 16 TILES of m by a run's columns over the whole k, its waves taking
// 32 STEPS of k each in turn straight to registers, the next ones read ahead, and adds
// their sums in LDS in order.  One launch, no sums in memory (k cut over workgroups and
// added by a second launch: 12.9 us for 4096 x 4096 and one column).  kc: 16 m, 64 bytes
// a row and step, 8.9 us at 3.8 TB/s with P in no cache.  sc: 32 m where that makes
// enough workgroups, for 64 bytes of a row (2048 -> 8192: 11.3 us, 16.3 with 16 m),
// else 16 (4096 -> 4096: 16.2 us, 17.6 with 32; 12.2 by 128 x 16 tiles and 16 pieces
// of k, which the estimate takes there); its pieces are transposed through LDS
// that the wave keeps to itself.
template <int TILES> struct Few {
    static constexpr int WAVES = TILES == 1 ? 8 : 16, STEPS = TILES == 1 ? 4 : 2;
};

template <typename T, bool PKC, int TILES, typename O = T>
__global__ __launch_bounds__(Few<TILES>::WAVES * 64) void few_columns_kernel(const TileArgs a)
{
    using F = Few<TILES>;
    using A = typename Elem<T>::Acc;
    using A4 = typename Elem<T>::Acc4;
    constexpr bool SCALED = !std::is_same_v<T, O>;
    constexpr int CH = 16 / sizeof(T), K = 4 * CH, WAVES = F::WAVES, STEPS = F::STEPS, M = 16 * TILES, SPAN = K * STEPS;
    constexpr int LANES = M / CH, ROWS = 64 / LANES;       // sc: lanes of a row of k, rows of one read
    static_assert(PKC || ROWS * TILES == 32, "TILES reads make a step");
    __shared__ __align__(16) A s_sum[WAVES][16][M];
    __shared__ __align__(16) char s_turn[PKC ? 16 : WAVES * STEPS * 32 * M * 2];
    Work w;
    if (!find_work<false, 16, 64>(a, &w)) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int64_t m0 = (int64_t)w.tm * M;
    const T *P = (const T *)a.P + w.group * a.gp;

    // kc: 16 bytes of row m0 + li from k = CH g; sc: 16 bytes of m of every ROWS'th row.
    const T *p;
    int64_t avail = CH;
    if constexpr (PKC) {
        p = P + (m0 + li < a.m ? m0 + li : a.m - 1) * a.ldp + CH * g;
    } else {
        const int64_t m = m0 + CH * (lane % LANES);
        avail = a.m - m;
        p = P + (int64_t)(lane / LANES) * a.ldp + m;
    }
    const int64_t over = a.m >= CH ? a.k - 1 : 0;          // as in Stage
    int col = w.n0 + li < w.nend ? w.n0 + li : w.nend - 1;
    if (a.qrow) col = a.qrow[col];
    const T *q = (const T *)a.Q + (int64_t)col * a.ldq + CH * g;

    const uint32x4 zero = {0, 0, 0, 0};
    auto read = [&](int k, uint32x4 (&pv)[STEPS][TILES], uint32x4 (&qv)[STEPS]) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int at = k + K * s, left = w.kend - at - CH * g;
            qv[s] = left >= CH ? load_chunk(q + at) : left > 0 ? load_chunk_part(q + at, left) : zero;
#pragma unroll
            for (int u = 0; u < TILES; ++u) {
                if constexpr (PKC) {
                    pv[s][u] = left >= CH ? load_chunk(p + at) : left > 0 ? load_chunk_part(p + at, left) : zero;
                } else {
                    const int row = at + lane / LANES + u * ROWS;
                    const T *r = p + (int64_t)(at + u * ROWS) * a.ldp;
                    pv[s][u] = row >= w.kend || avail <= 0 ? zero : avail >= CH || row < over ? load_chunk(r) : load_chunk_part(r, avail);
                }
            }
        }
    };
    A4 acc[TILES];
#pragma unroll
    for (int u = 0; u < TILES; ++u) acc[u] = A4{0, 0, 0, 0};
    auto multiply = [&](uint32x4 (&pv)[STEPS][TILES], uint32x4 (&qv)[STEPS]) {
        if constexpr (!PKC) {
            char *turn = s_turn + wave * STEPS * 32 * M * 2;
            wave_sync();
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int u = 0; u < TILES; ++u)
                    *reinterpret_cast<uint32x4 *>(turn + (s * 32 + u * ROWS) * M * 2 + lane * 16) = pv[s][u];
            wave_sync();
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int u = 0; u < TILES; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int k = 32 * s + 8 * g + 4 * h + (li >> 2);
                        const shortx4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) shortx4 *)(turn + k * M * 2 + u * 32 + (li & 3) * 8));
                        const uint32x2 v = __builtin_bit_cast(uint32x2, t);
                        pv[s][u][2 * h] = v[0];
                        pv[s][u][2 * h + 1] = v[1];
                    }
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int u = 0; u < TILES; ++u) acc[u] = mma(pv[s][u], qv[s], acc[u], T());
    };
    uint32x4 pa[STEPS][TILES], qa[STEPS], pb[STEPS][TILES], qb[STEPS];
    int k = w.k0 + wave * SPAN;
    constexpr int ROUND = WAVES * SPAN;
    if (k < w.kend) read(k, pa, qa);
    while (k < w.kend) {
        if (k + ROUND < w.kend) read(k + ROUND, pb, qb);
        multiply(pa, qa);
        k += ROUND;
        if (k >= w.kend) break;
        if (k + ROUND < w.kend) read(k + ROUND, pa, qa);
        multiply(pb, qb);
        k += ROUND;
    }
#pragma unroll
    for (int u = 0; u < TILES; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) s_sum[wave][li][16 * u + 4 * g + e] = acc[u][e];
    __syncthreads();
    const int i = threadIdx.x / M, j = threadIdx.x % M, n = w.n0 + i;
    const int64_t m = m0 + j;
    if (i >= 16 || n >= w.nend || m >= a.m) return;
    A v[1] = {0};
#pragma unroll
    for (int u = 0; u < WAVES; ++u) v[0] += s_sum[u][i][j];
    TileArgs b = a;
    if (!a.offsets) b.groups = 1;
    const int64_t row = a.crow ? (int64_t)a.crow[n] : n;
    O bias[1], res[1];
    load_bias<1>(b, w.group, m, bias);
    if (a.R) res[0] = ((const O *)a.R)[row * a.ldr + m];
    if constexpr (SCALED) {
        float by[1], f[1], added[1] = {(float)bias[0]};
        load_scales<1>(b, w.group, m, by);
        scale_sums<1>(v, scale_of(b, w.group, n), by, added, f);
        finish_sum<1, false, O, float>(b, res, row, m, f);
    } else {
        finish<1, T, float>(b, bias, res, row, m, v);
    }
}

// Adds the split partial sums and ends as the kernels above would.  256 threads are
// 256/LANES items of 4 values by LANES shares of the splits, each share added in
// order and then the shares in theirs.
template <typename T, bool KSUM, int LANES, typename O = T>
__global__ __launch_bounds__(256) void split_reduce_kernel(const TileArgs a)
{
    using A = typename Elem<T>::Acc;
    constexpr int V = 4, ITEMS = 256 / LANES;
    __shared__ A s_sum[LANES > 1 ? LANES : 1][ITEMS][V];
    const int64_t per = (a.m + V - 1) / V;
    const int64_t rows = KSUM && a.offsets ? a.n * a.groups : a.n;
    const int item = threadIdx.x % ITEMS, share = threadIdx.x / ITEMS;
    const int64_t at = (int64_t)blockIdx.x * ITEMS + item;
    const bool live = at < rows * per;
    const int64_t pr = live ? at / per : 0, m = live ? (at - pr * per) * V : 0;
    A s[V] = {0, 0, 0, 0};
    if (live) {
        const A *p = (const A *)a.part + (share * rows + pr) * a.m + m;
#pragma unroll 4
        for (int q = share; q < a.split; q += LANES, p += LANES * rows * a.m) {
            A t[V];
            load_some<V>(p, a.m - m, t);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += t[e];
        }
    }
    if constexpr (LANES > 1) {
#pragma unroll
        for (int e = 0; e < V; ++e) s_sum[share][item][e] = s[e];
        __syncthreads();
        if (share) return;
#pragma unroll
        for (int q = 1; q < LANES; ++q)
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += s_sum[q][item][e];
    }
    if (!live) return;
    TileArgs b = a;
    int group = 0;
    int64_t n = pr;
    if (KSUM && a.offsets) {
        group = (int)(pr / a.n);
        n = pr - group * a.n;
        b.C = (T *)a.C + group * a.gc;
    } else if (a.offsets) {
        int lo = 0, hi = a.groups;                    // the last offset that is <= n
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (a.offsets[mid] <= n) lo = mid;
            else hi = mid - 1;
        }
        group = lo;
    } else {
        b.groups = 1;
    }
    O bias[V], res[V];
    load_bias<V>(b, group, m, bias);
    const int64_t row = a.crow ? (int64_t)a.crow[n] : n;
    if (a.R) load_some<V>((const O *)a.R + row * a.ldr + m, a.m - m, res);
    if constexpr (!std::is_same_v<T, O>) {
        float by[V], f[V], added[V];
        load_scales<V>(b, group, m, by);
#pragma unroll
        for (int e = 0; e < V; ++e) added[e] = (float)bias[e];
        scale_sums<V>(s, scale_of(b, group, n), by, added, f);
        finish_sum<V, false, O, float>(b, res, row, m, f);
    } else {
        finish<V, T, A>(b, bias, res, row, m, s);
    }
}

// ------------------------------------------------------------------- host

// The shapes.  REG_* go through registers at any alignment, COPY_* copy to LDS.
// 256 x 256 and 256 x 128 carry the large products, 128 x 128 and 64 x 64 what
// leaves CUs idle in larger tiles, 128 x 32 and 128 x 16 few columns.  Float32's
// matrix steps bound it, so its widths of 64 to 128 fit m instead (100 of 128 rows
// would be a fifth of the steps for nothing) at 64 columns, where a CU holds
// enough workgroups to hide the rows it reads and stores.
struct TileShape { int bm, bn, threads; };
enum Shape { REG_128, REG_32, REG_16, REG_M128, REG_M112, REG_M96, REG_M80, REG_M64, COPY_256, COPY_TALL, COPY_128, FEW_16, FEW_32 };
constexpr TileShape TILE_SHAPES[] = {{128, 128, 256}, {128, 32, 256}, {128, 16, 256}, {128, 64, 256}, {112, 64, 256},
                                     {96, 64, 256}, {80, 64, 256}, {64, 64, 256}, {256, 256, 512}, {256, 128, 256},
                                     {128, 128, 256}, {16, 16, Few<1>::WAVES * 64}, {32, 16, Few<2>::WAVES * 64}};

// What a shape costs: its rate with a CU full of it (Tflop/s a CU), the time of 64 of
// k where latency bounds it (us), workgroups a CU, the start and end of a round (us).  Measured on products of 64 to
// 8,192 columns and 512 to 8,192 rows and k; the estimate below picks within 10 %
// of the best of them but for three (up to 20 %).  Of groups' products it only ranks
// the shapes (32 groups, 16,384 columns 2816 -> 1024: 138 us estimated, 194 measured;
// the sums over columns 93 and 181).
struct ShapeCost { Shape shape; double rate, latency; int held; double end = 2; };

// Whether every chunk that a copy reads lies whole in the operands, 16 bytes aligned.
template <typename T>
bool copies_fit(const TileArgs &a, bool pkc, bool qkc)
{
    const int64_t z = sizeof(T);
    const uintptr_t bits = (uintptr_t)a.P | (uintptr_t)a.Q | (uintptr_t)(a.ldp * z) | (uintptr_t)(a.ldq * z) |
                           (uintptr_t)(a.gp * z);
    const int64_t k = (pkc && !a.p_pad) || (qkc && !a.q_pad) ? a.k : 0, m = pkc || a.p_pad ? 0 : a.m, n = qkc || a.q_pad ? 0 : a.n;
    return (bits & 15) == 0 && (k | m | n) * z % 16 == 0 && a.ldp < (1 << 22) && a.ldq < (1 << 22);
}

// The workgroups that find_work counts on.
inline int64_t work_groups(const TileArgs &a, bool ksum)
{
    const int64_t total = (int64_t)a.tiles_m * a.tiles_n * a.split * (ksum && a.offsets ? a.groups : 1);
    return ((total + NUM_XCD - 1) / NUM_XCD + (a.offsets && !ksum ? 1 : 0)) * NUM_XCD;
}

template <typename T>
int plan_tile_product(TileArgs *a, bool pkc, bool qkc, int *shape, size_t *part_bytes, double *estimate)
{
    const bool ksum = !pkc && !qkc, grouped = a->offsets && !ksum;
    const int64_t batch = ksum && a->offsets ? a->groups : 1;
    const int64_t runs = grouped ? (a->groups < a->n ? a->groups : a->n) : 0;
    // Columns that share a matrix, and k of one sum, on average: the groups' sizes are
    // known on the device alone.  Worst where the average is just below a shape's limit
    // (64 groups, 2048 -> 1024, columns spread evenly and all in one group, us).  16:
    // bfloat16 with W along inp 115 and 87 for 1,024 columns, by wider tiles 43 and 24
    // for 1,025; along out 50 and 28, 44 and 29; Float32 131 and 84, 133 and 67.  48:
    // 57 and 33 for 3,071 columns, 55 and 43 for 3,100; Float32 184 and 130, 196 and 151.
    const int64_t share = grouped ? (a->n + a->groups - 1) / a->groups : a->n;
    const int64_t k = ksum && a->offsets ? (a->k + a->groups - 1) / a->groups : a->k;
    const int64_t sums = a->n * a->m * batch;
    const bool fit = copies_fit<T>(*a, pkc, qkc);
    auto tiles = [&](int s) {
        const int64_t tm = (a->m + TILE_SHAPES[s].bm - 1) / TILE_SHAPES[s].bm;
        const int64_t tn = (a->n + TILE_SHAPES[s].bn - 1) / TILE_SHAPES[s].bn;
        return tm * (tn + runs / 2) * batch;           // half the groups' last runs short, on average
    };
    // Sets a shape and its pieces of k; whether a launch, of fewer than 2^32 threads, takes it.
    auto set = [&](int s, int64_t p) {
        const TileShape &t = TILE_SHAPES[s];
        *shape = s;
        a->split = (int)p;
        a->tiles_m = (int)((a->m + t.bm - 1) / t.bm);
        a->tiles_n = (int)((a->n + t.bn - 1) / t.bn + runs);
        return work_groups(*a, ksum) < ((int64_t)1 << 32) / t.threads;
    };

    ShapeCost some[6];
    int count = 0;
    if constexpr (sizeof(T) == 1) {
        // Along k on both sides.  A step's bytes are 16-bit values', its k is twice
        // theirs; measured on 1 to 8,192 columns of 64 to 8,192 (48 products: 5 % past the
        // best on average, at most 35 %, with k = 64 and 13,574 rows of n in 4 groups).
        // Rows off 16 bytes through registers: two thirds of the rate.
        if (share <= 16 && set(FEW_16, 1)) some[count++] = {FEW_16, 1.0, 0.035, 4, 2.2};
        some[count++] = {REG_32, fit ? 3.7 : 2.6, 0.22, 5};
        some[count++] = {REG_M64, fit ? 4.4 : 2.9, 0.21, 5};
        if (fit && share > 48) {
            some[count++] = {COPY_128, 7.6, 0.36, 2, 3.7};
            some[count++] = {COPY_TALL, 7.7, 0.5, 2, 6.6};
            some[count++] = {COPY_256, 8.8, 0.9, 1, 10};
        }
    } else if (sizeof(T) == 2 && !ksum && share <= 16) {
        if (!set(FEW_16, 1)) {
            some[count++] = {REG_16, 1.0, 0.5, 6};
        } else if (pkc) {
            some[count++] = {FEW_16, 0.25, 0.07, 4};
        } else {
            some[count++] = {FEW_16, 0.2, 0.17, 4};
            some[count++] = {FEW_32, 0.25, 0.21, 2};
            some[count++] = {REG_16, 1.0, 0.5, 6};
        }
    } else if (!ksum && share <= 48) {
        some[count++] = share <= 16 ? ShapeCost{REG_16, 1.0, 0.5, 6} : ShapeCost{REG_32, 1.5, 0.5, 5};
        if (sizeof(T) > 2) some[0].rate = sizeof(T) == 4 ? 0.4 : 0.2, some[0].latency = 1.0;
    } else if constexpr (sizeof(T) == 2) {
        // 256 x 256 where there is more than one round of it and columns fill it:
        // 8,192 columns 2048 -> 8192 with gelu 284 us, 322 by 256 x 128.
        if (fit && !ksum && (!a->offsets || share >= 1024) && tiles(COPY_256) >= 512 && k > 192) {
            some[count++] = {COPY_256, 4.5, 1.3, 1};
        } else {
            if (fit && k > 192) {
                some[count++] = {COPY_TALL, 4.5, 0.95, 2};
                some[count++] = {COPY_128, 4.2, 0.62, 2};
            } else {
                some[count++] = {REG_128, 3.1, 0.75, 2};
            }
            some[count++] = {REG_M64, 2.2, 0.57, 5};
        }
    } else if constexpr (sizeof(T) == 4) {
        const int64_t each = (a->m + (a->m + 127) / 128 - 1) / ((a->m + 127) / 128);
        if (ksum || (fit && k > 256 && each > 112)) {
            some[count++] = fit ? ShapeCost{COPY_128, 0.55, 1.2, 2} : ShapeCost{REG_128, 0.48, 5.5, 2};
            some[count++] = {REG_M64, 0.45, 1.9, 4};
        } else {
            const Shape fits = each <= 64 ? REG_M64 : each <= 80 ? REG_M80 : each <= 96 ? REG_M96 : each <= 112 ? REG_M112 : REG_M128;
            some[count++] = {fits, 0.48, 1.2, 3};
        }
    } else {
        some[count++] = {REG_128, 0.25, 1.6, 2};
    }

    // Rounds of workgroups, each its steps of 64 of k; k cut in pieces costs a second
    // launch and its sums written and read.
    double best = 0;
    int best_shape = -1;
    int64_t split = 1;
    for (int i = 0; i < count; ++i) {
        const ShapeCost &o = some[i];
        const int64_t n = tiles(o.shape);
        const double work = 2e-6 * 64 * TILE_SHAPES[o.shape].bm * TILE_SHAPES[o.shape].bn / o.rate;
        for (int64_t p = 1; p == 1 || (o.shape != FEW_16 && o.shape != FEW_32 && p <= k / 128 && p * sums * (int64_t)sizeof(typename Elem<T>::Acc) <= (int64_t)1 << 28); p *= 2) {
            if (!set(o.shape, p)) break;
            const int64_t groups = n * p, slots = 256 * o.held;
            const int64_t held = (groups + 255) / 256 < o.held ? (groups + 255) / 256 : o.held;
            double rounds = (double)groups / slots;
            rounds = rounds <= 1 ? 1 : rounds < 3 ? (double)((groups + slots - 1) / slots) : rounds;
            const double step = held * work > o.latency ? held * work : o.latency;
            const double us = rounds * ((double)((k + 64 * p - 1) / (64 * p)) * step + o.end) + (p > 1 ? sizeof(T) == 1 ? 4.5 + 3e-6 * p * sums : 8 + 1e-6 * p * sums : 0);
            if (best_shape < 0 || us < best) {
                best = us;
                best_shape = o.shape;
                split = p;
            }
        }
    }
    if (best_shape < 0)
        return fail(JLUST_STATUS_INVALID_ARGUMENT, "linear: %lld x %lld sums (%lld groups) are more tiles than one launch takes",
                    (long long)a->m, (long long)a->n, (long long)a->groups);
    set(best_shape, split);
    if (estimate) *estimate = best;
    *part_bytes = split > 1 ? (size_t)split * sums * sizeof(typename Elem<T>::Acc) : 0;
    return JLUST_STATUS_SUCCESS;
}

template <typename T, bool PKC, bool QKC, int BM, int BN, int WM, int WN>
int launch_shape(const TileArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL((tile_product_kernel<T, PKC, QKC, BM, BN, WM, WN>),
                       dim3((unsigned)work_groups(a, !PKC && !QKC)), dim3(WM * WN * 64), 0, s, a);
    return check_launch("tile_product_kernel");
}

template <typename T, bool PKC, bool QKC, int BM, int BN, int WM, int WN, int BK, int NB>
int launch_copies(const TileArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL((tile_copy_kernel<T, PKC, QKC, BM, BN, WM, WN, BK, NB>),
                       dim3((unsigned)work_groups(a, !PKC && !QKC)), dim3(WM * WN * 64), 0, s, a);
    return check_launch("tile_copy_kernel");
}

template <typename T, bool PKC>
int launch_columns(const TileArgs &a, int shape, hipStream_t s)
{
    if constexpr (sizeof(T) == 2) switch (shape) {
        case FEW_16:
        case FEW_32:
            if (PKC || shape == FEW_16)
                hipLaunchKernelGGL((few_columns_kernel<T, PKC, 1>), dim3((unsigned)work_groups(a, false)), dim3(Few<1>::WAVES * 64), 0, s, a);
            else
                hipLaunchKernelGGL((few_columns_kernel<T, false, 2>), dim3((unsigned)work_groups(a, false)), dim3(Few<2>::WAVES * 64), 0, s, a);
            return check_launch("few_columns_kernel");
        case COPY_256: return launch_copies<T, PKC, true, 256, 256, 2, 4, 64, 2>(a, s);
        case COPY_TALL: return launch_copies<T, PKC, true, 256, 128, 2, 2, 32, 3>(a, s);
        case COPY_128: return launch_copies<T, PKC, true, 128, 128, 2, 2, 64, 2>(a, s);
        case REG_M64: return launch_shape<T, PKC, true, 64, 64, 2, 2>(a, s);
        case REG_32: return launch_shape<T, PKC, true, 128, 32, 4, 1>(a, s);
        case REG_16: return launch_shape<T, PKC, true, 128, 16, 4, 1>(a, s);
        }
    else switch (shape) {
        case REG_32: return launch_shape<T, PKC, true, 128, 32, 2, 2>(a, s);
        case REG_16: return launch_shape<T, PKC, true, 128, 16, 2, 1>(a, s);
        }
    if constexpr (sizeof(T) == 4) switch (shape) {
        case REG_M112: return launch_shape<T, PKC, true, 112, 64, 1, 4>(a, s);
        case REG_M96: return launch_shape<T, PKC, true, 96, 64, 1, 4>(a, s);
        case REG_M80: return launch_shape<T, PKC, true, 80, 64, 1, 4>(a, s);
        case REG_M64: return launch_shape<T, PKC, true, 64, 64, 1, 4>(a, s);
        case COPY_128: return launch_copies<T, PKC, true, 128, 128, 2, 2, 32, 2>(a, s);
        }
    if constexpr (sizeof(T) == 4) return launch_shape<T, PKC, true, 128, 64, 1, 4>(a, s);     // REG_M128
    else return launch_shape<T, PKC, true, 128, 128, 2, 2>(a, s);
}

template <typename T>
int launch_sums(const TileArgs &a, int shape, hipStream_t s)
{
    if constexpr (sizeof(T) == 2) {
        if (shape == COPY_TALL) return launch_copies<T, false, false, 256, 128, 2, 2, 32, 3>(a, s);
        if (shape == COPY_128) return launch_copies<T, false, false, 128, 128, 2, 2, 32, 3>(a, s);
    }
    if constexpr (sizeof(T) == 4)
        if (shape == COPY_128) return launch_copies<T, false, false, 128, 128, 2, 2, 32, 2>(a, s);
    if constexpr (sizeof(T) <= 4)
        if (shape == REG_M64) return launch_shape<T, false, false, 64, 64, 2, 2>(a, s);
    return launch_shape<T, false, false, 128, 128, 2, 2>(a, s);
}

template <typename T>
int launch_tile_product(const TileArgs &args, bool pkc, bool qkc, int shape, hipStream_t s)
{
    TileArgs a = args;
    if (a.split == 1) a.part = nullptr;
    const bool ksum = !pkc && !qkc;
    int st;
    if (ksum) st = launch_sums<T>(a, shape, s);
    else st = pkc ? launch_columns<T, true>(a, shape, s) : launch_columns<T, false>(a, shape, s);
    if (st || a.split == 1) return st;
    const int64_t rows = a.n * (ksum && a.offsets ? a.groups : 1), items = rows * ((a.m + 3) / 4);
    const bool shares = a.split > 16;
    const dim3 grid((unsigned)((items + (shares ? 15 : 255)) / (shares ? 16 : 256)));
    if (ksum && shares) hipLaunchKernelGGL((split_reduce_kernel<T, true, 16>), grid, dim3(256), 0, s, a);
    else if (ksum) hipLaunchKernelGGL((split_reduce_kernel<T, true, 1>), grid, dim3(256), 0, s, a);
    else if (shares) hipLaunchKernelGGL((split_reduce_kernel<T, false, 16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((split_reduce_kernel<T, false, 1>), grid, dim3(256), 0, s, a);
    return check_launch("split_reduce_kernel");
}

}  // namespace jlust
