// tile_kernel.hpp -- the matrix-core kernel of tile_product.hpp.
#pragma once

#include "tile_product.hpp"

namespace jlust {

typedef uint32_t uint32x2 __attribute__((ext_vector_type(2)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// One operand's tile of R rows by 128 bytes of k: global memory to registers to
// LDS.  kc: LDS row r holds its 8 chunks of 16 bytes at chunk ^ (r & 7), so the
// 16 rows that a wave reads at one k lie in different banks.  sc: LDS row k
// holds R elements; 16-bit ones have their 32-byte segments permuted by k, see
// `segment`.
template <typename T, bool KC, int R, int NT, bool IDX>
struct Stage {
    static constexpr int CH = 16 / sizeof(T);
    static constexpr int BK = 128 / sizeof(T);
    static constexpr int CHUNKS = R * 8;                       // R * 128 bytes
    static constexpr int CNT = (CHUNKS + NT - 1) / NT;
    static constexpr int PER = KC ? 8 : R / CH;                // chunks of one LDS row
    static constexpr int STEP = NT / PER;                      // LDS rows between a thread's chunks
    static constexpr bool WHOLE = CHUNKS % NT == 0;
    static_assert(NT % PER == 0, "a thread keeps its place in a row");

    const T *base;
    const T *p[KC ? CNT : 1];
    int64_t ld;
    int32_t row[IDX && !KC ? CNT : 1];
    int64_t avail;                       // sc: elements from this thread's first one to the edge
    const int32_t *idx;
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

    __device__ __forceinline__ void init(const T *b, int64_t ld_, const int32_t *idx_, int64_t r0, int64_t rend,
                                         int64_t k0, int64_t kend)
    {
        base = b;
        ld = ld_;
        idx = idx_;
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
            p[0] = b + c;
            rows(k0, kend);
        }
    }

    __device__ __forceinline__ void rows(int64_t k0, int64_t kend)
    {
        if constexpr (IDX && !KC)
            if (idx) {
#pragma unroll
                for (int i = 0; i < CNT; ++i) {
                    const int64_t k = k0 + lds_row(i);
                    row[i] = k < kend ? idx[k] : 0;
                }
            }
    }

    // Reads the tile of [k0, k0 + BK); what lies past kend is zero.
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
                    int64_t r = k;
                    if constexpr (IDX) r = idx ? (int64_t)row[i] : k;
                    const T *q = p[0] + r * ld;
                    v[i] = avail >= CH ? load_chunk(q) : load_chunk_part(q, avail);
                }
            }
            rows(k0 + BK, kend);
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
    // 16*tile + li, k = 32*s + 8*g .. + 7.
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

    // 32- and 64-bit operands: the values of 16-row tiles [0, TILES) from row
    // r0 for the CH steps of half s of the k range: f[tile][j] is lane (lr, g)'s
    // for k = CH*(g + 4s) + j.  kc: tile i's row lr is r0 + 16 i + lr; sc: it is
    // r0 + 16 CH (i/CH) + CH lr + i%CH, CH tiles from one read.
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
            static_assert(TILES % CH == 0, "sc tiles come CH at a time");
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const char *q = lds + (CH * (g + 4 * s) + j) * R * (int)sizeof(T);
#pragma unroll
                for (int i = 0; i < TILES; i += CH) {
                    T e[CH];
                    const uint32x4 c = *reinterpret_cast<const uint32x4 *>(q + (r0 + 16 * i + CH * lr) * sizeof(T));
                    __builtin_memcpy(e, &c, 16);
#pragma unroll
                    for (int u = 0; u < CH; ++u) f[i + u][j] = e[u];
                }
            }
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
__device__ __forceinline__ floatx4 mma(float a, float b, floatx4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ doublex4 mma(double a, double b, doublex4 c)
{
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}

// V sums of row n (before the map), columns mm ..: the epilogue.
template <int V, typename T, typename A>
__device__ __forceinline__ void finish(const TileArgs &a, int group, int64_t row, int64_t mm, A *s)
{
    constexpr bool FAST = sizeof(T) == 2;
    const int64_t left = a.m - mm;
    if (left <= 0) return;
    T *C = (T *)a.C + row * a.ldc + mm;
    const T *bias = a.bias && group < a.groups ? (const T *)a.bias + group * a.gb + mm : nullptr;
    const T *R = a.R ? (const T *)a.R + row * a.ldr + mm : nullptr;
    T *Z = a.Z ? (T *)a.Z + row * a.ldz + mm : nullptr;
    T t[V];
    if (left >= V) {
        if (bias) {
            load_vec<V>(bias, t);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += A(t[e]);
        }
        if (a.c_wide) {
            store_vec<V>((A *)a.C + row * a.ldc + mm, s);
            return;
        }
        if (Z) {
#pragma unroll
            for (int e = 0; e < V; ++e) t[e] = T(s[e]);
            store_vec<V>(Z, t);
        }
        if (a.act != JLUST_FN_IDENTITY) {
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] = activate<FAST>(a.act, s[e]);
        }
        if (R) {
            load_vec<V>(R, t);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += A(t[e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] = T(s[e]);
        store_vec<V>(C, t);
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (e >= left) break;
        A z = s[e];
        if (bias) z += A(bias[e]);
        if (a.c_wide) {
            ((A *)a.C + row * a.ldc + mm)[e] = z;
            continue;
        }
        if (Z) Z[e] = T(z);
        z = activate<FAST>(a.act, z);
        if (R) z += A(R[e]);
        C[e] = T(z);
    }
}

// A workgroup of WM x WN waves makes BM x BN sums; a wave (BM/WM) x (BN/WN) in
// registers.  One LDS tile of 128 bytes of k per row: while the waves multiply
// it, their loads of the next one are in flight to registers, and two
// workgroups a CU fill each other's waits.
template <typename T, bool PKC, bool QKC, int BM, int BN, int WM, int WN, bool IDX>
__global__ __launch_bounds__(WM *WN * 64, 2) void tile_product_kernel(const TileArgs a)
{
    using A = typename Elem<T>::Acc;
    using A4 = typename Elem<T>::Acc4;
    constexpr int NT = WM * WN * 64, BK = 128 / sizeof(T), CH = 16 / sizeof(T);
    constexpr int TM = BM / WM, TN = BN / WN, MT = TM / 16, NTL = TN / 16;
    constexpr bool KSUM = !PKC && !QKC;                 // groups cut k, not n
    __shared__ __align__(16) char lds[(BM + BN) * 128];
    char *lp = lds, *lq = lds + BM * 128;

    // Tiles in bands of 8 along n, m after m inside a band, each XCD a run of
    // its own: the workgroups that run at once on one XCD share P and Q tiles
    // in its L2.
    const int64_t total = (int64_t)a.tiles_m * a.tiles_n;
    const int64_t per = (total + NUM_XCD - 1) / NUM_XCD;
    const int64_t t = (int64_t)(blockIdx.x % NUM_XCD) * per + blockIdx.x / NUM_XCD;
    if (t >= total) return;
    const int64_t band = t / (8 * (int64_t)a.tiles_m), in = t - band * 8 * a.tiles_m;
    const int64_t wide = a.tiles_n - band * 8 < 8 ? a.tiles_n - band * 8 : 8;
    const int64_t tm = in / wide, tn = band * 8 + in % wide;

    int group = 0;
    int64_t n0 = tn * BN, nend = a.n, k0 = 0, kend = a.k;
    if (a.offsets) {
        if constexpr (KSUM) {
            group = blockIdx.z;
            k0 = a.offsets[group];
            kend = a.offsets[group + 1];
        } else {
            GroupRun r;
            if (!find_run(a.offsets, a.groups, a.n, tn, BN, &r)) return;
            group = r.group;
            n0 = r.begin;
            nend = r.end;
            if (group == a.groups) kend = 0;
        }
    }
    if (a.split > 1) {
        const int64_t piece = ((kend - k0 + a.split - 1) / a.split + BK - 1) / BK * BK;
        const int64_t lo = k0 + piece * blockIdx.y;
        kend = lo + piece < kend ? lo + piece : kend;
        k0 = lo;
    }
    const int64_t m0 = tm * BM;
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
        using SP = Stage<T, PKC, BM, NT, IDX>;
        using SQ = Stage<T, QKC, BN, NT, IDX>;
        SP sp;
        SQ sq;
        const int64_t sg = KSUM ? 0 : group;
        sp.init((const T *)a.P + sg * a.gp, a.ldp, PKC ? nullptr : a.prow, m0, a.m, k0, kend);
        sq.init((const T *)a.Q, a.ldq, a.qrow, n0, nend, k0, kend);
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
                if constexpr (sizeof(T) == 2) {
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

    // Lane (li, g) holds rows lr = 4g .. 4g+3 of every 16 x 16 tile's column li.
    // Tiles of an sc P in 32 and 64 bits interleave: V neighbours in m are V
    // tiles' values, else the four of one tile.
    constexpr bool MIX = sizeof(T) > 2 && !PKC, MIXN = sizeof(T) > 2 && !QKC;
    constexpr int V = MIX ? CH : 4;
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
        const int64_t n = n0 + wn0 + (MIXN ? 16 * CH * (j / CH) + CH * li + j % CH : 16 * j + li);
        if (n >= nend) continue;
        const int64_t row = a.crow ? (int64_t)a.crow[n] : n;
#pragma unroll
        for (int i = 0; i < MT; i += MIX ? CH : 1)
#pragma unroll
            for (int w = 0; w < (MIX ? 4 : 1); ++w) {
                A s[V];
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] = MIX ? acc[i + (MIX ? e : 0)][j][w] : acc[i][j][e & 3];
                const int64_t m = m0 + wm0 + 16 * i + (MIX ? CH * (4 * g + w) : 4 * g);
                if (a.part) {
                    // [split][group's rows][m]: rows of C in their order of n.
                    const int64_t rows = KSUM && a.offsets ? a.n * a.groups : a.n;
                    const int64_t pr = blockIdx.y * rows + (KSUM ? group * a.n : 0) + n;
                    A *d = (A *)a.part + pr * a.m + m;
                    if (m + V <= a.m) store_vec<V>(d, s);
                    else
                        for (int e = 0; e < V; ++e)
                            if (m + e < a.m) d[e] = s[e];
                } else {
                    TileArgs b = a;
                    if constexpr (KSUM) b.C = (T *)a.C + group * a.gc;
                    if (!a.offsets) b.groups = 1;
                    finish<V, T, A>(b, group, row, m, s);
                }
            }
    }
}

// Adds the split partial sums in order and ends as the kernel above would.
template <typename T, bool KSUM>
__global__ __launch_bounds__(256) void split_reduce_kernel(const TileArgs a)
{
    using A = typename Elem<T>::Acc;
    constexpr int V = 4;
    const int64_t per = (a.m + V - 1) / V;
    const int64_t rows = KSUM && a.offsets ? a.n * a.groups : a.n;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= rows * per) return;
    const int64_t pr = at / per, m = (at - pr * per) * V;
    A s[V] = {0, 0, 0, 0};
    const A *p = (const A *)a.part + pr * a.m + m;
    for (int q = 0; q < a.split; ++q, p += rows * a.m) {
        A t[V] = {0, 0, 0, 0};
        if (m + V <= a.m) load_vec<V>(p, t);
        else
            for (int e = 0; e < V; ++e)
                if (m + e < a.m) t[e] = p[e];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += t[e];
    }
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
    finish<V, T, A>(b, group, a.crow ? (int64_t)a.crow[n] : n, m, s);
}

// ------------------------------------------------------------------- host

struct TileShape { int bm, bn; };

// The shapes by index.  16-bit values: 256 x 128 carries the large products
// (LDS reads per flop fall with the wave's tile); 128 x 128 where that leaves
// CUs idle; 128 x 32 and 128 x 16 for few columns, where the weights' bytes
// count.  32 and 64 bits have no 256 x 128: its sums would not fit the registers.
constexpr TileShape TILE_SHAPES[] = {{256, 128}, {128, 128}, {128, 32}, {128, 16}};

template <typename T>
void plan_tile_product(TileArgs *a, bool pkc, bool qkc, int *shape, size_t *part_bytes)
{
    constexpr int64_t BK = 128 / sizeof(T);
    const bool ksum = !pkc && !qkc;
    const int64_t batch = ksum && a->offsets ? a->groups : 1;
    auto tiles = [&](int s) {
        const int64_t tm = (a->m + TILE_SHAPES[s].bm - 1) / TILE_SHAPES[s].bm;
        int64_t tn = (a->n + TILE_SHAPES[s].bn - 1) / TILE_SHAPES[s].bn;
        if (a->offsets && !ksum) tn += a->groups < a->n ? a->groups : a->n;   // every group's last run may be short
        a->tiles_m = (int)tm;
        a->tiles_n = (int)tn;
        return tm * tn * batch;
    };
    // Columns that share a matrix, on average.
    const int64_t share = a->offsets && !ksum ? (a->n + a->groups - 1) / a->groups : a->n;
    int s = sizeof(T) == 2 ? 0 : 1;
    if (!ksum && share <= 16) s = 3;
    else if (!ksum && share <= 48) s = 2;
    else if (s == 0 && tiles(0) < 512) s = 1;
    const int64_t count = tiles(s);
    // k is cut where fewer tiles than two a CU would run, into pieces of 4 steps at least.
    const int64_t k = ksum && a->offsets ? (a->k + a->groups - 1) / a->groups : a->k;
    int64_t split = 1;
    if (count < 512) {
        split = (512 + count - 1) / count;
        if (split > k / (4 * BK)) split = k / (4 * BK);
        if (split > 64) split = 64;
        if (split < 1) split = 1;
    }
    a->split = (int)split;
    *shape = s;
    *part_bytes = split > 1 ? (size_t)split * a->n * a->m * batch * sizeof(typename Elem<T>::Acc) : 0;
}

template <typename T, bool PKC, bool QKC, int BM, int BN, int WM, int WN, bool IDX>
int launch_shape(const TileArgs &a, hipStream_t s)
{
    const int64_t per = ((int64_t)a.tiles_m * a.tiles_n + NUM_XCD - 1) / NUM_XCD;
    const unsigned z = !PKC && !QKC && a.offsets ? (unsigned)a.groups : 1u;
    hipLaunchKernelGGL((tile_product_kernel<T, PKC, QKC, BM, BN, WM, WN, IDX>),
                       dim3((unsigned)(per * NUM_XCD), (unsigned)a.split, z), dim3(WM * WN * 64), 0, s, a);
    return check_launch("tile_product_kernel");
}

template <typename T, bool PKC>
int launch_columns(const TileArgs &a, int shape, hipStream_t s)
{
    switch (shape) {
    case 0:
        if constexpr (sizeof(T) == 2) return launch_shape<T, PKC, true, 256, 128, 2, 2, false>(a, s);
    case 1: return launch_shape<T, PKC, true, 128, 128, 2, 2, false>(a, s);
    case 2:
        if constexpr (sizeof(T) == 2) return launch_shape<T, PKC, true, 128, 32, 4, 1, false>(a, s);
        else return launch_shape<T, PKC, true, 128, 32, 2, 2, false>(a, s);
    default:
        if constexpr (sizeof(T) == 2) return launch_shape<T, PKC, true, 128, 16, 4, 1, false>(a, s);
        else return launch_shape<T, PKC, true, 128, 16, 2, 1, false>(a, s);
    }
}

template <typename T, bool IDX>
int launch_sums(const TileArgs &a, int shape, hipStream_t s)
{
    if constexpr (sizeof(T) == 2)
        if (shape == 0) return launch_shape<T, false, false, 256, 128, 2, 2, IDX>(a, s);
    return launch_shape<T, false, false, 128, 128, 2, 2, IDX>(a, s);
}

template <typename T>
int launch_tile_product(const TileArgs &args, bool pkc, bool qkc, int shape, hipStream_t s)
{
    TileArgs a = args;
    if (a.split == 1) a.part = nullptr;
    const bool ksum = !pkc && !qkc;
    int st;
    if (ksum) st = a.prow || a.qrow ? launch_sums<T, true>(a, shape, s) : launch_sums<T, false>(a, shape, s);
    else st = pkc ? launch_columns<T, true>(a, shape, s) : launch_columns<T, false>(a, shape, s);
    if (st || a.split == 1) return st;
    const int64_t rows = a.n * (ksum && a.offsets ? a.groups : 1), items = rows * ((a.m + 3) / 4);
    const dim3 grid((unsigned)((items + 255) / 256));
    if (ksum) hipLaunchKernelGGL((split_reduce_kernel<T, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((split_reduce_kernel<T, false>), grid, dim3(256), 0, s, a);
    return check_launch("split_reduce_kernel");
}

}  // namespace jlust
