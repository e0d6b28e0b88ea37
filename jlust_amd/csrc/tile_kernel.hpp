// tile_kernel.hpp -- the matrix-core kernel of tile_product.hpp.
#pragma once

#include "tile_product.hpp"
#include "wave.hpp"

namespace jlust {

typedef uint32_t uint32x2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
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
__device__ __forceinline__ floatx16 mma(uint32x4 a, uint32x4 b, floatx16 c, __bf16)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mma(uint32x4 a, uint32x4 b, floatx16 c, _Float16)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
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

// V sums of row `row` of C, columns mm ..: the epilogue.
template <int V, typename T, typename A>
__device__ __forceinline__ void finish(const TileArgs &a, const T *bias, int64_t row, int64_t mm, A *s)
{
    const int64_t left = a.m - mm;
    if (left <= 0) return;
    T t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] += A(bias[e]);
    if (a.c_wide) {
        store_some<V>((A *)a.C + row * a.ldc + mm, left, s);
        return;
    }
    if (a.Z) {
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] = T(s[e]);
        store_some<V>((T *)a.Z + row * a.ldz + mm, left, t);
    }
    activate_all<sizeof(T) == 2, V>(a.act, s);
    if (a.R) {
        load_some<V>((const T *)a.R + row * a.ldr + mm, left, t);
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += A(t[e]);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = T(s[e]);
    store_some<V>((T *)a.C + row * a.ldc + mm, left, t);
}

// This workgroup's tile.  Tiles lie in bands of 8 along n, m after m inside a
// band, each XCD a run of its own: the workgroups that run at once on one XCD
// share P and Q tiles in its L2.
__device__ __forceinline__ bool tile_of(const TileArgs &a, int *tm, int *tn)
{
    const int64_t total = (int64_t)a.tiles_m * a.tiles_n, per = (total + NUM_XCD - 1) / NUM_XCD;
    const int64_t t = (int64_t)(blockIdx.x % NUM_XCD) * per + blockIdx.x / NUM_XCD;
    if (t >= total) return false;
    const int64_t band = t / (8 * (int64_t)a.tiles_m);
    const int in = (int)(t - band * 8 * a.tiles_m);
    const int wide = a.tiles_n - (int)band * 8 < 8 ? a.tiles_n - (int)band * 8 : 8;
    *tm = in / wide;
    *tn = (int)band * 8 + in % wide;
    return true;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The rows of n, the k range and the group of a tile (extents are below 2^31);
// false if it has none.
struct TileRange { int group, n0, nend, k0, kend; };

template <bool KSUM, int BN, int BK>
__device__ __forceinline__ bool tile_range(const TileArgs &a, int tn, TileRange *t)
{
    *t = TileRange{0, tn * BN, (int)a.n, 0, (int)a.k};
    if (a.offsets) {
        if constexpr (KSUM) {
            t->group = blockIdx.z;
            t->k0 = a.offsets[t->group];
            t->kend = a.offsets[t->group + 1];
        } else {
            GroupRun r;
            if (!find_run(a.offsets, a.groups, a.n, tn, BN, &r)) return false;
            t->group = r.group;
            t->n0 = (int)r.begin;
            t->nend = (int)r.end;
            if (t->group == a.groups) t->kend = 0;
        }
    }
    if (a.split > 1) {
        const int piece = ((t->kend - t->k0 + a.split - 1) / a.split + BK - 1) / BK * BK;
        const int lo = t->k0 + piece * (int)blockIdx.y;
        t->kend = lo + (int64_t)piece < t->kend ? lo + piece : t->kend;
        t->k0 = lo;
    }
    return true;
}

// The end of a wave's sums, TM along m by 16 * RUNS along n.  The matrix steps
// leave a lane 4 values of a row; 16 rows at a time go through the wave's part of
// the LDS tile (put(run, its place) writes them, chunk c of row r at chunk c ^
// (r & FLIP)), so that a lane ends 16 bytes of C and a row's lanes a whole line.
// row_of(run, r) is their place along n.
template <typename A, int TM> struct SumRows {
    static constexpr int CHUNKS = TM * (int)sizeof(A) / 16, FLIP = CHUNKS < 16 ? CHUNKS - 1 : 15;
    __device__ __forceinline__ static int at(int r, int c) { return r * CHUNKS * 16 + ((c ^ (r & FLIP)) << 4); }
};

template <typename T, bool KSUM, int TM, int RUNS, typename Put, typename RowOf>
__device__ __forceinline__ void finish_tile(const TileArgs &a, char *lds, int group, int n0, int nend, int64_t m0, Put &&put,
                                            RowOf &&row_of)
{
    using A = typename Elem<T>::Acc;
    using SR = SumRows<A, TM>;
    constexpr int CH = 16 / sizeof(T), ACH = 16 / sizeof(A), LANES = TM / CH, ROWS = 64 / LANES;
    const int lane = threadIdx.x & 63;
    char *mine = lds + (threadIdx.x >> 6) * (16 * TM * (int)sizeof(A));
    const int64_t m = m0 + lane % LANES * CH, left = a.m - m;
    TileArgs b = a;
    if constexpr (KSUM) b.C = (T *)a.C + group * a.gc;
    if (!a.offsets) b.groups = 1;
    T bias[CH];
    load_bias<CH>(b, group, m, bias);
    const int64_t part_rows = KSUM && a.offsets ? a.n * a.groups : a.n;
    const int64_t part_row = blockIdx.y * part_rows + (KSUM ? group * a.n : 0);
#pragma unroll
    for (int run = 0; run < RUNS; ++run) {
        wave_sync();
        put(run, mine);
        wave_sync();
#pragma unroll 1
        for (int r = lane / LANES; r < 16; r += ROWS) {
            const int64_t n = n0 + row_of(run, r);
            if (n >= nend || left <= 0) continue;
            A v[CH];
#pragma unroll
            for (int e = 0; e < CH; e += ACH) __builtin_memcpy(v + e, mine + SR::at(r, (lane % LANES * CH + e) / ACH), 16);
            if (a.part) {
                store_some<CH>((A *)a.part + (part_row + n) * a.m + m, left, v);
            } else {
                finish<CH, T, A>(b, bias, a.crow ? (int64_t)a.crow[n] : n, m, v);
            }
        }
    }
}

// A workgroup of WM x WN waves makes BM x BN sums; a wave (BM/WM) x (BN/WN) in
// registers.  One LDS tile of 128 bytes of k per row: while the waves multiply
// it, their loads of the next one are in flight to registers, and two
// workgroups a CU fill each other's waits.
template <typename T, bool PKC, bool QKC, int BM, int BN, int WM, int WN, bool IDX>
__global__ __launch_bounds__(WM *WN * 64, 2) void tile_product_kernel(const TileArgs a)
{
    using A4 = typename Elem<T>::Acc4;
    constexpr int NT = WM * WN * 64, BK = 128 / sizeof(T), CH = 16 / sizeof(T);
    constexpr int TM = BM / WM, TN = BN / WN, MT = TM / 16, NTL = TN / 16;
    constexpr bool KSUM = !PKC && !QKC;                 // groups cut k, not n
    constexpr int TILE = (BM + BN) * 128, SUMS = WM * WN * 16 * TM * (int)sizeof(typename Elem<T>::Acc);
    __shared__ __align__(16) char lds[TILE > SUMS ? TILE : SUMS];
    char *lp = lds, *lq = lds + BM * 128;

    int tm, tn;
    TileRange r;
    if (!tile_of(a, &tm, &tn) || !tile_range<KSUM, BN, BK>(a, tn, &r)) return;
    const int group = uniform(r.group), n0 = uniform(r.n0), nend = uniform(r.nend), k0 = uniform(r.k0), kend = uniform(r.kend);
    const int64_t m0 = (int64_t)tm * BM;
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

    __syncthreads();
    // Lane (li, g) holds rows 4g .. 4g+3 of every 16 x 16 tile's column li.  Tiles of
    // an sc P in 32 and 64 bits interleave (Stage::frag): neighbours in m are
    // neighbouring tiles' values, else the four of one tile; the same along n.
    constexpr bool MIX = sizeof(T) > 2 && !PKC, MIXN = sizeof(T) > 2 && !QKC;
    constexpr int ACH = 16 / sizeof(typename Elem<T>::Acc);
    auto put = [&](int j, char *to) {
#pragma unroll
        for (int i = 0; i < MT; i += MIX ? CH : 1)
#pragma unroll
            for (int w = 0; w < 4; w += MIX ? 1 : ACH) {
                typename Elem<T>::Acc v[ACH];
#pragma unroll
                for (int e = 0; e < ACH; ++e) v[e] = MIX ? acc[i + (MIX ? e : 0)][j][w] : acc[i][j][(w + (MIX ? 0 : e)) & 3];
                const int at = 16 * i + (MIX ? CH * (4 * g + w) : 4 * g + w);       // in m
                __builtin_memcpy(to + SumRows<typename Elem<T>::Acc, TM>::at(li, at / ACH), v, 16);
            }
    };
    finish_tile<T, KSUM, TM, NTL>(a, lds, group, n0 + wn0, nend, m0 + wm0, put, [](int j, int r) {
        return MIXN ? 16 * CH * (j / CH) + CH * r + j % CH : 16 * j + r;
    });
}

// ----------------------------------------------- 16-bit tiles by copies to LDS

__device__ uint32_t tile_zeros[4];             // what a copy reads for k past the end

// One operand's tile of R rows by BK of k, copied from global memory to LDS
// without a register between: a wave's copy writes 64 chunks of 16 bytes in lane
// order, so the order that the LDS reads want is given by what each lane reads.
// kc rows have their chunks permuted as in Stage (64-byte rows: by r / 4, four of
// them making one pass over the banks), sc rows their segments.
template <typename T, bool KC, int R, int NT, int BK, bool IDX>
struct Copy {
    static constexpr int PER = KC ? BK / 8 : R / 8, CNT = R * BK / 8 / NT, BYTES = R * BK * 2, STEP = NT / PER;
    static_assert(R * BK / 8 % NT == 0 && NT % PER == 0, "whole copies");
    // kc rows may lie anywhere (qrow), so each slot has its address; sc slots lie
    // at 32-bit distances from the step's first row, or IDX finds their rows.
    const T *base;
    const T *p[KC ? CNT : 1];
    uint32_t off[KC ? 1 : CNT];
    int64_t ld;
    const int32_t *idx;
    int32_t row[IDX && !KC ? CNT : 1];

    __device__ __forceinline__ static int lds_row(int i) { return threadIdx.x / PER + i * STEP; }
    __device__ __forceinline__ static int flip(int r)
    {
        return BK == 64 ? (r >> 1 & 7) ^ (r & 1) << 2 : (r >> 2 & 3) ^ (r & 2);
    }
    __device__ __forceinline__ static int segment(int seg, int k)
    {
        static_assert(R / 16 >= 8, "rows of 256 bytes at least");
        return seg ^ (k & 3) << 1;
    }
    // The first of the 8 elements along its row that slot i reads.
    __device__ __forceinline__ static int first(int i)
    {
        const int c = threadIdx.x % PER, r = lds_row(i);
        if constexpr (KC) return (c ^ flip(r)) * 8;
        else return segment(c >> 1, r) * 16 + (c & 1) * 8;
    }

    __device__ __forceinline__ void init(const T *b, int64_t ld_, const int32_t *idx_, int r0, int rend, int k0, int kend)
    {
        ld = ld_;
        idx = idx_;
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
            if constexpr (!IDX) base += k0 * ld;
#pragma unroll
            for (int i = 0; i < CNT; ++i) {
                int c = r0 + first(i);
                c = c < rend ? c : r0;             // columns past the edge are computed and not stored
                off[i] = c + (IDX ? 0 : lds_row(i) * (uint32_t)ld);
            }
            rows(k0, kend);
        }
    }

    __device__ __forceinline__ void rows(int k0, int kend)
    {
        if constexpr (IDX && !KC)
#pragma unroll
            for (int i = 0; i < CNT; ++i) {
                const int k = k0 + lds_row(i);
                row[i] = k < kend ? (idx ? idx[k] : k) : 0;
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
            else if constexpr (IDX) q = base + ((int64_t)row[i] * ld + off[i]);
            else q = base + off[i];
            if constexpr (TAIL) {
                const int k = k0 + (KC ? first(i) : lds_row(i));
                if (k >= kend) q = (const T *)tile_zeros;
            }
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)q,
                                             (__attribute__((address_space(3))) void *)(lds + (i * NT + wave * 64) * 16), 16, 0, 0);
            if constexpr (KC) p[i] += BK;
        }
        if constexpr (!KC && !IDX) base += BK * ld;
        rows(k0 + BK, kend);
    }

    // Where a lane reads what it feeds to a 32x32x16 step: row 32 tile + lane % 32,
    // k = 8 (lane / 32) .. + 7; the other tiles and steps lie at flips of its bits
    // and at fixed distances.
    __device__ __forceinline__ static int place(int tile)
    {
        const int lane = threadIdx.x & 63, li = lane & 15;
        if constexpr (KC) return (32 * tile + (lane & 31)) * BK * 2 + (((lane >> 5) ^ flip(lane & 31)) << 4);
        const int k = 8 * (lane >> 5) + (li >> 2);
        return k * R * 2 + (segment(2 * tile + (lane >> 4 & 1), k) << 5) + ((li & 3) << 3);
    }

    // That of step s of tile `tile` + i (`tile` a multiple of the tiles, a power of
    // two, that it is read for).
    __device__ __forceinline__ static uint32x4 frag(const char *lds, int at, int i, int s)
    {
        if constexpr (KC) {
            return *reinterpret_cast<const uint32x4 *>(lds + (at ^ s << 5) + i * 64 * BK);
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

// As tile_product_kernel for 16-bit values whose chunks lie whole and aligned, NB
// LDS tiles in turn: while one is multiplied, the copies of the next NB - 1 are
// under way, and a step has one barrier.
template <typename T, bool PKC, bool QKC, int BM, int BN, int WM, int WN, int BK, int NB, bool IDX>
__global__ __launch_bounds__(WM *WN * 64, BM == 128 && BK == 32 ? 3 : 2) void tile_copy_kernel(const TileArgs a)
{
    constexpr int NT = WM * WN * 64, TM = BM / WM, TN = BN / WN, MT = TM / 32, NTL = TN / 32;
    constexpr bool KSUM = !PKC && !QKC;
    using CP = Copy<T, PKC, BM, NT, BK, IDX>;
    using CQ = Copy<T, QKC, BN, NT, BK, IDX>;
    // Arrays of their own: the compiler then knows which copies an LDS read waits for.
    constexpr int TILE = CP::BYTES + CQ::BYTES, SUMS = WM * WN * 16 * TM * 4;
    __shared__ __align__(16) char lds0[TILE > SUMS ? TILE : SUMS];
    __shared__ __align__(16) char lds1[TILE];
    __shared__ __align__(16) char lds2[NB > 2 ? TILE : 16];
    int tm, tn;
    TileRange r;
    if (!tile_of(a, &tm, &tn) || !tile_range<KSUM, BN, BK>(a, tn, &r)) return;
    const int group = uniform(r.group), n0 = uniform(r.n0), nend = uniform(r.nend), k0 = uniform(r.k0), kend = uniform(r.kend);
    const int m0 = tm * BM;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm0 = wave % WM * TM, wn0 = wave / WM * TN;

    floatx16 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = floatx16{0};

    if (k0 < kend) {
        CP cp;
        CQ cq;
        cp.init((const T *)a.P + (KSUM ? 0 : group * a.gp), a.ldp, PKC ? nullptr : a.prow, m0, a.m, k0, kend);
        cq.init((const T *)a.Q, a.ldq, a.qrow, n0, nend, k0, kend);
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
        const int at_p = CP::place(wm0 / 32), at_q = CQ::place(wn0 / 32);
        auto multiply = [&](const char *from) {
            int pa = at_p, qa = at_q;
            asm("" : "+v"(pa), "+v"(qa));          // its flips are made here, not held in registers over the loop
#pragma unroll
            for (int s = 0; s < BK / 16; ++s) {
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
        };
        // One step: its tile is there once all but the later tiles' copies are.
        auto step = [&](const char *from, char *to, int k) {
            if (NB > 2 && !IDX && k + BK < kend) copies_done<(NB - 2) * EACH>();
            else copies_done<0>();
            if (k + (NB - 1) * BK < kend) start(to, k + (NB - 1) * BK);
            multiply(from);
        };
        // The same where that tile's copies, and the next's, are whole.
        auto copy = [&](char *to, int k) {
            cp.template start<false>(to, k, kend);
            cq.template start<false>(to + CP::BYTES, k, kend);
            __builtin_amdgcn_sched_barrier(0);      // not after the products, where they would be late
        };
        auto steady = [&](const char *from, char *to, int k) {
            copies_done<IDX ? 0 : (NB - 2) * EACH>();
            copy(to, k + (NB - 1) * BK);
            multiply(from);
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
    // Lane l holds m = 8 q + 4 (l / 32) .. + 3 of column l % 32 in its values 4 q .. + 3.
    auto put = [&](int run, char *to) {
        const int lane = threadIdx.x & 63;
        if ((lane >> 4 & 1) != (run & 1)) return;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][run / 2][4 * q + e];
                __builtin_memcpy(to + SumRows<float, TM>::at(lane & 15, 8 * i + 2 * q + (lane >> 5)), v, 16);
            }
    };
    finish_tile<T, KSUM, TM, 2 * NTL>(a, lds0, group, n0 + wn0, nend, m0 + wm0, put, [](int run, int r) { return 16 * run + r; });
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
    T bias[V];
    load_bias<V>(b, group, m, bias);
    finish<V, T, A>(b, bias, a.crow ? (int64_t)a.crow[n] : n, m, s);
}

// ------------------------------------------------------------------- host

struct TileShape { int bm, bn; };
enum { REG_128, REG_32, REG_16, COPY_256, COPY_TALL, COPY_128 };
constexpr TileShape TILE_SHAPES[] = {{128, 128}, {128, 32}, {128, 16}, {256, 256}, {256, 128}, {128, 128}};

// Whether every chunk that a copy reads lies whole in the operands, 16 bytes aligned.
inline bool copies_fit(const TileArgs &a, bool pkc, bool qkc)
{
    const uintptr_t bits = (uintptr_t)a.P | (uintptr_t)a.Q | (uintptr_t)(a.ldp * 2) | (uintptr_t)(a.ldq * 2) |
                           (uintptr_t)(a.gp * 2) | (uintptr_t)(a.gq * 2);
    const int64_t k = pkc || qkc ? a.k : 0, m = pkc ? 0 : a.m, n = qkc ? 0 : a.n;
    return (bits & 15) == 0 && (k | m | n) % 8 == 0 && a.ldp < (1 << 22) && a.ldq < (1 << 22);
}

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
    int s = REG_128;
    if (!ksum && share <= 16) s = REG_16;
    else if (!ksum && share <= 48) s = REG_32;
    else if (sizeof(T) == 2 && copies_fit(*a, pkc, qkc)) {
        if (!ksum && tiles(COPY_256) >= 512) s = COPY_256;
        else s = tiles(COPY_TALL) >= 512 ? COPY_TALL : COPY_128;
    }
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

template <typename T, bool PKC, bool QKC, int BM, int BN, int WM, int WN, int BK, int NB, bool IDX>
int launch_copies(const TileArgs &a, hipStream_t s)
{
    const int64_t per = ((int64_t)a.tiles_m * a.tiles_n + NUM_XCD - 1) / NUM_XCD;
    const unsigned z = !PKC && !QKC && a.offsets ? (unsigned)a.groups : 1u;
    hipLaunchKernelGGL((tile_copy_kernel<T, PKC, QKC, BM, BN, WM, WN, BK, NB, IDX>),
                       dim3((unsigned)(per * NUM_XCD), (unsigned)a.split, z), dim3(WM * WN * 64), 0, s, a);
    return check_launch("tile_copy_kernel");
}

template <typename T, bool PKC>
int launch_columns(const TileArgs &a, int shape, hipStream_t s)
{
    if constexpr (sizeof(T) == 2) switch (shape) {
        case COPY_256: return launch_copies<T, PKC, true, 256, 256, 2, 4, 64, 2, false>(a, s);
        case COPY_TALL: return launch_copies<T, PKC, true, 256, 128, 2, 2, 32, 3, false>(a, s);
        case COPY_128: return launch_copies<T, PKC, true, 128, 128, 2, 2, 64, 2, false>(a, s);
        case REG_32: return launch_shape<T, PKC, true, 128, 32, 4, 1, false>(a, s);
        case REG_16: return launch_shape<T, PKC, true, 128, 16, 4, 1, false>(a, s);
        }
    else switch (shape) {
        case REG_32: return launch_shape<T, PKC, true, 128, 32, 2, 2, false>(a, s);
        case REG_16: return launch_shape<T, PKC, true, 128, 16, 2, 1, false>(a, s);
        }
    return launch_shape<T, PKC, true, 128, 128, 2, 2, false>(a, s);
}

template <typename T, bool IDX>
int launch_sums(const TileArgs &a, int shape, hipStream_t s)
{
    if constexpr (sizeof(T) == 2) {
        if (shape == COPY_TALL) return launch_copies<T, false, false, 256, 128, 2, 2, 32, 3, IDX>(a, s);
        if (shape == COPY_128) return launch_copies<T, false, false, 128, 128, 2, 2, 32, 3, IDX>(a, s);
    }
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
