// Orthogonalised updates: the Newton-Schulz iteration on a gradient (or momentum) matrix and the optimizer step around
// it.  The reference trains with Adam only (function/VAE_CNN_NN.py:204); this is the other optimizer for the same
// matrices.
//
//     X_0 = G / max(|G|_F, eps)   (transposed if G is tall: m <= n below)
//     A = X X^T,   B = b A + c A^2,   X <- a X + B X          `steps` times
//
// Numerics.  X is carried as two fp16 parts of X * 2^e (22 significand bits; the power of two comes from a bound on
// the singular values, so no largest magnitude has to be found) and every product is h h + h l + l h on the fp16
// matrix instruction, accumulated in fp32.  What the iteration amplifies (up to |a| = 3.4 times per step) is noise in
// the directions of small singular values; B maps into the span of the large ones, so errors of A, of B and of the
// product B X hardly reach those directions - only the rounding of X itself and of a X does.  The epilogue therefore
// adds a X in fp32 from both parts.  Measured against float64 this is at or below the error of the same iteration in
// plain fp32 (1e-6 .. 6e-6 of the norm, by spectrum; 1024 x 4624 of rank 16, whose empty directions hold nothing but
// rounding, 3.3e-5 and 5.1e-5).  One product of the high parts only (a X still from both) is the
// caller's choice: 0.3e-3 .. 1.9e-3 of the norm by itself, which takes a bf16 result of 1024 x 4624 Gaussian entries from 1.66e-3
// (its own rounding, with all parts) to 2.14e-3.
//
// Layout.  A matrix [R][K] lives as tiles of 32 rows x 16 k, [R/32][K/16][part 2][32 rows x 32 bytes], the two
// 16-byte halves of a row swapped where (row & 8): a 1 KiB tile is one LDS-DMA piece, a matrix operand with k along
// the row is one ds_read_b128 per lane, and the operand with k down the column (X in B X) is two transposing
// ds_read_b64_tr_b16 per lane of the same tile - so X needs no second, transposed copy.  With that swap the 16 lanes that
// a ds_read_b128 serves per clock fall on all 64 banks (4.1 clk per wave; 8.0 without it or with (row & 4)).
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <type_traits>
#include "common.h"
#include "../../include/mdnvae_hip.h"

namespace mdnvae {

typedef _Float16 mu_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 mu_h4 __attribute__((ext_vector_type(4)));
typedef short mu_s4 __attribute__((ext_vector_type(4)));
typedef short mu_s8 __attribute__((ext_vector_type(8)));
typedef float mu_acc __attribute__((ext_vector_type(16)));
typedef float mu_f4 __attribute__((ext_vector_type(4)));

constexpr int MU_FRAG = 1024;            // one part of one 32 x 16 tile
constexpr int MU_STEP = 2 * MU_FRAG;     // both parts
constexpr int MU_MAX = 32;               // table entries per launch (kernel arguments stay under 4 KB)
constexpr int MU_NORM_BLOCK = 8192;     // entries of G per workgroup of the norm pass

#define MU_GLOBAL_PTR(p) ((const __attribute__((address_space(1))) void*)(p))
#define MU_LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

// One entry: `count` matrices of one shape.  Workspace of a matrix: X (two buffers, 4 mp np bytes each), A, B (4 mp mp
// each), partial sums of A (splits > 1).  Matrix i of the entry starts at off + i * mu_matrix_bytes.
struct MuGeo {
    long off;
    int m, n, mp, np;                    // m <= n, and padded to the tile
    int trans;                           // the caller's matrix is [n][m]
    int tile;                            // of X X^T (m and n are padded to it)
    int splits, kper;                    // of the k steps of X X^T
    int count;
};
// Kernel arguments over N entries, 1 or MU_MAX.  The arguments are in no cache yet when a kernel starts, and a round trip to
// them is 0.6 us.  So a call over one shape has kernels of its own, without a table to look the entry up in (16 x 512 x 512 322 ->
// 302 us, 1024 x 4624 with one term 288 -> 267), and those over a table do so in one round trip (mu_entry).
template <int N>
struct MuTab {
    int start[N + 1];                    // first workgroup of each entry; INT_MAX past the last
    MuGeo e[N];
};
template <int N>
struct MuStarts { int s[N + 1]; };
// p: result or parameter, g: gradient (or the matrix itself), mom: momentum or null; matrix i at + i * stride elements
template <int N>
struct MuPtrs {
    void* p[N];
    const void* g[N];
    float* mom[N];
    float lr_scale[N];
};

__host__ __device__ inline long mu_tri(int t) { return (long)t * (t + 1) / 2; }
__host__ __device__ inline long mu_matrix_bytes(const MuGeo& g) {
    return 8L * g.mp * g.np + 8L * g.mp * g.mp + (g.splits > 1 ? (long)g.splits * mu_tri(g.mp / g.tile) * g.tile * g.tile * 4 : 0);
}

// The entry of a workgroup.  Each lane fetches one entry; which is the workgroup's is a ballot over the starts, and its values
// come from that lane: one round trip to the arguments instead of two, starts and then the entry (a convolutional encoder's
// list with one term 180 -> 160 us).
struct MuEntry {
    MuGeo ge;
    int e, first;                        // index and first workgroup
};
__device__ __forceinline__ int mu_lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ long mu_lane_value(long v, int lane) {
    const unsigned lo = (unsigned)mu_lane_value((int)v, lane), hi = (unsigned)mu_lane_value((int)(v >> 32), lane);
    return (long)((unsigned long)hi << 32 | lo);
}
template <int N>
__device__ __forceinline__ MuEntry mu_entry(const MuTab<N>& tab, int tl) {
    MuEntry o;
    if constexpr (N == 1) {
        o.ge = tab.e[0];
        o.e = o.first = 0;
    } else {
        static_assert(N == 32, "lanes 0 to 31");
        const int l = threadIdx.x & 31, start = tab.start[l];
        const MuGeo g = tab.e[l];
        o.e = __popc((unsigned)__ballot(tl >= start)) - 1;
        o.first = mu_lane_value(start, o.e);
        o.ge.off = mu_lane_value(g.off, o.e);
        o.ge.m = mu_lane_value(g.m, o.e);
        o.ge.n = mu_lane_value(g.n, o.e);
        o.ge.mp = mu_lane_value(g.mp, o.e);
        o.ge.np = mu_lane_value(g.np, o.e);
        o.ge.trans = mu_lane_value(g.trans, o.e);
        o.ge.tile = mu_lane_value(g.tile, o.e);
        o.ge.splits = mu_lane_value(g.splits, o.e);
        o.ge.kper = mu_lane_value(g.kper, o.e);
        o.ge.count = mu_lane_value(g.count, o.e);
    }
    return o;
}
// entry e of a pointer array, the same way
template <int N, typename P>
__device__ __forceinline__ P* mu_pick(P* const (&a)[N], int e) {
    if constexpr (N == 1) return a[0];
    else return reinterpret_cast<P*>(mu_lane_value(reinterpret_cast<long>(a[threadIdx.x & 31]), e));
}

// u of one entry: with momentum, M <- mu M + g and u = g + mu M (Nesterov) or M; without, g itself
struct MuMom { float mu; int nesterov; };
template <typename T>
__device__ __forceinline__ float mu_update(const T* g, float* mom, long i, const MuMom& mm) {
    const float gv = (float)g[i];
    if (!mom) return gv;
    const float m = mm.mu * mom[i] + gv;
    mom[i] = m;
    return mm.nesterov ? gv + mm.mu * m : m;
}

// ---- norm pass: momentum, and each workgroup's sum of squares (float64: the squares of finite fp32 numbers neither
// overflow nor vanish).  Bound by memory: 4624 x 4624 fp32 20 us, 4.3 TB/s; 1024 x 4624 6 us ---------------------------------
template <int N, typename T>
__global__ __launch_bounds__(256) void mu_norm_kernel(MuTab<N> tab, MuPtrs<N> ptrs, MuMom mm, double* __restrict__ partial) {
    __shared__ double red[4];
    const MuEntry entry = mu_entry(tab, blockIdx.x);
    const MuGeo& ge = entry.ge;
    const int e = entry.e;
    const long len = (long)ge.m * ge.n, per = (len + MU_NORM_BLOCK - 1) / MU_NORM_BLOCK;
    const long local = blockIdx.x - entry.first, mat = local / per, blk = local - mat * per;
    const T* g = static_cast<const T*>(mu_pick(ptrs.g, e)) + mat * len;
    float* mom = mu_pick(ptrs.mom, e);
    const long lo = blk * MU_NORM_BLOCK;
    long hi = min(len, lo + MU_NORM_BLOCK);
    double s = 0.0;
    typedef T vec __attribute__((ext_vector_type(4)));
    if (((reinterpret_cast<uintptr_t>(g + lo) & (4 * sizeof(T) - 1)) | (reinterpret_cast<uintptr_t>(mom) & 15)) == 0) {
        constexpr int V = MU_NORM_BLOCK / 1024;            // four entries per access, all loads ahead of the stores
        auto at = [&](int i) { return lo + (i * 256 + threadIdx.x) * 4; };
        auto take = [&](const vec& gv, const mu_f4& mv, long i) {
            mu_f4 out;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float gk = (float)gv[k];
                out[k] = mom ? mm.mu * mv[k] + gk : gk;
                const double u = mom && mm.nesterov ? (double)(gk + mm.mu * out[k]) : (double)out[k];
                s += u * u;
            }
            if (mom) *reinterpret_cast<mu_f4*>(mom + i) = out;
        };
        vec gv[V];
        mu_f4 mv[V];
        if (hi - lo == MU_NORM_BLOCK) {
#pragma unroll
            for (int i = 0; i < V; ++i) gv[i] = *reinterpret_cast<const vec*>(g + at(i));
            if (mom) {
#pragma unroll
                for (int i = 0; i < V; ++i) mv[i] = *reinterpret_cast<const mu_f4*>(mom + at(i));
            }
#pragma unroll
            for (int i = 0; i < V; ++i) take(gv[i], mv[i], at(i));
            hi = lo;                                       // no tail
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (at(i) + 4 <= hi) {
                    gv[i] = *reinterpret_cast<const vec*>(g + at(i));
                    if (mom) mv[i] = *reinterpret_cast<const mu_f4*>(mom + at(i));
                }
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (at(i) + 4 <= hi) take(gv[i], mv[i], at(i));
        }
        const long tail = lo + ((hi - lo) & ~3L) + threadIdx.x;
        if (tail < hi) {
            const double u = (double)mu_update(g, mom, tail, mm);
            s += u * u;
        }
    } else {
        for (long i = lo + threadIdx.x; i < hi; i += 256) {
            const double u = (double)mu_update(g, mom, i, mm);
            s += u * u;
        }
    }
    s = block_sum<256, double>(s, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// u scale / max(|u|_F, eps) as ldexp(u, shift) * factor, since the reciprocal alone may lie outside fp32: |u|_F^2 = m 4^e with m
// in [0.25, 1), shift = -e, factor = scale / sqrt(m).  A norm that is not finite (an infinity or a NaN in the matrix)
// gives NaN, and with it a result that is NaN throughout.
struct MuNorm {
    int shift;
    float factor;
    __device__ __forceinline__ MuNorm(double sum, float eps, float scale) {
        const double least = (double)eps * (double)eps;
        const double s = sum < least ? least : sum;
        const int two_e = ((int)((__double_as_longlong(s) >> 52) & 0x7ff) - 1022 + 1) & ~1;      // a normal number: eps is an fp32
        const float m = (float)ldexp(s, -two_e);
        shift = -(two_e >> 1);
        float r = __builtin_amdgcn_rsqf(m);
        r = r * fmaf(-0.5f * m * r, r, 1.5f);               // one Newton step on the hardware's estimate
        factor = s <= 1.7e308 ? scale * r : __uint_as_float(0x7fc00000u);
    }
    __device__ __forceinline__ float operator()(float u) const { return ldexpf(u, shift) * factor; }
};

// t = h + l to 22 bits.  t is made a number in a register first: left to itself the compiler rounds the product that t came
// from straight to fp16 for one use of h and through fp32 for the other, and where the two differ (once in 2^13) h + l is
// off by an fp16 step - 5e-6 of a tensor's norm.
__device__ __forceinline__ void mu_parts(float t, _Float16& h, _Float16& l) {
    asm("" : "+v"(t));
    h = (_Float16)t;
    l = (_Float16)fmaf((float)h, -1.0f, t);                 // one instruction that takes h as it is
}

// byte offset of (row, 16-byte half) inside a tile
__device__ __forceinline__ int mu_at(int row, int half) { return row * 32 + ((half ^ ((row >> 3) & 1)) << 4); }

// ---- split pass: X_0 in parts; one workgroup = 32 rows x 64 columns of X, through LDS so that lanes run along the
// caller's contiguous dimension.  4624 x 4624 fp32 53 us, 3.3 TB/s read and written; 1024 x 4624 12 us ----------------------
template <int N, typename T>
__global__ __launch_bounds__(256) void mu_split_kernel(MuTab<N> tab, MuStarts<N> norm, MuPtrs<N> ptrs, MuMom mm, float eps, float scale,
                                                       const double* __restrict__ partial, char* __restrict__ ws) {
    __shared__ float tile[32][65];
    __shared__ double red[4];
    const MuEntry entry = mu_entry(tab, blockIdx.x);
    const MuGeo& ge = entry.ge;
    const int e = entry.e;
    const int nt = ge.np / 64, per = (ge.mp / 32) * nt;
    const int local = blockIdx.x - entry.first, mat = local / per, t = local - mat * per;
    const int r0 = (t / nt) * 32, c0 = (t % nt) * 64;
    const long len = (long)ge.m * ge.n, nper = (len + MU_NORM_BLOCK - 1) / MU_NORM_BLOCK;
    const double* part = partial + (N == 1 ? 0 : norm.s[e]) + mat * nper;
    const T* g = static_cast<const T*>(mu_pick(ptrs.g, e)) + mat * len;
    const float* mom = mu_pick(ptrs.mom, e);
    // this thread's eight entries: along the caller's rows (lanes over columns) or down them; loads first, clamped to entry 0
    const int tr = ge.trans ? threadIdx.x & 31 : threadIdx.x >> 6, tc = ge.trans ? threadIdx.x >> 5 : threadIdx.x & 63;
    float gv[8], mv[8];
    bool ok[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int r = r0 + tr + (ge.trans ? 0 : 4 * k), c = c0 + tc + (ge.trans ? 8 * k : 0);
        ok[k] = r < ge.m && c < ge.n;
        const long at = ok[k] ? (ge.trans ? (long)c * ge.m + r : (long)r * ge.n + c) : 0;
        gv[k] = (float)g[at];
        mv[k] = mom ? mom[at] : 0.0f;
    }
    double s = 0.0;
    for (long i = threadIdx.x; i < nper; i += 256) s += part[i];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        // the momentum is this step's already
        const float u = !mom ? gv[k] : mm.nesterov ? gv[k] + mm.mu * mv[k] : mv[k];
        tile[tr + (ge.trans ? 0 : 4 * k)][tc + (ge.trans ? 8 * k : 0)] = ok[k] ? u : 0.0f;
    }
    __syncthreads();
    const MuNorm normal((red[0] + red[1]) + (red[2] + red[3]), eps, scale);
    const int r = threadIdx.x >> 3, c8 = threadIdx.x & 7;
    mu_h8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        _Float16 h, l;
        mu_parts(normal(tile[r][c8 * 8 + k]), h, l);
        hi[k] = h;
        lo[k] = l;
    }
    char* dst = ws + ge.off + mat * mu_matrix_bytes(ge) + ((long)(r0 >> 5) * (ge.np >> 4) + (c0 >> 4) + (c8 >> 1)) * MU_STEP + mu_at(r, c8 & 1);
    *reinterpret_cast<mu_h8*>(dst) = hi;
    *reinterpret_cast<mu_h8*>(dst + MU_FRAG) = lo;
}

// ---- products --------------------------------------------------------------------------------------------------------
// GRAM: A = X X^T (upper tiles, mirrored), POLY: B = b A + c A^2 (the same), STEP: X <- a X + B X.
enum { MU_GRAM = 0, MU_POLY = 1, MU_STEP_X = 2 };

struct MuScale {
    float f_acc;       // what the accumulator is multiplied with (scales undone, the destination's applied, coefficient)
    float f_add;       // what the tile already there (A in POLY, X in STEP) is multiplied with
};

// lane offsets of the two ways to read an operand of 32 x 16 out of LDS
struct MuLane {
    int direct;        // rows of the tile are operand rows
    int tr;            // columns of two adjacent 16-row half tiles (512 bytes each) are operand rows: k 0..3 of the lane's
};                     // eight here, k 4..7 four rows (128 bytes) further on
__device__ __forceinline__ MuLane mu_lane(int lane) {
    MuLane o;
    o.direct = mu_at(lane & 31, lane >> 5);
    const int g = lane >> 4, n16 = g & 1, h = g >> 1, r = (lane & 15) >> 2, ch = lane & 3;
    o.tr = n16 * 512 + (8 * h + r) * 32 + (((ch >> 1) ^ h) << 4) + (ch & 1) * 8;
    return o;
}
__device__ __forceinline__ mu_h8 mu_join(mu_s4 a, mu_s4 b) {
    mu_s8 f;
    f[0] = a[0]; f[1] = a[1]; f[2] = a[2]; f[3] = a[3];
    f[4] = b[0]; f[5] = b[1]; f[6] = b[2]; f[7] = b[3];
    return __builtin_bit_cast(mu_h8, f);
}
__device__ __forceinline__ mu_h8 mu_tr(const char* p) {
    return mu_join(__builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) mu_s4*)(p)),
                   __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) mu_s4*)(p + 128)));
}
// N operands 1 KiB apart.  In the products' loop the builtin would make the compiler wait for every LDS-DMA in flight (it
// cannot tell that they go elsewhere), which takes the ring's depth away: 1.6x the time of a step.  So the reads and their
// wait are one block of assembly.
template <int N>
__device__ __forceinline__ void mu_tr_block(const char* p, mu_h8 (&out)[N]) {
    const unsigned at = (unsigned)(size_t)(__attribute__((address_space(3))) const char*)(p);
    mu_s4 a[2 * N];
    if constexpr (N == 4) {
        asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%9\n\t"
                     "ds_read_b64_tr_b16 %2, %8 offset:%10\n\tds_read_b64_tr_b16 %3, %8 offset:%11\n\t"
                     "ds_read_b64_tr_b16 %4, %8 offset:%12\n\tds_read_b64_tr_b16 %5, %8 offset:%13\n\t"
                     "ds_read_b64_tr_b16 %6, %8 offset:%14\n\tds_read_b64_tr_b16 %7, %8 offset:%15\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(a[4]), "=&v"(a[5]), "=&v"(a[6]), "=&v"(a[7])
                     : "v"(at), "n"(128), "n"(MU_FRAG), "n"(MU_FRAG + 128), "n"(2 * MU_FRAG), "n"(2 * MU_FRAG + 128), "n"(3 * MU_FRAG),
                       "n"(3 * MU_FRAG + 128)
                     : "memory");
    } else if constexpr (N == 2) {
        asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:128\n\t"
                     "ds_read_b64_tr_b16 %2, %4 offset:1024\n\tds_read_b64_tr_b16 %3, %4 offset:1152\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3])
                     : "v"(at)
                     : "memory");
    } else {
        static_assert(N == 1, "one, two or four operands");
        asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:128\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(a[0]), "=&v"(a[1])
                     : "v"(at)
                     : "memory");
    }
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = mu_join(a[2 * i], a[2 * i + 1]);
}

// stages of the ring: two workgroups of 128 x 128 fill a CU's 160 KB; four to nine measured alike
constexpr int MU_RING = 5;

// acc += operand rows [TILE] x operand columns [TILE] over k steps [k0, k1).  Four waves (2 x 2), wave tile TILE/2 squared.
// Ring of NBUF stages, one k step each, filled by LDS-DMA; one counted wait and one barrier per step.  The operands of
// step i + 1 are read from LDS into a second set of registers under the matrix instructions of step i, and reads and
// DMAs are dealt out between the matrix instructions: a wave issues in order, and sixteen DMAs of a step take the
// CU's address unit 256 clk - issued in one go ahead of the products they cost that time in every step.
// TR: the row operand is X read down its columns (rsrc: tile (0, first n step), nsteps: n steps of a row of tiles).
// early(): EXTRA loads into registers that the epilogue wants, issued eight steps before the end and not behind it (B X at
// 4624 x 4624 590 -> 576 us).
// The counted waits rely on exactly EXTRA loads: mu_load_block's are eight bytes each, no two of a lane
// adjacent (half tiles lie 16 bytes apart in an order that depends on the row, parts 1 KiB), so none can be joined.  A CPU test
// counts them in the built library.
template <int TILE, int TERMS, bool TR, int EXTRA, typename EARLY>
__device__ __forceinline__ void mu_mainloop(const char* rsrc, const char* csrc, int nsteps, int KS, int k0, int k1, char* smem,
                                            mu_acc (&acc)[TILE / 64][TILE / 64], EARLY early) {
    constexpr int NBUF = MU_RING;
    constexpr int F = TILE / 32, W = TILE / 64;          // tiles per side, of the workgroup and of a wave
    constexpr int NP = TERMS == 3 ? 2 : 1;
    constexpr int SIDE = F * NP, PPW = 2 * SIDE / 4;     // pieces of one side, pieces per wave
    constexpr int STAGE = 2 * SIDE * MU_FRAG;
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wid >> 1, wc = wid & 1;
    const MuLane ln = mu_lane(lane);
    const char* src[PPW];
    bool tr[PPW];
#pragma unroll
    for (int i = 0; i < PPW; ++i) {
        const int q = wid + 4 * i, side = q / SIDE, f = (q % SIDE) / NP, part = (q % SIDE) % NP;
        tr[i] = TR && side == 0;
        if (tr[i]) src[i] = rsrc + (2L * f + (lane >> 5)) * MU_STEP + part * MU_FRAG + (lane & 31) * 16;
        else src[i] = (side == 0 ? rsrc : csrc) + (long)f * KS * MU_STEP + part * MU_FRAG + lane * 16;
    }
    auto stage = [&](int i, int buf, int ks) {
        const long at = tr[i] ? (long)(ks >> 1) * nsteps * MU_STEP + (ks & 1) * 512 : (long)ks * MU_STEP;
        __builtin_amdgcn_global_load_lds(MU_GLOBAL_PTR(src[i] + at), MU_LDS_PTR(smem + buf * STAGE + (wid + 4 * i) * MU_FRAG), 16, 0, 0);
    };
    constexpr int OPS = W * NP;                          // operands of a side
    mu_h8 r[2][OPS], c[2][OPS];
    const char* my_r = smem + wr * OPS * MU_FRAG + (TR ? ln.tr : ln.direct);
    const char* my_c = smem + (SIDE + wc * OPS) * MU_FRAG + ln.direct;
    constexpr int READS = TR ? OPS : 2 * OPS;            // single reads; the transposing ones go as a block
    auto read = [&](int n, int set, int buf) {
        if (n < OPS) c[set][n] = *reinterpret_cast<const mu_h8*>(my_c + buf * STAGE + n * MU_FRAG);
        else r[set][n - OPS] = *reinterpret_cast<const mu_h8*>(my_r + buf * STAGE + (n - OPS) * MU_FRAG);
    };
    constexpr int MF = (TERMS == 3 ? 3 : 1) * W * W;     // matrix instructions of a step
    auto multiply = [&](int n, int set) {
        const int t = n / (W * W), i = n / W % W, j = n % W;      // smallest terms first; a term of all blocks, then the next
        const int pr = TERMS == 3 && t == 0 ? 1 : 0, pc = TERMS == 3 && t == 1 ? 1 : 0;
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(r[set][i * NP + pr], c[set][j * NP + pc], acc[i][j], 0, 0, 0);
    };
    const int nk = k1 - k0;                              // at least one
    // past the end the last step is fetched again, into a buffer nobody reads any more: every wave always has the same
    // number of operations in flight, and one counted wait fits every iteration
#pragma unroll
    for (int s = 0; s < NBUF - 1; ++s)
#pragma unroll
        for (int i = 0; i < PPW; ++i) stage(i, s, k0 + min(s, nk - 1));
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NBUF - 2) * PPW) : "memory");
#pragma unroll
    for (int n = 0; n < READS; ++n) read(n, 0, 0);
    if constexpr (TR) mu_tr_block(my_r, r[0]);
    int b_read = 1, b_fill = NBUF - 1;
    // step `it`: its operands are in (or on their way to) register set `set`
    auto step = [&](int set, int it, auto extra) {
        // own pieces of step it + 1 have landed, own reads of step it are done: after the barrier everybody's, and the buffer
        // of step it - 1 (read before the previous barrier) is free
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NBUF - 3) * PPW + decltype(extra)::value) : "memory");
        const int fill = k0 + min(it + NBUF - 1, nk - 1);
        constexpr int HALF = MF * 2 / 3 > 0 ? MF * 2 / 3 : 1;      // reads go first: they have to be back by the next step
#pragma unroll
        for (int n = 0; n < MF; ++n) {
            multiply(n, set);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < READS; ++k)
                if (k * HALF / READS == n) read(k, set ^ 1, b_read);
            if constexpr (TR) {
                if (n == MF / 2) mu_tr_block(my_r + b_read * STAGE, r[set ^ 1]);
            }
#pragma unroll
            for (int k = 0; k < PPW; ++k)
                if (((k + 1) * MF - 1) / PPW == n) stage(k, b_fill, fill);
            __builtin_amdgcn_sched_barrier(0);
        }
        b_fill = b_fill + 1 == NBUF ? 0 : b_fill + 1;
        b_read = b_read + 1 == NBUF ? 0 : b_read + 1;
    };
    std::integral_constant<int, 0> none;
    int it = 0;
    if constexpr (EXTRA > 0) {
        static_assert((NBUF - 3) * PPW + EXTRA < 64, "the counter of loads in flight has six bits");
        static_assert(NBUF == 5, "three steps wait for stages older than the extra loads");
        std::integral_constant<int, EXTRA> more;
        if (nk >= 8) {
            for (; it + 8 < nk; it += 2) {
                step(0, it, none);
                step(1, it + 1, none);
            }
            early();
            step(0, it, more);
            step(1, it + 1, more);
            step(0, it + 2, more);
            step(1, it + 3, none);
            it += 4;
        } else {
            early();
        }
    }
    for (; it + 1 < nk; it += 2) {
        step(0, it, none);
        step(1, it + 1, none);
    }
    if (it < nk) {
#pragma unroll
        for (int n = 0; n < MF; ++n) multiply(n, 0);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the epilogue reuses the stages
}

// accumulator register e of a 32 x 32 block: row (e & 3) + 8 (e >> 2) + 4 (lane >> 5), column lane & 31.
// Block with its first row at k = kr (of the destination's row) and columns = rows of destination row tile `rt`:
// four consecutive k per register group leave as 8 bytes per part.
__device__ __forceinline__ long mu_block_at(int rt, int KS, int kr, int q, int lane) {
    const int col = lane & 31, h = lane >> 5;
    return ((long)rt * KS + (kr >> 4) + (q >> 1)) * MU_STEP + mu_at(col, q & 1) + h * 8;
}
template <int NP>
__device__ __forceinline__ void mu_put(char* at, const float (&v)[4]) {
    mu_h4 hi, lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        _Float16 h, l;
        mu_parts(v[k], h, l);
        hi[k] = h;
        lo[k] = l;
    }
    *reinterpret_cast<mu_h4*>(at) = hi;
    if constexpr (NP == 2) *reinterpret_cast<mu_h4*>(at + MU_FRAG) = lo;
}
// the same place read: a block's worth at once (16 values per lane), before anything is stored - a load behind a store that
// might alias it waits for its own round trip, sixteen times in a tile
struct MuOld {
    mu_h4 hi[4], lo[4];
};
template <int NP>
__device__ __forceinline__ void mu_load_block(MuOld& o, const char* fm, int rt, int KS, int kr, int lane) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const char* at = fm + mu_block_at(rt, KS, kr, q, lane);
        o.hi[q] = *reinterpret_cast<const mu_h4*>(at);
        if constexpr (NP == 2) o.lo[q] = *reinterpret_cast<const mu_h4*>(at + MU_FRAG);
    }
}
template <int NP>
__device__ __forceinline__ float mu_old(const MuOld& o, int q, int k) {
    return NP == 2 ? (float)o.hi[q][k] + (float)o.lo[q][k] : (float)o.hi[q][k];
}

// LDS written by some lanes of the wave, read by others: the hardware keeps a wave's LDS operations in order, the
// compiler has to be told
__device__ __forceinline__ void mu_wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One 32 x 32 block of a symmetric matrix: rb counts along k of the direct image, cb along its rows.  `mirror`: also the block
// on the other side of the diagonal, transposed through 4 KiB of LDS that belong to the wave.
template <int NP, bool POLY>
__device__ __forceinline__ void mu_emit_block(const mu_acc& acc, char* dst, const MuOld& old, int KS, int rb, int cb, bool mirror,
                                              const MuScale& sc, char* mine) {
    const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = acc[4 * q + k] * sc.f_acc + (POLY ? mu_old<NP>(old, q, k) * sc.f_add : 0.0f);
        mu_put<NP>(dst + mu_block_at(cb, KS, rb * 32, q, lane), v);
        if (mirror) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int row = 8 * q + 4 * h + k;
                _Float16 hi, lo;
                mu_parts(v[k], hi, lo);
                char* t = mine + (col >> 4) * 1024 + mu_at(row, (col >> 3) & 1) + (col & 7) * 2;
                *reinterpret_cast<_Float16*>(t) = hi;
                if constexpr (NP == 2) *reinterpret_cast<_Float16*>(t + 2048) = lo;
            }
        }
    }
    if (mirror) {
        mu_wave_fence();
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const mu_h8 v = *reinterpret_cast<const mu_h8*>(mine + p * 2048 + s * 1024 + lane * 16);
                *reinterpret_cast<mu_h8*>(dst + ((long)rb * KS + cb * 2 + s) * MU_STEP + p * MU_FRAG + lane * 16) = v;
            }
        mu_wave_fence();
    }
}
// tile t of the upper triangle, column by column: (i <= j)
__device__ __forceinline__ void mu_pair(int t, int& i, int& j) {
    j = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((j + 1) * (j + 2) / 2 <= t) ++j;
    while (j * (j + 1) / 2 > t) --j;
    i = t - j * (j + 1) / 2;
}
// the same tiles in bands of eight columns, rows of a band one after the other: 64 neighbours share 8 + 8 operand panels
__device__ __forceinline__ void mu_pair_banded(int t, int T, int& i, int& j) {
    mu_pair(t, i, j);
    const int j0 = j & ~7, w = min(8, T - j0), r = t - j0 * (j0 + 1) / 2, rect = j0 * w;
    if (r < rect) {
        i = r / w;
        j = j0 + r - i * w;
    } else {
        mu_pair(r - rect, i, j);
        i += j0;
        j += j0;
    }
}

// workgroups of one XCD (every eighth) take consecutive tiles, which share operand panels through its L2
__device__ __forceinline__ int mu_tile_index(int total) {
    const int chunk = (total + 7) >> 3;
    const int t = (blockIdx.x & 7) * chunk + (blockIdx.x >> 3);
    return t < total ? t : -1;
}

// GRAM and POLY, tiles of the upper triangle.  4624 x 4624 fp32 284 to 310 us each, 1.06 to 1.15 PFLOP/s of fp16 products (the card's
// large library products: 1.0): the clock falls to 1.7 GHz under them, the matrix pipes are 62 to 64 % busy.  1024 x 4624 20
// to 22 and 13 us.
template <int N, int TILE, int TERMS, int MODE>
__global__ __launch_bounds__(256) void mu_sym_kernel(MuTab<N> tab, int total, char* __restrict__ ws, int ping, MuScale sc) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int tl = mu_tile_index(total);
    const MuEntry entry = mu_entry(tab, max(tl, 0));        // ahead of the branch: its loads go with that of `total`
    if (tl < 0) return;
    const MuGeo& ge = entry.ge;
    const int T = ge.mp / TILE, ntri = T * (T + 1) / 2;
    const int splits = MODE == MU_GRAM ? ge.splits : 1;
    const int local = tl - entry.first, mat = local / (ntri * splits), rest = local - mat * ntri * splits;
    const int s = rest / ntri, t = rest - s * ntri;
    int ti, tj;
    mu_pair_banded(t, T, ti, tj);
    char* base = ws + ge.off + mat * mu_matrix_bytes(ge);
    const long xs = 4L * ge.mp * ge.np, as = 4L * ge.mp * ge.mp;
    char* A = base + 2 * xs;
    const int KS = MODE == MU_GRAM ? ge.np >> 4 : ge.mp >> 4;
    const char* src = MODE == MU_GRAM ? base + ping * xs : A;
    const int k0 = s * ge.kper, k1 = MODE == MU_GRAM ? min(KS, k0 + ge.kper) : KS;
    mu_acc acc[TILE / 64][TILE / 64];
#pragma unroll
    for (int i = 0; i < TILE / 64; ++i)
#pragma unroll
        for (int j = 0; j < TILE / 64; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.0f;
    const long rows = (long)(TILE / 32) * KS * MU_STEP;
    constexpr int W = TILE / 64, F = TILE / 32, NP = TERMS == 3 ? 2 : 1;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rb0 = ti * F + (wid >> 1) * W, cb0 = tj * F + (wid & 1) * W;
    MuOld old[W][W];                                   // POLY: the tile of A
    mu_mainloop<TILE, TERMS, false, MODE == MU_POLY ? W * W * 4 * NP : 0>(
        src + ti * rows, src + tj * rows, 0, KS, MODE == MU_GRAM ? k0 : 0, k1, smem, acc, [&] {
#pragma unroll
            for (int i = 0; i < W; ++i)
#pragma unroll
                for (int j = 0; j < W; ++j) mu_load_block<NP>(old[i][j], A, cb0 + j, KS, (rb0 + i) * 32, lane);
        });
    if (MODE == MU_GRAM && splits > 1) {
        // this split's share, as the registers lie (the reducing kernel has the same lanes): 256 bytes per store
        float* part = reinterpret_cast<float*>(A + 2 * as) + ((long)s * ntri + t) * TILE * TILE;
#pragma unroll
        for (int i = 0; i < TILE / 64; ++i)
#pragma unroll
            for (int j = 0; j < TILE / 64; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    mu_f4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    reinterpret_cast<mu_f4*>(part)[((wid * (TILE / 64) + i) * (TILE / 64) + j) * 256 + q * 64 + lane] = v;
                }
        return;
    }
    char* dst = MODE == MU_POLY ? A + as : A;
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j)
            mu_emit_block<NP, MODE == MU_POLY>(acc[i][j], dst, old[i][j], ge.mp >> 4, rb0 + i, cb0 + j, ti != tj, sc, smem + wid * 4096);
}

// The sum of the splits in fixed order, then what the product kernel does when there is one.  A wave per 32 x 32 block (the
// blocks of a tile lie one after the other in a share): 16 of them per tile, for there are few tiles where there are splits.
// Seven shares of 1024 x 1024 6 us, 2.8 TB/s with its start (one workgroup per tile: 35 us).
template <int N, int TILE, int TERMS>
__global__ __launch_bounds__(256) void mu_reduce_kernel(MuTab<N> tab, char* __restrict__ ws, MuScale sc) {
    __shared__ __attribute__((aligned(1024))) char smem[4 * 4096];
    constexpr int W = TILE / 64, WGS = W * W;              // workgroups per tile, four blocks each
    const MuEntry entry = mu_entry(tab, blockIdx.x / WGS);
    const MuGeo& ge = entry.ge;
    if (ge.splits == 1) return;
    const int T = ge.mp / TILE, ntri = T * (T + 1) / 2;
    const int local = blockIdx.x / WGS - entry.first, mat = local / ntri, t = local - mat * ntri;
    int ti, tj;
    mu_pair_banded(t, T, ti, tj);
    char* base = ws + ge.off + mat * mu_matrix_bytes(ge);
    const long xs = 4L * ge.mp * ge.np, as = 4L * ge.mp * ge.mp;
    char* A = base + 2 * xs;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int block = (blockIdx.x % WGS) * 4 + wid;        // (wave of the product kernel, i, j)
    const mu_f4* part = reinterpret_cast<const mu_f4*>(A + 2 * as) + ((long)t * 4 * WGS + block) * 256 + lane;
    mu_acc acc;
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] = 0.0f;
#pragma unroll 4
    for (int s = 0; s < ge.splits; ++s) {
        const mu_f4* p = part + (long)s * ntri * (TILE * TILE / 4);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const mu_f4 v = p[q * 64];
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[4 * q + k] += v[k];
        }
    }
    const int w = block / WGS, ij = block % WGS;
    const int rb = ti * (TILE / 32) + (w >> 1) * W + ij / W, cb = tj * (TILE / 32) + (w & 1) * W + ij % W;
    mu_emit_block<TERMS == 3 ? 2 : 1, false>(acc, A, MuOld(), ge.mp >> 4, rb, cb, ti != tj, sc, smem + wid * 4096);
}

// STEP: D rows = 128 (64) columns n of X, D columns = rows m, so that a lane's four consecutive rows are consecutive in X's
// tiles.  LAST: the result leaves in the caller's layout and type.  4624 x 4624 fp32 576 to 640 us, 1.0 to 1.1 PFLOP/s; 1024 x
// 4624 44 to 46 us on tiles of 64 x 64 (with one term 24 on 128 x 128), for 296 tiles of 128 x 128 are more than the CUs take in one round.
template <int N, typename T, int TILE, int TERMS, bool LAST>
__global__ __launch_bounds__(256) void mu_step_kernel(MuTab<N> tab, int total, MuPtrs<N> ptrs, char* __restrict__ ws, int ping, MuScale sc,
                                                      float decay, int is_step) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int tl = mu_tile_index(total);
    const MuEntry entry = mu_entry(tab, max(tl, 0));        // ahead of the branch: its loads go with that of `total`
    if (tl < 0) return;
    const MuGeo& ge = entry.ge;
    const int e = entry.e;
    const int TM = ge.mp / TILE, TN = ge.np / TILE;
    const int local = tl - entry.first, mat = local / (TM * TN), rest = local - mat * TM * TN;
    // bands of eight tile columns, rows of a band one after the other: 64 neighbours share 8 + 8 operand panels
    const int n0 = rest / (8 * TM) * 8, w = min(8, TN - n0), inband = rest - n0 * TM;
    const int tm = inband / w, tn = n0 + inband - tm * w;
    char* base = ws + ge.off + mat * mu_matrix_bytes(ge);
    const long xs = 4L * ge.mp * ge.np, as = 4L * ge.mp * ge.mp;
    const char* X = base + ping * xs;
    char* Y = base + (ping ^ 1) * xs;
    const char* B = base + 2 * xs + as;
    const int NS = ge.np >> 4, KS = ge.mp >> 4;
    constexpr int W = TILE / 64, F = TILE / 32;
    mu_acc acc[W][W];
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.0f;
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wid >> 1, wc = wid & 1, h = lane >> 5;
    MuOld old[W][W];
    mu_mainloop<TILE, TERMS, true, W * W * 8>(
        X + (long)tn * (TILE / 16) * MU_STEP, B + (long)tm * F * KS * MU_STEP, NS, KS, 0, KS, smem, acc, [&] {
#pragma unroll
            for (int i = 0; i < W; ++i)
#pragma unroll
                for (int j = 0; j < W; ++j)
                    mu_load_block<2>(old[i][j], X, tm * F + wc * W + j, NS, (tn * F + wr * W + i) * 32, lane);
        });
    const long len = (long)ge.m * ge.n;
    T* out = LAST ? static_cast<T*>(mu_pick(ptrs.p, e)) + mat * len : nullptr;
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int nb = tn * F + wr * W + i, mb = tm * F + wc * W + j;
            float v[16];
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[4 * q + k] = acc[i][j][4 * q + k] * sc.f_acc + mu_old<2>(old[i][j], q, k) * sc.f_add;
            if constexpr (!LAST) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float four[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                    mu_put<2>(Y + mu_block_at(mb, NS, nb * 32, q, lane), four);
                }
            } else {
                // lanes along the caller's contiguous dimension: m as it is, n through 32 x 33 floats that belong to the wave
                long at[16];
                bool ok[16];
                if (ge.trans) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const int m = mb * 32 + (lane & 31), n = nb * 32 + 8 * (k >> 2) + 4 * h + (k & 3);
                        at[k] = (long)n * ge.m + m;
                        ok[k] = m < ge.m && n < ge.n;
                    }
                } else {
                    float* mine = reinterpret_cast<float*>(smem) + wid * 32 * 33;
#pragma unroll
                    for (int k = 0; k < 16; ++k) mine[(lane & 31) * 33 + 8 * (k >> 2) + 4 * h + (k & 3)] = v[k];
                    mu_wave_fence();
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        v[k] = mine[(2 * k + h) * 33 + (lane & 31)];
                        const int m = mb * 32 + 2 * k + h, n = nb * 32 + (lane & 31);
                        at[k] = (long)m * ge.n + n;
                        ok[k] = m < ge.m && n < ge.n;
                    }
                    mu_wave_fence();
                }
                if (is_step) {
                    T p[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) p[k] = out[ok[k] ? at[k] : 0];      // entry 0 stands in: sixteen 16-bit loads in flight
#pragma unroll
                    for (int k = 0; k < 16; ++k) v[k] = decay * (float)p[k] - ptrs.lr_scale[e] * v[k];
                }
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (ok[k]) out[at[k]] = (T)v[k];
            }
        }
}

// ---- small matrices: the whole step in one workgroup ----------------------------------------------------------------------
// X and A in parts fit LDS (mp np + mp mp <= 38912 entries, mp and np multiples of 32; mu_small): norm, all iterations and the
// parameter step in one launch, one matrix per workgroup of up to 16 waves.  A 32 x 32 block of a product belongs to one
// wave.  Where two X and both A and B fit (up to 96 x 96) a product goes to the other buffer; else its registers are held until
// a barrier says that everybody has read what they overwrite.  Always both parts: such a matrix is bound by latencies and
// barriers, not by its products (68 x 68, five iterations: 28 us, 3.9 of them per iteration, of which the matrix
// instructions on the SIMD with three of the nine waves are 2.2).  A wave with one block of X keeps it, and its block of A, in
// fp32 registers from product to product instead of joining the parts it reads back (31 us).
constexpr int MU_SMALL_ENTRIES = 38912;
constexpr int MU_SMALL_NT = 1024;
constexpr int MU_SMALL_BLOCKS = (MU_SMALL_ENTRIES / 1024 + 15) / 16;      // 32 x 32 blocks of X per wave

__host__ __device__ inline bool mu_small_apart(int mp, int np) { return 2 * (mp * np + mp * mp) <= MU_SMALL_ENTRIES; }

struct MuSteps {                                   // per iteration: the three products' scales
    int steps;
    MuScale gram[MDNVAE_MUON_MAX_STEPS], poly[MDNVAE_MUON_MAX_STEPS], step[MDNVAE_MUON_MAX_STEPS];
};

// acc = 32 rows x 32 columns over K (even) k steps: operand rows at `rows` (read along a row, or, TR, down the columns of X
// whose tile rows are `pitch` bytes apart), the next step's operands on their way while this one's are multiplied
template <bool TR>
__device__ __forceinline__ void mu_small_product(const char* rows, const char* cols, int K, long pitch, const MuLane& ln, int tr_extra,
                                                 mu_acc& acc) {
    mu_h8 r[2][2], c[2][2];
    auto load = [&](int set, int ks) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            c[set][s] = *reinterpret_cast<const mu_h8*>(cols + ks * MU_STEP + s * MU_FRAG + ln.direct);
            if constexpr (TR) r[set][s] = mu_tr(rows + (ks >> 1) * pitch + (ks & 1) * 512 + s * MU_FRAG + tr_extra + ln.tr);
            else r[set][s] = *reinterpret_cast<const mu_h8*>(rows + ks * MU_STEP + s * MU_FRAG + ln.direct);
        }
    };
    auto multiply = [&](int set) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(r[set][1], c[set][0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(r[set][0], c[set][1], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(r[set][0], c[set][0], acc, 0, 0, 0);
    };
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] = 0.0f;
    load(0, 0);
    for (int ks = 0; ks < K; ks += 2) {
        load(1, ks + 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(0);
        if (ks + 2 < K) load(0, ks + 2);
        __builtin_amdgcn_sched_barrier(0);
        multiply(1);
    }
}

// BL: blocks of X per wave, NT: most threads
template <int N, typename T, int BL, int NT>
__global__ __launch_bounds__(NT) void mu_small_kernel(MuTab<N> tab, MuPtrs<N> ptrs, MuMom mm, float eps, float x_scale, MuSteps st,
                                                               float decay, int is_step) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    __shared__ double red[MU_SMALL_NT / 64];
    const MuEntry entry = mu_entry(tab, blockIdx.x);
    const MuGeo& ge = entry.ge;
    const int e = entry.e;
    const int m_valid = ge.m, n_valid = ge.n, trans = ge.trans;
    const long len = (long)m_valid * n_valid, mat = blockIdx.x - entry.first;
    const T* g = static_cast<const T*>(mu_pick(ptrs.g, e)) + mat * len;
    float* mom = mu_pick(ptrs.mom, e);
    T* out = static_cast<T*>(mu_pick(ptrs.p, e)) + mat * len;
    const int NS = ge.np >> 4, KS = ge.mp >> 4, MB = ge.mp >> 5, NB = ge.np >> 5;
    const int x_bytes = 4 * ge.mp * ge.np, a_bytes = 4 * ge.mp * ge.mp;
    const bool apart = mu_small_apart(ge.mp, ge.np);
    char* X = smem;                                         // and, apart, Y, A, B behind it
    char* Y = apart ? X + x_bytes : X;
    char* A = Y + x_bytes;
    char* B = apart ? A + a_bytes : A;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, nt = blockDim.x, waves = nt >> 6;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const MuLane ln = mu_lane(lane);

    {   // G (momentum) in, eight columns of a row per chunk; every load is issued whether its entry exists or not (entry 0
        // stands in).  Until the norm is known a chunk waits as eight floats in the 32 bytes its two parts will have.
        const int per_row = ge.np >> 3, chunks = ge.mp * per_row;
        auto place = [&](int r, int c8) { return X + ((r >> 5) * NS + (c8 >> 1)) * MU_STEP + mu_at(r & 31, c8 & 1); };
        const float m0 = mom ? mm.mu * mom[0] + (float)g[0] : 0.0f;
        double s = 0.0;
#pragma unroll 1
        for (int ch = tid; ch < chunks; ch += nt) {
            const int r = ch / per_row, c8 = ch - r * per_row;
            int at[8];                                      // within the matrix: fits an int
            float u[8], m[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int c = c8 * 8 + k;
                at[k] = r < m_valid && c < n_valid ? (trans ? c * m_valid + r : r * n_valid + c) : -1;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = (float)g[max(at[k], 0)];
            if (mom) {
#pragma unroll
                for (int k = 0; k < 8; ++k) m[k] = mom[max(at[k], 0)];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    m[k] = mm.mu * m[k] + u[k];
                    u[k] = mm.nesterov ? u[k] + mm.mu * m[k] : m[k];
                    if (at[k] > 0) mom[at[k]] = m[k];       // entry 0: once everybody has read it
                }
            }
            mu_f4 lo4, hi4;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (at[k] < 0) u[k] = 0.0f;
                s += (double)u[k] * (double)u[k];
                if (k < 4) lo4[k] = u[k];
                else hi4[k - 4] = u[k];
            }
            *reinterpret_cast<mu_f4*>(place(r, c8)) = lo4;
            *reinterpret_cast<mu_f4*>(place(r, c8) + MU_FRAG) = hi4;
        }
        s = wave_sum(s);
        if (lane == 0) red[wid] = s;
        __syncthreads();
        if (mom && tid == 0) mom[0] = m0;
        s = 0.0;
        for (int i = 0; i < waves; ++i) s += red[i];
        const MuNorm normal(s, eps, x_scale);
        for (int ch = tid; ch < chunks; ch += nt) {         // the thread's own chunks
            const int r = ch / per_row, c8 = ch - r * per_row;
            char* dst = place(r, c8);
            const mu_f4 lo4 = *reinterpret_cast<const mu_f4*>(dst), hi4 = *reinterpret_cast<const mu_f4*>(dst + MU_FRAG);
            mu_h8 hi, lo;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                _Float16 a, b;
                mu_parts(normal(k < 4 ? lo4[k & 3] : hi4[k & 3]), a, b);
                hi[k] = a;
                lo[k] = b;
            }
            *reinterpret_cast<mu_h8*>(dst) = hi;
            *reinterpret_cast<mu_h8*>(dst + MU_FRAG) = lo;
        }
        __syncthreads();
    }

    auto put = [&](char* at, const mu_acc& v, int q) {
        const float four[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        mu_put<2>(at, four);
    };
    const int rb = wid / MB, cb = wid - rb * MB;
    const bool mine = wid < MB * MB;                        // at most 16 blocks of A: one per wave
    // the two n steps of a block of X are MU_STEP apart here, not 512 bytes
    const int tr_extra = ((lane >> 4) & 1) * (MU_STEP - 512);
    // the scales of all iterations, one per lane: a memory access less in every phase
    const int sl = min(lane, st.steps - 1);
    const float gram_acc = st.gram[sl].f_acc, poly_acc = st.poly[sl].f_acc, poly_add = st.poly[sl].f_add, step_acc = st.step[sl].f_acc,
                step_add = st.step[sl].f_add;
    mu_acc x;
    if constexpr (BL == 1) {
        if (wid < MB * NB) {
            MuOld old;
            mu_load_block<2>(old, X, wid % MB, NS, wid / MB * 32, lane);
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = mu_old<2>(old, k >> 2, k & 3);
        }
    }
    auto at_step = [](float v, int it) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), it)); };
    for (int it = 0; it < st.steps; ++it) {
        // A = X X^T
        mu_acc acc;
        if (mine) {
            mu_small_product<false>(X + rb * NS * MU_STEP, X + cb * NS * MU_STEP, NS, 0, ln, 0, acc);
            const float f = at_step(gram_acc, it);
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[k] *= f;
#pragma unroll
            for (int q = 0; q < 4; ++q) put(A + mu_block_at(cb, KS, rb * 32, q, lane), acc, q);
        }
        __syncthreads();
        // B = b A + c A^2
        if (mine) {
            const mu_acc kept = acc;                        // the wave's block of A is still in its registers
            mu_small_product<false>(A + rb * KS * MU_STEP, A + cb * KS * MU_STEP, KS, 0, ln, 0, acc);
            const float f = at_step(poly_acc, it), f_add = at_step(poly_add, it);
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[k] = acc[k] * f + kept[k] * f_add;
        }
        if (!apart) __syncthreads();
        if (mine) {
#pragma unroll
            for (int q = 0; q < 4; ++q) put(B + mu_block_at(cb, KS, rb * 32, q, lane), acc, q);
        }
        __syncthreads();
        // X <- a X + B X
        mu_acc y[BL];
#pragma unroll
        for (int b = 0; b < BL; ++b) {
            const int id = wid + b * waves;
            if (id < MB * NB) {
                const int nb = id / MB, mb = id - nb * MB;
                mu_small_product<true>(X + nb * 2 * MU_STEP, B + mb * KS * MU_STEP, KS, (long)NS * MU_STEP, ln, tr_extra, y[b]);
            }
            __builtin_amdgcn_sched_barrier(0);              // a block's operands in registers at a time
        }
        if (!apart) __syncthreads();
        const bool last = it + 1 == st.steps;
        const float f = at_step(step_acc, it), f_add = at_step(step_add, it);
#pragma unroll
        for (int b = 0; b < BL; ++b) {
            const int id = wid + b * waves;
            if (id < MB * NB) {
                const int nb = id / MB, mb = id - nb * MB;
                if constexpr (BL == 1) {                    // one block: the wave still has its X
#pragma unroll
                    for (int k = 0; k < 16; ++k) y[b][k] = x[k] = y[b][k] * f + x[k] * f_add;
                } else {
                    MuOld old;
                    mu_load_block<2>(old, X, mb, NS, nb * 32, lane);
#pragma unroll
                    for (int k = 0; k < 16; ++k) y[b][k] = y[b][k] * f + mu_old<2>(old, k >> 2, k & 3) * f_add;
                }
                if (!last) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) put(Y + mu_block_at(mb, NS, nb * 32, q, lane), y[b], q);
                } else {
                    const int m = mb * 32 + (lane & 31), n = nb * 32 + 4 * h;
                    const int left = m < m_valid ? n_valid - n : 0;                 // columns from n on that exist
                    const int step = trans ? m_valid : 1;
                    T* dst = out + (trans ? n * m_valid + m : m * n_valid + n);
                    const float lr_scale = ptrs.lr_scale[e];
                    T p[16];
                    if (is_step) {
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const int c = 8 * (k >> 2) + (k & 3);
                            p[k] = c < left ? dst[c * step] : (T)0.0f;
                        }
#pragma unroll
                        for (int k = 0; k < 16; ++k) y[b][k] = decay * (float)p[k] - lr_scale * y[b][k];
                    }
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const int c = 8 * (k >> 2) + (k & 3);
                        if (c < left) dst[c * step] = (T)y[b][k];
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        char* const swap = X;
        X = Y;
        Y = swap;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
struct MuCoef { int steps; float a, b, c, eps; };

// Power-of-two scales of the iterates.  s_k bounds the singular values of X_k: s_0 = 1 and s_{k+1} is the largest
// |s (a + b s^2 + c s^4)| on [0, s_k] (its ends and the roots of the derivative).  Entries of X are at most s_k,
// those of A at most s_k^2, those of B at most the largest |b t + c t^2| on [0, s_k^2]; a factor of two is kept for rounding.
// Returns false where one of A, B or the next X passes 256 (X itself 16, then): the iteration would leave what two fp16 parts
// hold.  Below the bounds the parts are exact to 2^-40 of them, so a matrix whose norm is far below eps, which X_0 keeps, has that much
// fewer bits.
static bool mu_scales(const MuCoef& co, MuSteps& st, float& x0_scale) {
    const double a = co.a, b = co.b, c = co.c;
    double s = 1.0;
    st.steps = co.steps;
    // the least bound is far below what coefficients that shrink X come to (0.1, 0, 0 in sixteen steps: 1e-16), so that X stays in
    // the middle of fp16's range with them too; the factors below stay inside fp32
    auto scale = [](double bound) { return std::exp2(std::floor(std::log2(32768.0 / std::max(bound, 1e-36)))); };
    double sx = scale(s);
    x0_scale = (float)sx;
    for (int k = 0; k < co.steps; ++k) {
        const double top = s * s;
        double pb = std::fabs(b * top + c * top * top), next = std::fabs(s * (a + b * top + c * top * top));
        if (c != 0.0) {
            const double t = -b / (2 * c);
            if (t > 0 && t < top) pb = std::max(pb, std::fabs(b * t + c * t * t));
        }
        double roots[2];
        int nr = 0;
        if (c != 0.0) {
            const double d = 9 * b * b - 20 * a * c;
            if (d >= 0) {
                roots[nr++] = (-3 * b + std::sqrt(d)) / (10 * c);
                roots[nr++] = (-3 * b - std::sqrt(d)) / (10 * c);
            }
        } else if (b != 0.0) {
            roots[nr++] = -a / (3 * b);
        }
        for (int i = 0; i < nr; ++i)
            if (roots[i] > 0 && roots[i] < top) {
                const double r = std::sqrt(roots[i]);
                next = std::max(next, std::fabs(r * (a + b * roots[i] + c * roots[i] * roots[i])));
            }
        if (!(top <= 256 && pb <= 256 && next <= 256)) return false;
        const double sa = scale(top), sb = scale(pb), sn = scale(next);
        const bool last = k + 1 == co.steps;
        st.gram[k] = {(float)(sa / (sx * sx)), 0.0f};
        st.poly[k] = {(float)(c * sb / (sa * sa)), (float)(b * sb / sa)};
        st.step[k] = {(float)((last ? 1.0 : sn) / (sb * sx)), (float)(a * (last ? 1.0 : sn) / sx)};
        sx = sn;
        s = next;
    }
    return true;
}

struct MuJob {                                   // one shape: `count` matrices behind one pointer each
    long rows, cols, count;
    void* p;
    const void* g;
    float* mom;
    float lr_scale;
};

static long mu_up(long v, long t) { return (v + t - 1) / t * t; }
constexpr int MU_CUS = 256;
// A launch's extent in work-items has 32 bits, and one that passes them is not refused but runs short: what is left out stays
// unwritten (2^24 + 3 matrices of 1 x 1, 256 threads each).
constexpr long MU_GRID = (1L << 24) - 8;         // workgroups of 256 threads, rounded up to eight
constexpr long MU_GRID_SMALL = (1L << 22) - 1;   // of up to 1024

// Whether each matrix goes to one workgroup: X and A have to fit, and X is a block per wave, or there are matrices for all CUs.  With
// more blocks one workgroup takes longer over them than the tiled launches do (64 x 544 87 and 78 us, an optimizer step over
// twenty 133 and 94), but a batch does not (300 of 32 x 1184 209 and 310 us).
static bool mu_small(const MuJob& j) {
    const long m = mu_up(std::min(j.rows, j.cols), 32), n = mu_up(std::max(j.rows, j.cols), 32);
    return m <= 128 && n <= MU_SMALL_ENTRIES && m * n + m * m <= MU_SMALL_ENTRIES &&
           (m * n <= 32 * 32 * (MU_SMALL_NT / 64) || j.count >= MU_CUS);
}

constexpr int MU_SPLITS[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32};     // of X X^T that a plan tries
constexpr long MU_PASS_BYTES = 1L << 30;         // workspace beyond which a batch is run in several passes
constexpr long MU_MAX_SIDE = 65536, MU_MAX_LONG = 1L << 24, MU_MAX_ENTRIES = 1L << 36;

static bool mu_shape_ok(long rows, long cols) {
    const long m = std::min(rows, cols), n = std::max(rows, cols);
    return m >= 1 && m <= MU_MAX_SIDE && n <= MU_MAX_LONG && m * n <= MU_MAX_ENTRIES;
}

// The matrices of one pass that take the tiled kernels: at most MU_MAX shapes.
struct MuPlan {
    int tile, tile_poly, tile_step, n;
    MuGeo geo[MU_MAX];
    long norm_blocks, bytes;
};

// What a launch of `wgs` workgroups takes (us, without what both tiles share), if the longest of them has `ks` k steps.  One workgroup per
// CU is bound by its own chain of loads, reads and products; where more share a CU their products add up, and the fullest CU
// decides.  A 128 x 128 tile is four times the work of 64 x 64 for two to three times the time of a step, but starts and ends
// more slowly and leaves CUs idle sooner.  The numbers are a fit to products of 160 x 1000 to 4 x 1024 x 2048, each tile and 1 to
// 12 splits measured.  With 64 and with 128 (five iterations, fp32): 160 x 1000 112 and 127 us, 1000 x 1000 200 and 209, 1024 x 4624
// 440 and 435, 4 x 1024 x 2048 681 and 628, 2000 x 2000 759 and 687.
static double mu_cost(double wgs, double ks, int tile, int terms) {
    const double n = wgs / MU_CUS, whole = n > 4 ? n + 0.5 : std::ceil(n);       // from the fifth on they even out
    if (tile == 64) return terms == 3 ? ks * std::max(0.13, 0.125 * whole) : ks * std::max(0.11, 0.07 * whole);
    const double full = std::ceil(n);
    if (terms == 3) return 3.0 + ks * (n <= 1 ? 0.22 + 0.12 * n : 0.30 * full);
    return 2.4 + ks * (n <= 1 ? 0.13 + 0.07 * n : 0.137 * full);
}

static void mu_plan(const MuJob* jobs, int n, int terms, MuPlan& pl) {
    double best = 0.0;
    long best_per = 0;
    for (int tile = 64; tile <= 128; tile += 64) {
        // X X^T: `per` k steps per workgroup at most; a split costs a launch more, and its shares are written and read again
        double gram = 0.0, square[2], step[2], rows[MU_MAX], ks[MU_MAX], tri[MU_MAX], longest = 0.0, per = 0.0;
        for (int i = 0; i < n; ++i) {
            rows[i] = (double)mu_up(std::min(jobs[i].rows, jobs[i].cols), tile);
            ks[i] = (double)(mu_up(std::max(jobs[i].rows, jobs[i].cols), tile) / 16);
            tri[i] = (double)jobs[i].count * (double)mu_tri((int)rows[i] / tile);
            longest = std::max(longest, ks[i]);
        }
        for (const int splits : MU_SPLITS) {
            const double target = std::ceil(longest / splits), inverse = 1.0 / target;
            double work = 0.0, shares = 0.0;
            for (int i = 0; i < n; ++i) {
                work += tri[i] * ks[i];
                if (ks[i] > target) shares += tri[i] * std::ceil(ks[i] * inverse);
            }
            const double t = mu_cost(work * inverse, target, tile, terms) + (splits > 1 ? 4.5 + shares * tile * tile * 8 / 6.0e6 : 0.0);
            if (splits == 1 || t < gram) gram = t, per = target;
        }
        // A^2 and B X: 64 x 64 tiles of matrices padded to 128 may be the faster ones
        for (int k = 0; k < 2; ++k) {
            const int tk = k ? 128 : 64;
            double most = 1.0, p = 0.0, q = 0.0;
            for (int i = 0; i < n; ++i) {
                const double k_steps = rows[i] / 16, tiles = rows[i] / tk, work = (double)jobs[i].count * tiles * k_steps;
                most = std::max(most, k_steps);
                p += work * (tiles + 1) / 2;
                q += work * (ks[i] * 16 / tk);
            }
            square[k] = mu_cost(p / most, most, tk, terms);
            step[k] = mu_cost(q / most, most, tk, terms);
        }
        const int poly128 = tile == 128 && square[1] <= square[0], step128 = tile == 128 && step[1] <= step[0];
        const double cost = gram + square[poly128] + step[step128];
        if (tile == 64 || cost < best) {
            best = cost;
            best_per = (long)per;
            pl.tile = tile;
            pl.tile_poly = poly128 ? 128 : 64;
            pl.tile_step = step128 ? 128 : 64;
        }
    }
    const int tile = pl.tile;
    pl.n = n;
    for (int i = 0; i < n; ++i) {
        MuGeo& g = pl.geo[i];
        g.m = (int)std::min(jobs[i].rows, jobs[i].cols);
        g.n = (int)std::max(jobs[i].rows, jobs[i].cols);
        g.mp = (int)mu_up(g.m, tile);
        g.np = (int)mu_up(g.n, tile);
        g.tile = tile;
        g.trans = jobs[i].rows > jobs[i].cols;
        g.count = (int)jobs[i].count;
    }
    pl.norm_blocks = 0;
    for (int i = 0; i < n; ++i) {
        MuGeo& g = pl.geo[i];
        const long ks = g.np / 16;
        const long s = (ks + best_per - 1) / best_per;
        g.kper = (int)((ks + s - 1) / s);
        g.splits = (int)((ks + g.kper - 1) / g.kper);
        pl.norm_blocks += jobs[i].count * (((long)g.m * g.n + MU_NORM_BLOCK - 1) / MU_NORM_BLOCK);
    }
    pl.bytes = mu_up(pl.norm_blocks * 8, 1024);
    for (int i = 0; i < n; ++i) {
        pl.geo[i].off = pl.bytes;
        pl.bytes += jobs[i].count * mu_matrix_bytes(pl.geo[i]);
    }
}

struct MuRun {                                   // what the launches of a call share
    MuCoef co;
    MuSteps st;
    float x0_scale, decay;
    MuMom mm;
    int is_step;
    hipStream_t stream;
};

template <int N>
static void mu_pointers(const MuJob* jobs, int n, MuPtrs<N>& pt) {
    for (int i = 0; i < N; ++i) {
        pt.p[i] = i < n ? jobs[i].p : nullptr;
        pt.g[i] = i < n ? jobs[i].g : nullptr;
        pt.mom[i] = i < n ? jobs[i].mom : nullptr;
        pt.lr_scale[i] = i < n ? jobs[i].lr_scale : 0.0f;
    }
}

// first workgroup of each entry, and their number (0: more than a grid holds)
template <int N, typename F>
static int mu_starts(const MuPlan& pl, int (&start)[N], F per_matrix) {
    long at = 0;
    for (int i = 0; i < N; ++i) {
        start[i] = i < pl.n ? (int)at : INT_MAX;
        if (i < pl.n) at += pl.geo[i].count * per_matrix(pl.geo[i]);
        if (at > MU_GRID) return 0;
    }
    return (int)at;
}

template <int N, typename T>
static int mu_run_small(const MuJob* jobs, int n, const MuRun& r) {
    MuTab<N> tab;
    MuPtrs<N> pt;
    mu_pointers(jobs, n, pt);
    long at = 0, most = 0, blocks = 4;
    for (int i = 0; i <= N; ++i) tab.start[i] = INT_MAX;
    for (int i = 0; i < n; ++i) {
        MuGeo& g = tab.e[i];
        g.off = 0;
        g.m = (int)std::min(jobs[i].rows, jobs[i].cols);
        g.n = (int)std::max(jobs[i].rows, jobs[i].cols);
        g.mp = (int)mu_up(g.m, 32);
        g.np = (int)mu_up(g.n, 32);
        g.trans = jobs[i].rows > jobs[i].cols;
        g.tile = 32;
        g.splits = g.kper = 1;
        g.count = (int)jobs[i].count;
        tab.start[i] = (int)at;
        at += jobs[i].count;
        most = std::max(most, (mu_small_apart(g.mp, g.np) ? 8L : 4L) * g.mp * (g.np + g.mp));
        blocks = std::max(blocks, (long)(g.mp / 32) * (g.np / 32));
        MV_REQUIRE(at <= MU_GRID_SMALL, E_SHAPE, "mdnvae_orthogonalize: too many matrices for one launch");
    }
    // up to twelve blocks of X (96 x 128) leave a wave half as many registers again (68 x 68: 28 us; 32 with the 128 registers
    // that sixteen waves have)
    auto kern = blocks <= 12 ? mu_small_kernel<N, T, 1, 768>
                : blocks <= MU_SMALL_NT / 64 ? mu_small_kernel<N, T, 1, MU_SMALL_NT> : mu_small_kernel<N, T, MU_SMALL_BLOCKS, MU_SMALL_NT>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             4 * MU_SMALL_ENTRIES);
    MV_REQUIRE(e == hipSuccess, (int)e, "mu_small_kernel: cannot raise the LDS limit: %s", hipGetErrorString(e));
    hipLaunchKernelGGL(kern, dim3((unsigned)at), dim3((unsigned)std::min((long)MU_SMALL_NT, blocks * 64)), (size_t)most, r.stream, tab, pt,
                       r.mm, r.co.eps, r.x0_scale, r.st, r.decay, r.is_step);
    MV_LAUNCH_CHECK("mu_small_kernel");
    return 0;
}

template <int TILE, int TERMS>
constexpr size_t mu_lds() {
    constexpr size_t lds = (size_t)MU_RING * 2 * (TILE / 32) * (TERMS == 3 ? 2 : 1) * MU_FRAG;
    static_assert(lds <= 160 * 1024 && lds >= 4 * 4224, "the ring fits LDS and holds the epilogues' blocks");
    return lds;
}
static int mu_allow_lds(const void* kernel, size_t lds) {
    const hipError_t e = lds > 64 * 1024 ? hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) : hipSuccess;
    MV_REQUIRE(e == hipSuccess, (int)e, "muon: cannot raise the LDS limit: %s", hipGetErrorString(e));
    return 0;
}
static dim3 mu_grid(int n) { return dim3((unsigned)((n + 7) / 8 * 8)); }      // whole rounds of the eight XCDs

template <int N, int TILE, int TERMS, int MODE>
static int mu_launch_sym(const MuTab<N>& tab, int n, char* ws, int ping, const MuScale& sc, hipStream_t st) {
    auto kern = mu_sym_kernel<N, TILE, TERMS, MODE>;
    constexpr size_t lds = mu_lds<TILE, TERMS>();
    if (const int rc = mu_allow_lds(reinterpret_cast<const void*>(kern), lds)) return rc;
    hipLaunchKernelGGL(kern, mu_grid(n), dim3(256), lds, st, tab, n, ws, ping, sc);
    MV_LAUNCH_CHECK("mu_sym_kernel");
    return 0;
}
template <int N, typename T, int TILE, int TERMS, bool LAST>
static int mu_launch_step(const MuTab<N>& tab, int n, const MuPtrs<N>& pt, char* ws, int ping, const MuScale& sc, const MuRun& r) {
    auto kern = mu_step_kernel<N, T, TILE, TERMS, LAST>;
    constexpr size_t lds = mu_lds<TILE, TERMS>();
    if (const int rc = mu_allow_lds(reinterpret_cast<const void*>(kern), lds)) return rc;
    hipLaunchKernelGGL(kern, mu_grid(n), dim3(256), lds, r.stream, tab, n, pt, ws, ping, sc, r.decay, r.is_step);
    MV_LAUNCH_CHECK("mu_step_kernel");
    return 0;
}

template <int N, typename T, int TERMS>
static int mu_run_tiled(const MuJob* jobs, const MuPlan& pl, const MuRun& r, char* ws) {
    MuPtrs<N> pt;
    mu_pointers(jobs, pl.n, pt);
    MuTab<N> tab;
    for (int i = 0; i < N; ++i) tab.e[i] = pl.geo[i < pl.n ? i : 0];
    MuStarts<N> norm;
    const int n_norm = mu_starts(pl, norm.s, [](const MuGeo& g) { return ((long)g.m * g.n + MU_NORM_BLOCK - 1) / MU_NORM_BLOCK; });
    MuTab<N> tnorm = tab, tsplit = tab, tgram = tab, treduce = tab, tpoly = tab, tstep = tab;
    for (int i = 0; i <= N; ++i) tnorm.start[i] = norm.s[i];
    const int n_split = mu_starts(pl, tsplit.start, [](const MuGeo& g) { return (long)(g.mp / 32) * (g.np / 64); });
    const int n_gram = mu_starts(pl, tgram.start, [](const MuGeo& g) { return mu_tri(g.mp / g.tile) * g.splits; });
    const int n_reduce = mu_starts(pl, treduce.start, [](const MuGeo& g) { return mu_tri(g.mp / g.tile); });
    const int n_poly = mu_starts(pl, tpoly.start, [&](const MuGeo& g) { return mu_tri(g.mp / pl.tile_poly); });
    const int n_step = mu_starts(pl, tstep.start, [&](const MuGeo& g) { return (long)(g.mp / pl.tile_step) * (g.np / pl.tile_step); });
    MV_REQUIRE(n_norm && n_split && n_gram && n_reduce && n_poly && n_step, E_SHAPE, "mdnvae_orthogonalize: too many tiles for one launch");
    bool split = false;
    for (int i = 0; i < pl.n; ++i) split = split || pl.geo[i].splits > 1;
    double* partial = reinterpret_cast<double*>(ws);
    hipLaunchKernelGGL((mu_norm_kernel<N, T>), dim3(n_norm), dim3(256), 0, r.stream, tnorm, pt, r.mm, partial);
    MV_LAUNCH_CHECK("mu_norm_kernel");
    hipLaunchKernelGGL((mu_split_kernel<N, T>), dim3(n_split), dim3(256), 0, r.stream, tsplit, norm, pt, r.mm, r.co.eps, r.x0_scale,
                       (const double*)partial, ws);
    MV_LAUNCH_CHECK("mu_split_kernel");
    for (int it = 0; it < r.st.steps; ++it) {
        const int ping = it & 1;
        const bool last = it + 1 == r.st.steps;
        int rc = pl.tile == 128 ? mu_launch_sym<N, 128, TERMS, MU_GRAM>(tgram, n_gram, ws, ping, r.st.gram[it], r.stream)
                                : mu_launch_sym<N, 64, TERMS, MU_GRAM>(tgram, n_gram, ws, ping, r.st.gram[it], r.stream);
        if (rc) return rc;
        if (split) {
            if (pl.tile == 128)
                hipLaunchKernelGGL((mu_reduce_kernel<N, 128, TERMS>), dim3(n_reduce * 4), dim3(256), 0, r.stream, treduce, ws, r.st.gram[it]);
            else
                hipLaunchKernelGGL((mu_reduce_kernel<N, 64, TERMS>), dim3(n_reduce), dim3(256), 0, r.stream, treduce, ws, r.st.gram[it]);
            MV_LAUNCH_CHECK("mu_reduce_kernel");
        }
        rc = pl.tile_poly == 128 ? mu_launch_sym<N, 128, TERMS, MU_POLY>(tpoly, n_poly, ws, ping, r.st.poly[it], r.stream)
                                 : mu_launch_sym<N, 64, TERMS, MU_POLY>(tpoly, n_poly, ws, ping, r.st.poly[it], r.stream);
        if (rc) return rc;
        if (pl.tile_step == 128)
            rc = last ? mu_launch_step<N, T, 128, TERMS, true>(tstep, n_step, pt, ws, ping, r.st.step[it], r)
                      : mu_launch_step<N, T, 128, TERMS, false>(tstep, n_step, pt, ws, ping, r.st.step[it], r);
        else
            rc = last ? mu_launch_step<N, T, 64, TERMS, true>(tstep, n_step, pt, ws, ping, r.st.step[it], r)
                      : mu_launch_step<N, T, 64, TERMS, false>(tstep, n_step, pt, ws, ping, r.st.step[it], r);
        if (rc) return rc;
    }
    return 0;
}

template <typename T, int TERMS>
static int mu_run(const MuJob* jobs, int n, bool small, const MuRun& r, char* ws) {
    if (n == 0) return 0;
    if (small) return n == 1 ? mu_run_small<1, T>(jobs, n, r) : mu_run_small<MU_MAX, T>(jobs, n, r);
    MuPlan pl;
    mu_plan(jobs, n, TERMS, pl);
    return n == 1 ? mu_run_tiled<1, T, TERMS>(jobs, pl, r, ws) : mu_run_tiled<MU_MAX, T, TERMS>(jobs, pl, r, ws);
}
static int mu_dispatch(const MuJob* jobs, int n, bool small, int dtype, int terms, const MuRun& r, char* ws) {
    if (dtype == MDNVAE_F32)
        return terms == 3 ? mu_run<float, 3>(jobs, n, small, r, ws) : mu_run<float, 1>(jobs, n, small, r, ws);
    return terms == 3 ? mu_run<__bf16, 3>(jobs, n, small, r, ws) : mu_run<__bf16, 1>(jobs, n, small, r, ws);
}

// matrices of a batch that go through one pass
static long mu_batch_per_pass(long batch, long rows, long cols, int terms) {
    MuJob j = {rows, cols, batch, nullptr, nullptr, nullptr, 0.0f};
    if (mu_small(j)) return std::min(batch, MU_GRID_SMALL);
    if (batch == 1) return batch;
    j.count = 1;
    MuPlan pl;
    mu_plan(&j, 1, terms, pl);                    // what one matrix takes alone: more splits than in company, if anything
    return std::max(1L, std::min(batch, MU_PASS_BYTES / std::max(1L, pl.bytes)));
}

static int mu_check(const char* who, int dtype, int terms, int steps, float a, float b, float c, float eps, MuRun& r) {
    MV_REQUIRE(dtype == MDNVAE_F32 || dtype == MDNVAE_BF16, E_ARG, "%s: unknown element type %d", who, dtype);
    MV_REQUIRE(terms == 1 || terms == 3, E_ARG, "%s: products have 1 or 3 terms (got %d)", who, terms);
    MV_REQUIRE(steps >= 1 && steps <= MDNVAE_MUON_MAX_STEPS, E_ARG, "%s: steps = %d outside [1, %d]", who, steps, MDNVAE_MUON_MAX_STEPS);
    MV_REQUIRE(eps > 0.0f && std::isfinite(eps), E_ARG, "%s: eps must be positive and finite", who);
    MV_REQUIRE(std::isfinite(a) && std::isfinite(b) && std::isfinite(c), E_ARG, "%s: coefficients must be finite", who);
    r.co = {steps, a, b, c, eps};
    MV_REQUIRE(mu_scales(r.co, r.st, r.x0_scale), E_ARG,
               "%s: with these coefficients the iteration may leave [-256, 256] (singular values start in [0, 1])", who);
    return 0;
}

}  // namespace mdnvae
using namespace mdnvae;

extern "C" size_t mdnvae_orthogonalize_workspace_bytes(long batch, long rows, long cols) {
    if (batch < 1 || !mu_shape_ok(rows, cols)) return 0;
    MuJob j = {rows, cols, batch, nullptr, nullptr, nullptr, 0.0f};
    if (mu_small(j)) return 0;
    MuPlan pl;
    long bytes = 0;
    for (int terms = 1; terms <= 3; terms += 2) {
        const long per = mu_batch_per_pass(batch, rows, cols, terms);
        for (const long count : {per, batch % per}) {                    // the last pass plans for itself
            if (!count) continue;
            j.count = count;
            mu_plan(&j, 1, terms, pl);
            bytes = std::max(bytes, pl.bytes);
        }
    }
    return (size_t)bytes;
}

extern "C" int mdnvae_orthogonalize(const void* x, void* out, long batch, long rows, long cols, int dtype, int steps, float a, float b,
                                    float c, float eps, int terms, void* workspace, size_t workspace_bytes, void* stream) {
    MV_REQUIRE(batch >= 0 && rows >= 0 && cols >= 0, E_ARG, "mdnvae_orthogonalize: negative size");
    MuRun r = {};
    const int bad = mu_check("mdnvae_orthogonalize", dtype, terms, steps, a, b, c, eps, r);
    if (bad) return bad;
    if (batch == 0 || rows == 0 || cols == 0) return 0;
    MV_REQUIRE(mu_shape_ok(rows, cols) && batch <= (1L << 30), E_SHAPE,
               "mdnvae_orthogonalize: %ld x [%ld, %ld] is larger than the kernels index", batch, rows, cols);
    MV_REQUIRE(x && out, E_ARG, "mdnvae_orthogonalize: null pointer");
    const uintptr_t from = reinterpret_cast<uintptr_t>(x), to = reinterpret_cast<uintptr_t>(out);
    const uintptr_t length = (uintptr_t)batch * (uintptr_t)rows * (uintptr_t)cols * (dtype == MDNVAE_F32 ? 4 : 2);
    MV_REQUIRE(from == to || from + length <= to || to + length <= from, E_ARG, "mdnvae_orthogonalize: out overlaps x (it may only be x itself)");
    const size_t need = mdnvae_orthogonalize_workspace_bytes(batch, rows, cols);
    MV_REQUIRE(workspace_bytes >= need && (workspace || need == 0), E_ARG, "mdnvae_orthogonalize: workspace of %zu bytes, %zu are needed",
               workspace_bytes, need);
    MV_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, E_ALIGN, "mdnvae_orthogonalize: workspace must be 256-byte aligned");
    r.stream = (hipStream_t)stream;
    r.decay = 0.0f;
    r.is_step = 0;
    const long per = mu_batch_per_pass(batch, rows, cols, terms), size = dtype == MDNVAE_F32 ? 4 : 2;
    const bool small = mu_small(MuJob{rows, cols, batch, nullptr, nullptr, nullptr, 0.0f});     // of all passes, as the workspace is
    for (long at = 0; at < batch; at += per) {
        MuJob j = {rows, cols, std::min(per, batch - at), static_cast<char*>(out) + at * rows * cols * size,
                   static_cast<const char*>(x) + at * rows * cols * size, nullptr, 0.0f};
        const int rc = mu_dispatch(&j, 1, small, dtype, terms, r, static_cast<char*>(workspace));
        if (rc) return rc;
    }
    return 0;
}

// The matrices of a step in order, `f(jobs, index, n, small)` for each group of up to MU_MAX that is launched together; stops at
// the first result that is not 0.  Matrices that fit one workgroup are a group of their own, unless there are others, one group
// holds all and the plan for it takes 64 x 64 tiles: then their tiles cost the launches of the others less than a launch of
// their own (a convolutional encoder's list of 192 x 1728 and smaller ones 191 -> 177 us in both types, of half and a quarter of
// its widths 177 -> 134 and 140 -> 102).  A 128 x 128 tile is too much
// for them (the gated mixture's 1077 -> 1095 us).  With one term per product they stay apart: a workgroup of their own keeps both
// parts, and what else is in the list must not take them away.
template <typename F>
static int mu_groups(const long* rows, const long* cols, int count, int terms, F f) {
    MuJob every[MU_MAX];
    int tiled = 0, all = 0;
    for (int i = 0; i < count; ++i) {
        if (rows[i] == 0 || cols[i] == 0) continue;
        const MuJob j = {rows[i], cols[i], 1, nullptr, nullptr, nullptr, 0.0f};
        tiled += !mu_small(j);
        if (all < MU_MAX) every[all] = j;
        ++all;
    }
    bool together = false;
    if (terms == 3 && tiled > 0 && tiled < all && all <= MU_MAX) {
        MuPlan pl;
        mu_plan(every, all, terms, pl);
        together = pl.tile == 64;
    }
    for (int pass = 0; pass < 2; ++pass) {
        MuJob jobs[MU_MAX];
        int index[MU_MAX], n = 0;
        for (int i = 0; i < count; ++i) {
            if (rows[i] == 0 || cols[i] == 0) continue;
            MuJob j = {rows[i], cols[i], 1, nullptr, nullptr, nullptr, 0.0f};
            if ((!together && mu_small(j)) != (pass == 1)) continue;
            jobs[n] = j;
            index[n++] = i;
            if (n == MU_MAX) {
                const int rc = f(jobs, index, n, pass == 1);
                if (rc) return rc;
                n = 0;
            }
        }
        if (n) {
            const int rc = f(jobs, index, n, pass == 1);
            if (rc) return rc;
        }
    }
    return 0;
}

// Whether what a step writes (parameters, momenta) overlaps anything else it touches; -1 without memory for the check.
struct MuSpan { uintptr_t lo, hi; int written; };
static int mu_overlap(void* const* params, const void* const* grads, float* const* momenta, const long* rows, const long* cols, int count,
                      int size) {
    MuSpan* s = static_cast<MuSpan*>(std::malloc((size_t)count * 3 * sizeof(MuSpan)));
    if (!s) return -1;
    long n = 0;
    for (int i = 0; i < count; ++i) {
        const uintptr_t len = (uintptr_t)rows[i] * (uintptr_t)cols[i];
        if (!len) continue;
        const void* at[3] = {params[i], grads[i], momenta[i]};
        for (int k = 0; k < 3; ++k) {
            const uintptr_t lo = reinterpret_cast<uintptr_t>(at[k]);
            s[n++] = {lo, lo + len * (k == 2 ? 4 : size), k != 1};
        }
    }
    std::sort(s, s + n, [](const MuSpan& a, const MuSpan& b) { return a.lo < b.lo; });
    uintptr_t end = 0, end_written = 0;
    int bad = 0;
    for (long i = 0; i < n && !bad; ++i) {
        bad = s[i].lo < (s[i].written ? end : end_written);
        end = std::max(end, s[i].hi);
        if (s[i].written) end_written = std::max(end_written, s[i].hi);
    }
    std::free(s);
    return bad;
}

extern "C" size_t mdnvae_muon_workspace_bytes(const long* rows, const long* cols, int count) {
    if (count < 1 || !rows || !cols) return 0;
    for (int i = 0; i < count; ++i)
        if (rows[i] < 0 || cols[i] < 0 || (rows[i] > 0 && cols[i] > 0 && !mu_shape_ok(rows[i], cols[i]))) return 0;
    long most = 0;
    for (int terms = 1; terms <= 3; terms += 2)
        mu_groups(rows, cols, count, terms, [&](MuJob* jobs, const int*, int n, bool small) {
            if (!small) {
                MuPlan pl;
                mu_plan(jobs, n, terms, pl);
                most = std::max(most, pl.bytes);
            }
            return 0;
        });
    return (size_t)most;
}

extern "C" int mdnvae_muon_step(void* const* params, const void* const* grads, float* const* momenta, const long* rows, const long* cols,
                                int count, int dtype, float lr, float momentum, int nesterov, float weight_decay, int scale_mode,
                                int steps, float a, float b, float c, float eps, int terms, void* workspace, size_t workspace_bytes,
                                void* stream) {
    MV_REQUIRE(count >= 0, E_ARG, "mdnvae_muon_step: negative count");
    MuRun r = {};
    const int bad = mu_check("mdnvae_muon_step", dtype, terms, steps, a, b, c, eps, r);
    if (bad) return bad;
    MV_REQUIRE(std::isfinite(lr) && std::isfinite(weight_decay) && momentum >= 0.0f && momentum < 1.0f, E_ARG,
               "mdnvae_muon_step: lr and weight_decay must be finite, momentum in [0, 1)");
    MV_REQUIRE(scale_mode >= MDNVAE_MUON_SCALE_NONE && scale_mode <= MDNVAE_MUON_SCALE_RMS, E_ARG, "mdnvae_muon_step: unknown scale mode %d",
               scale_mode);
    if (count == 0) return 0;
    MV_REQUIRE(params && grads && momenta && rows && cols, E_ARG, "mdnvae_muon_step: null pointer");
    for (int i = 0; i < count; ++i) {
        MV_REQUIRE(rows[i] >= 0 && cols[i] >= 0, E_ARG, "mdnvae_muon_step: negative size of matrix %d", i);
        if (rows[i] == 0 || cols[i] == 0) continue;
        MV_REQUIRE(mu_shape_ok(rows[i], cols[i]), E_SHAPE, "mdnvae_muon_step: matrix %d [%ld, %ld] is larger than the kernels index", i, rows[i],
                   cols[i]);
        MV_REQUIRE(params[i] && grads[i] && momenta[i], E_ARG, "mdnvae_muon_step: null pointer of matrix %d", i);
    }
    const int overlap = mu_overlap(params, grads, momenta, rows, cols, count, dtype == MDNVAE_F32 ? 4 : 2);
    MV_REQUIRE(overlap >= 0, E_ARG, "mdnvae_muon_step: no host memory");
    MV_REQUIRE(overlap == 0, E_ARG, "mdnvae_muon_step: a parameter or momentum overlaps another tensor of the step (in the list twice?)");
    const size_t need = mdnvae_muon_workspace_bytes(rows, cols, count);
    MV_REQUIRE(workspace_bytes >= need && (workspace || need == 0), E_ARG, "mdnvae_muon_step: workspace of %zu bytes, %zu are needed",
               workspace_bytes, need);
    MV_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, E_ALIGN, "mdnvae_muon_step: workspace must be 256-byte aligned");
    r.stream = (hipStream_t)stream;
    r.decay = (float)(1.0 - (double)lr * (double)weight_decay);
    r.mm = {momentum, nesterov};
    r.is_step = 1;
    return mu_groups(rows, cols, count, terms, [&](MuJob* jobs, const int* index, int n, bool small) {
        for (int k = 0; k < n; ++k) {
            const int i = index[k];
            const double ro = (double)rows[i], co = (double)cols[i];
            const double s = scale_mode == MDNVAE_MUON_SCALE_SHAPE ? std::sqrt(std::max(1.0, ro / co))
                             : scale_mode == MDNVAE_MUON_SCALE_RMS ? 0.2 * std::sqrt(std::max(ro, co)) : 1.0;
            jobs[k].p = params[i];
            jobs[k].g = grads[i];
            jobs[k].mom = momenta[i];
            jobs[k].lr_scale = (float)((double)lr * s);
        }
        return mu_dispatch(jobs, n, small, dtype, terms, r, static_cast<char*>(workspace));
    });
}
