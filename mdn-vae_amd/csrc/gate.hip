// Balance loss of a gate: how evenly the rows of a batch spread over its experts (mixture components), with per-expert
// counts and the gradient.  The gate is that of the trait-gated mixture head (no counterpart in the reference).
//
//     p_t = softmax(l_t),  c_e = #{valid rows t : e among the top_k largest of l_t},  P_e = mean of p_te over the n valid rows
//     loss = E / (k n) sum_e c_e P_e           (1 where rows spread evenly, E / k ... E where they all agree)
//     dloss / dl_te = p_te (w_e - sum_j p_tj w_j),   w_e = E / (k n^2) (c_e - mean c)
//
// (counts carry no gradient; the mean is taken out of c in float64, where softmax gradients cancel it anyway.)  Ties go to
// the lowest index; an expert whose logit is -inf is masked out of that row (probability 0, never counted), and a
// row of nothing else is not valid; NaN counts as larger than every number.
//
// Two sweeps over the logits, since every gradient depends on the counts of all rows: statistics, then gradient.  A row
// belongs to a group of L lanes, eight (sixteen above 128 experts) values each; experts stay with their lane, so sums of
// p and counts are kept in registers over the rows of a wave.  Sums of p are fp32 over at most 32 rows of a lane and the groups
// of its wave; from there on float64, for equal rows round alike and their errors add up (512 rows of a lane: 6e-6).
// Selection: every lane sorts its keys once (a network of 19 or 63 exchanges), then k rounds of "largest head of the group, its
// lane moves on" find the k-th largest key; whoever is above it is taken, and of those equal to it as many of the lowest index
// as are missing (ballots; only where the group saw a tie).  Sixteen lanes of sixteen values rather than thirty-two of eight for 256
// experts: four rows per wave share each round, and all its exchanges stay within a DPP row (290 -> 95 us for 262144 rows,
// 2.8 TB/s: bound by its instructions, about 620 per four rows).
#include <algorithm>
#include "common.h"
#include "../../include/mdnvae_hip.h"

namespace mdnvae {

constexpr unsigned GT_NEG_INF = 0x007fffffu;      // key of -inf; 0 = no expert in this slot

template <int L, int NV, int VEC>
struct GateMap {                                  // slot v of lane l holds expert at(l, v)
    static __device__ __forceinline__ int at(int l, int v) { return ((v / VEC) * L + l) * VEC + v % VEC; }
};

// order-preserving key: -inf < ... < -0 = +0 < ... < +inf < NaN
__device__ __forceinline__ unsigned gt_key(float z) {
    if (z != z) return 0xffffffffu;
    const unsigned u = __float_as_uint(z + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// reductions over groups of L consecutive lanes; every lane gets the result
template <int CTRL>
__device__ __forceinline__ unsigned gt_dpp(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int L, typename F>
__device__ __forceinline__ unsigned gt_reduce(unsigned v, F f) {
    if constexpr (L >= 2) v = f(v, gt_dpp<0xB1>(v));       // quad_perm 1,0,3,2
    if constexpr (L >= 4) v = f(v, gt_dpp<0x4E>(v));       // quad_perm 2,3,0,1
    if constexpr (L >= 8) v = f(v, gt_dpp<0x141>(v));      // row_half_mirror: the other quad of eight
    if constexpr (L >= 16) v = f(v, gt_dpp<0x140>(v));     // row_mirror: the other eight of sixteen
    if constexpr (L >= 32) v = f(v, (unsigned)__shfl_xor((int)v, 16, 64));
    if constexpr (L >= 64) v = f(v, (unsigned)__shfl_xor((int)v, 32, 64));
    return v;
}
template <int L>
__device__ __forceinline__ unsigned gt_max(unsigned v) {
    return gt_reduce<L>(v, [](unsigned a, unsigned b) { return a > b ? a : b; });
}
template <int L>
__device__ __forceinline__ float gt_fmax(float v) {
    return __uint_as_float(gt_reduce<L>(__float_as_uint(v), [](unsigned a, unsigned b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <int L>
__device__ __forceinline__ float gt_sum(float v) {
    return __uint_as_float(gt_reduce<L>(__float_as_uint(v), [](unsigned a, unsigned b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

// exp(x), x <= 0 (or NaN, -inf): 2^t by the hardware with t = x log2 e rounded, and what the rounding left out as a first-order
// factor - a couple of 2^-24 for all x, at a third of the instructions of expf.  Below 2^-126 it gives zero: next to a row's largest,
// which is 1, that is no share of its sum
__device__ __forceinline__ float gt_exp(float x) {
    const float log2e = 1.44269504f, tail = 1.92596299e-8f, ln2 = 0.693147181f;
    const float y = fmaxf(x, -150.0f);                      // zero either way; keeps -inf out of the remainder (NaN: below)
    const float t = y * log2e;
    const float rest = fmaf(y, log2e, -t) + y * tail;
    const float p = __builtin_amdgcn_exp2f(t);
    return x != x ? x : fmaf(p, rest * ln2, p);
}

template <typename T, int L, int NV, int VEC>
__device__ __forceinline__ void gt_load(const T* row, int E, int l, bool in, float (&z)[NV]) {
    typedef T vec __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int j = 0; j < NV / VEC; ++j) {
        const int e = GateMap<L, NV, VEC>::at(l, j * VEC);
        if constexpr (VEC == 4) {
            vec v;
            const bool here = in && e < E;                 // E is a multiple of four
            if (here) v = *reinterpret_cast<const vec*>(row + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[j * 4 + i] = here ? (float)v[i] : -INFINITY;
        } else {
            z[j] = (in && e < E) ? (float)row[e] : -INFINITY;
        }
    }
}

// softmax of a row in place, m its largest logit; false (and zeros) where the row has no expert left
template <int L, int NV>
__device__ __forceinline__ bool gt_softmax_at(float (&z)[NV], float m) {
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        z[v] = gt_exp(z[v] - m);
        s += z[v];
    }
    s = gt_sum<L>(s);
    const float inv = 1.0f / s;
    const bool any = m != -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) z[v] = any ? z[v] * inv : 0.0f;
    return any;
}
template <int L, int NV>
__device__ __forceinline__ bool gt_softmax(float (&z)[NV]) {
    float m = z[0];
    bool nan = z[0] != z[0];
#pragma unroll
    for (int v = 1; v < NV; ++v) {
        m = fmaxf(m, z[v]);
        nan = nan || z[v] != z[v];
    }
    if (nan) m = INFINITY;                                  // a NaN shows in every probability of the row
    return gt_softmax_at<L, NV>(z, gt_fmax<L>(m));
}

__device__ __forceinline__ void gt_exchange(unsigned& a, unsigned& b) {    // a >= b afterwards
    const unsigned hi = a > b ? a : b, lo = a > b ? b : a;
    a = hi;
    b = lo;
}
// descending; odd-even merge network
template <int N>
__device__ __forceinline__ void gt_sort(unsigned (&s)[N]) {
#pragma unroll
    for (int p = 1; p < N; p <<= 1)
#pragma unroll
        for (int k = p; k >= 1; k >>= 1)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) gt_exchange(s[i + j], s[i + j + k]);
}

// top_k rounds on sorted lists of which the first D entries can matter; the lists' next heads
template <int L, int NV, int D>
__device__ __forceinline__ unsigned gt_rounds(const unsigned (&sorted)[NV], int top_k, int lane, unsigned& first, unsigned& t, int& need) {
    const int base = lane & ~(L - 1), l = lane & (L - 1);
    unsigned s[D];
#pragma unroll
    for (int v = 0; v < D; ++v) s[v] = sorted[v];
    for (int r = 0; r < top_k; ++r) {
        const unsigned m = gt_max<L>(s[0]);
        if (r == 0) first = m;
        need = m == t ? need + 1 : 1;
        t = m;
        const unsigned long long heads = __ballot(s[0] == m) >> base;     // bit 0: the group's first lane
        bool own;
        if constexpr (L == 64) own = l == __ffsll((long long)heads) - 1;
        else own = l == __ffs((int)(unsigned)(heads & ((1ull << (L & 63)) - 1ull))) - 1;
        const unsigned move = own ? ~0u : 0u;               // as a mask: "own ? s[v + 1] : s[v]" becomes an indexed register read
#pragma unroll
        for (int v = 0; v + 1 < D; ++v) s[v] = (s[v + 1] & move) | (s[v] & ~move);
        s[D - 1] &= ~move;
    }
    return s[0];
}

// Which slots of the row are among its top_k: those with key >= the result (keys that lose a tie are cleared).  largest: the
// row's largest logit (+inf where it holds a NaN).
template <int L, int NV, int VEC>
__device__ __forceinline__ unsigned gt_select(const float (&z)[NV], int top_k, unsigned (&key)[NV], float& largest) {
    unsigned s[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) s[v] = key[v] = gt_key(z[v]);
    const int lane = threadIdx.x & 63, base = lane & ~(L - 1);
    const unsigned long long group = (L == 64 ? ~0ull : ((1ull << (L & 63)) - 1ull)) << base;
    unsigned t = 0, first = 0;
    int need = 0;
    bool tie;
    if (top_k == 1) {
#pragma unroll
        for (int v = 1; v < NV; ++v) s[0] = s[0] > s[v] ? s[0] : s[v];
        first = t = gt_max<L>(s[0]);
        need = 1;
        int same = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) same += key[v] == t ? 1 : 0;
        tie = same > 1 || __popcll(__ballot(same > 0) & group) > 1;
    } else {
        gt_sort<NV>(s);
        // a lane gives at most top_k entries, and the one after them is looked at for ties
        const unsigned next = NV > 9 && top_k < 9 ? gt_rounds<L, NV, NV < 9 ? NV : 9>(s, top_k, lane, first, t, need)
                                                  : gt_rounds<L, NV, NV>(s, top_k, lane, first, t, need);
        tie = next == t;
    }
    largest = first == 0xffffffffu ? INFINITY : __uint_as_float((first >> 31) ? first & 0x7fffffffu : ~first);
    const unsigned floor_key = t > GT_NEG_INF ? t : GT_NEG_INF + 1;       // nothing at or below -inf is ever taken
    if (__ballot(tie && t > GT_NEG_INF)) {
        // among the keys equal to t the lowest `need` indices stay: experts are ordered by (chunk, lane, place in the chunk)
        const unsigned long long below = group & ((1ull << lane) - 1ull);
        int before = 0;
#pragma unroll
        for (int j = 0; j < NV / VEC; ++j) {
            int lower = 0, all = 0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const unsigned long long eq = __ballot(key[j * VEC + i] == t) & group;
                lower += __popcll(eq & below);
                all += __popcll(eq);
            }
            int at = before + lower;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (key[j * VEC + i] == t) {
                    if (at >= need) key[j * VEC + i] = 0u;
                    ++at;
                }
            before += all;
        }
    }
    return floor_key;
}

struct GateArgs {
    const void* logits;
    const unsigned char* valid;       // null: every row
    long T;
    int E, top_k;
};

// rows [first, T) in steps of `stride` of this group: its lanes' sums of p, counts, and the number of valid rows.  The trip
// count is that of the whole wave (ballots), rows past the end count as padding.  flush(): takes the sums of p and sets them to
// zero, after every GT_FLUSH rows of a lane.
constexpr int GT_FLUSH = 32;
template <typename T, int L, int NV, int VEC, typename FLUSH>
__device__ __forceinline__ void gt_stats(const GateArgs& a, long wave_first, long stride, float (&ps)[NV], int (&cn)[NV], int& rows,
                                         FLUSH flush) {
    const int lane = threadIdx.x & 63, l = lane & (L - 1), gr = lane / L;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        ps[v] = 0.0f;
        cn[v] = 0;
    }
    rows = 0;
    const T* logits = static_cast<const T*>(a.logits);
    float z[NV], next[NV];
    auto fetch = [&](long r0, float (&d)[NV]) {
        const long r = r0 + gr;
        const bool in = r < a.T && (!a.valid || a.valid[r] != 0);
        gt_load<T, L, NV, VEC>(logits + (in ? r : 0) * a.E, a.E, l, in, d);
    };
    if (wave_first < a.T) fetch(wave_first, z);
    int held = 0;
    for (long r0 = wave_first; r0 < a.T; r0 += stride) {
        if (r0 + stride < a.T) fetch(r0 + stride, next);           // under this row's arithmetic
        unsigned key[NV];
        float largest;
        const unsigned floor_key = gt_select<L, NV, VEC>(z, a.top_k, key, largest);
        rows += gt_softmax_at<L, NV>(z, largest) ? 1 : 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            ps[v] += z[v];
            cn[v] += key[v] >= floor_key ? 1 : 0;
            z[v] = next[v];
        }
        if (++held == GT_FLUSH) {
            flush();
            held = 0;
        }
    }
}

// sums over the groups of a wave
template <int L, int NV, typename N>
__device__ __forceinline__ void gt_wave_total(N (&s)[NV]) {
#pragma unroll
    for (int o = L; o < 64; o <<= 1)
#pragma unroll
        for (int v = 0; v < NV; ++v) s[v] += __shfl_xor(s[v], o, 64);
}
template <int L>
__device__ __forceinline__ int gt_wave_total(int rows) {
#pragma unroll
    for (int o = L; o < 64; o <<= 1) rows += __shfl_xor(rows, o, 64);
    return rows;
}

// gradient of the same rows; w: the lane's weights
template <typename T, int L, int NV, int VEC>
__device__ __forceinline__ void gt_grads(const GateArgs& a, long wave_first, long stride, const float (&w)[NV], T* grad) {
    typedef T vec __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63, l = lane & (L - 1), gr = lane / L;
    const T* logits = static_cast<const T*>(a.logits);
    for (long r0 = wave_first; r0 < a.T; r0 += stride) {
        const long r = r0 + gr;
        const bool in = r < a.T, live = in && (!a.valid || a.valid[r] != 0);
        float z[NV];
        gt_load<T, L, NV, VEC>(logits + (live ? r : 0) * a.E, a.E, l, live, z);
        const bool any = gt_softmax<L, NV>(z);
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) dot += z[v] * w[v];
        dot = gt_sum<L>(dot);
        if (!in) continue;
        T* out = grad + r * a.E;
#pragma unroll
        for (int j = 0; j < NV / VEC; ++j) {
            const int e = GateMap<L, NV, VEC>::at(l, j * VEC);
            if (e >= a.E) continue;
            float g[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) g[i] = any ? z[j * VEC + i] * (w[j * VEC + i] - dot) : 0.0f;
            if constexpr (VEC == 4) {
                vec o;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = (T)g[i];
                *reinterpret_cast<vec*>(out + e) = o;
            } else {
                out[e] = (T)g[0];
            }
        }
    }
}

// weight of one expert in the gradient: upstream gradients g_loss (null: 1) of the loss and g_mean (null: 0) of P
__device__ __forceinline__ float gt_weight(int count, double count_mean, int n, int E, int top_k, float g_loss, float g_mean) {
    if (n == 0) return 0.0f;
    const double per = 1.0 / (double)n;
    return (float)((double)g_loss * ((double)E / (double)top_k) * per * per * ((double)count - count_mean) + (double)g_mean * per);
}

constexpr int GT_NT = 256;

// sweep 1: one partial row of sums and counts per workgroup.  Four waves per SIMD, one for each workgroup that a CU gets; with
// thirty-two lanes per row that would take spills of 12 to 120 registers, and three it is.
template <typename T, int L, int NV, int VEC>
__global__ __launch_bounds__(GT_NT, L == 32 ? 3 : 4) void gate_stats_kernel(GateArgs a, float* __restrict__ part_p, int* __restrict__ part_c,
                                                           int* __restrict__ part_n) {
    __shared__ union {                                     // one after the other
        double sums[GT_NT / 64][L * NV];
        int counts[GT_NT / 64][L * NV];
    } table;
    auto& sp = table.sums;
    auto& sc = table.counts;
    __shared__ int sn[GT_NT / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int G = 64 / L;
    float ps[NV];
    int cn[NV], rows;
    const long stride = (long)gridDim.x * (GT_NT / 64) * G;
    if (lane < L) {                                        // a lane's entries are its own until the barrier
#pragma unroll
        for (int v = 0; v < NV; ++v) sp[wave][GateMap<L, NV, VEC>::at(lane, v)] = 0.0;
    }
    auto flush = [&] {
        gt_wave_total<L, NV>(ps);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (lane < L) sp[wave][GateMap<L, NV, VEC>::at(lane, v)] += (double)ps[v];
            ps[v] = 0.0f;
        }
    };
    gt_stats<T, L, NV, VEC>(a, ((long)blockIdx.x * (GT_NT / 64) + wave) * G, stride, ps, cn, rows, flush);
    flush();
    gt_wave_total<L, NV>(cn);
    rows = gt_wave_total<L>(rows);
    if (lane == 0) sn[wave] = rows;
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += GT_NT)
        part_p[(long)blockIdx.x * a.E + e] = (float)((sp[0][e] + sp[1][e]) + (sp[2][e] + sp[3][e]));
    if (threadIdx.x == 0) part_n[blockIdx.x] = (sn[0] + sn[1]) + (sn[2] + sn[3]);
    __syncthreads();
    if (lane < L) {
#pragma unroll
        for (int v = 0; v < NV; ++v) sc[wave][GateMap<L, NV, VEC>::at(lane, v)] = cn[v];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += GT_NT)
        part_c[(long)blockIdx.x * a.E + e] = (sc[0][e] + sc[1][e]) + (sc[2][e] + sc[3][e]);
}

// the workgroups' rows summed: 16 experts per workgroup, 64 threads each, float64, fixed order
__global__ __launch_bounds__(1024) void gate_reduce_kernel(const float* __restrict__ part_p, const int* __restrict__ part_c,
                                                          const int* __restrict__ part_n, int nb, int E, int* __restrict__ counts,
                                                          float* __restrict__ mean_probs, int* __restrict__ n_valid) {
    __shared__ double sp[64][17];
    __shared__ int sc[64][17], sn[16];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4, e = blockIdx.x * 16 + x;
    int n = 0;
    for (int b = threadIdx.x; b < nb; b += 1024) n += part_n[b];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if ((threadIdx.x & 63) == 0) sn[threadIdx.x >> 6] = n;
    double p = 0.0;
    int c = 0;
    if (e < E) {
#pragma unroll 4
        for (int b = y; b < nb; b += 64) {
            p += (double)part_p[(long)b * E + e];
            c += part_c[(long)b * E + e];
        }
    }
    sp[y][x] = p;
    sc[y][x] = c;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) n += sn[i];
    if (y == 0 && e < E) {
        p = 0.0;
        c = 0;
#pragma unroll 16
        for (int i = 0; i < 64; ++i) {
            p += sp[i][x];
            c += sc[i][x];
        }
        counts[e] = c;
        mean_probs[e] = n > 0 ? (float)(p / (double)n) : 0.0f;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) n_valid[0] = n;
}

// loss from counts and means, by one wave (fixed order); also the mean count
__device__ __forceinline__ float gt_loss(const int* counts, const float* mean_probs, int n, int E, int top_k, double& count_mean) {
    const int lane = threadIdx.x & 63;
    double s = 0.0, c = 0.0;
    for (int e = lane; e < E; e += 64) {
        s += (double)counts[e] * (double)mean_probs[e];
        c += (double)counts[e];
    }
    s = wave_sum(s);
    c = wave_sum(c);
    s = __shfl(s, 0, 64);
    count_mean = __shfl(c, 0, 64) / (double)E;
    return n > 0 ? (float)(s * (double)E / ((double)top_k * (double)n)) : 0.0f;
}

__global__ __launch_bounds__(64) void gate_loss_kernel(const int* __restrict__ counts, const float* __restrict__ mean_probs,
                                                       const int* __restrict__ n_valid, int E, int top_k, float* __restrict__ loss) {
    double mean;
    const float v = gt_loss(counts, mean_probs, n_valid[0], E, top_k, mean);
    if (threadIdx.x == 0) loss[0] = v;
}

// few partial rows (nb E <= GT_SMALL_PARTIALS): every workgroup of the gradient sums them itself, in the same order, which saves
// the launch in between
constexpr int GT_SMALL_PARTIALS = 2048;
struct GatePartials { const float* p; const int* c; const int* n; int nb; };

// sweep 2.  Rows in the opposite order of sweep 1: what that read last is still in the cache behind the L2s.
// REDUCE: counts, mean_probs and n_valid come from the partial rows (and are written, by workgroup 0) instead of from memory.
template <typename T, int L, int NV, int VEC, bool REDUCE>
__global__ __launch_bounds__(GT_NT) void gate_grad_kernel(GateArgs a, GatePartials parts, int* __restrict__ counts,
                                                          float* __restrict__ mean_probs, int* __restrict__ n_valid,
                                                          const float* __restrict__ g_loss, const float* __restrict__ g_mean,
                                                          float* __restrict__ loss, T* __restrict__ grad) {
    constexpr int G = 64 / L;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & (L - 1);
    __shared__ int s_count[REDUCE ? L * NV : 1], s_n[REDUCE ? GT_NT / 64 : 1];
    __shared__ float s_mean[REDUCE ? L * NV : 1];
    const int* count = counts;
    const float* mean = mean_probs;
    int n;
    if constexpr (REDUCE) {
        n = 0;
        for (int b = threadIdx.x; b < parts.nb; b += GT_NT) n += parts.n[b];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
        if (lane == 0) s_n[wave] = n;
        __syncthreads();
        n = 0;
#pragma unroll
        for (int i = 0; i < GT_NT / 64; ++i) n += s_n[i];
        for (int e = wave; e < a.E; e += GT_NT / 64) {
            double p = 0.0;
            int c = 0;
            for (int b = lane; b < parts.nb; b += 64) {
                p += (double)parts.p[(long)b * a.E + e];
                c += parts.c[(long)b * a.E + e];
            }
            p = wave_sum(p);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
            if (lane == 0) {
                s_count[e] = c;
                s_mean[e] = n > 0 ? (float)(p / (double)n) : 0.0f;
                if (blockIdx.x == 0) {
                    counts[e] = c;
                    mean_probs[e] = s_mean[e];
                }
            }
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) n_valid[0] = n;
        __syncthreads();
        count = s_count;
        mean = s_mean;
    } else {
        n = n_valid[0];
    }
    double count_mean;
    const float value = gt_loss(count, mean, n, a.E, a.top_k, count_mean);
    if (loss && blockIdx.x == 0 && threadIdx.x == 0) loss[0] = value;
    const float gl = g_loss ? g_loss[0] : 1.0f;
    float w[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int e = GateMap<L, NV, VEC>::at(l, v);
        w[v] = e < a.E ? gt_weight(count[e], count_mean, n, a.E, a.top_k, gl, g_mean ? g_mean[e] : 0.0f) : 0.0f;
    }
    const long per = (long)gridDim.x * (GT_NT / 64) * G;
    const long mine = ((long)blockIdx.x * (GT_NT / 64) + wave) * G;
    const long sweeps = (a.T + per - 1) / per;
    for (long s = sweeps - 1; s >= 0; --s) {
        const long first = s * per + mine;
        if (first < a.T) gt_grads<T, L, NV, VEC>(a, first, a.T, w, grad);      // one group of rows
    }
}

// few rows: everything in one workgroup and one launch
constexpr int GT_ONE_NT = 1024;
template <typename T, int L, int NV, int VEC>
__global__ __launch_bounds__(GT_ONE_NT) void gate_one_kernel(GateArgs a, float* __restrict__ loss, int* __restrict__ counts,
                                                             float* __restrict__ mean_probs, int* __restrict__ n_valid,
                                                             T* __restrict__ grad) {
    constexpr int W = GT_ONE_NT / 64, G = 64 / L;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float (*sp)[L * NV] = reinterpret_cast<float (*)[L * NV]>(smem);
    int (*sc)[L * NV] = reinterpret_cast<int (*)[L * NV]>(smem + sizeof(float) * W * L * NV);
    __shared__ int sn[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & (L - 1);
    float ps[NV];
    int cn[NV], rows;
    gt_stats<T, L, NV, VEC>(a, (long)wave * G, (long)W * G, ps, cn, rows, [] {});      // eight rows of a lane at most: gt_one
    gt_wave_total<L, NV>(ps);
    gt_wave_total<L, NV>(cn);
    rows = gt_wave_total<L>(rows);
    if (lane < L) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            sp[wave][GateMap<L, NV, VEC>::at(lane, v)] = ps[v];
            sc[wave][GateMap<L, NV, VEC>::at(lane, v)] = cn[v];
        }
    }
    if (lane == 0) sn[wave] = rows;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) n += sn[i];
    float* mean = &sp[0][0];
    int* count = &sc[0][0];
    for (int e = threadIdx.x; e < a.E; e += GT_ONE_NT) {           // E <= 1024: one expert per thread
        double p = 0.0;
        int c = 0;
        for (int i = 0; i < W; ++i) {
            p += (double)sp[i][e];
            c += sc[i][e];
        }
        mean[e] = n > 0 ? (float)(p / (double)n) : 0.0f;           // row 0 of the table, read by this thread only so far
        count[e] = c;
        mean_probs[e] = mean[e];
        counts[e] = c;
    }
    __syncthreads();
    double count_mean;
    const float value = gt_loss(count, mean, n, a.E, a.top_k, count_mean);
    if (threadIdx.x == 0) {
        loss[0] = value;
        if (n_valid) n_valid[0] = n;
    }
    if (!grad) return;
    float w[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int e = GateMap<L, NV, VEC>::at(l, v);
        w[v] = e < a.E ? gt_weight(count[e], count_mean, n, a.E, a.top_k, 1.0f, 0.0f) : 0.0f;
    }
    gt_grads<T, L, NV, VEC>(a, (long)wave * G, (long)W * G, w, grad);
}

// ---- host --------------------------------------------------------------------------------------------------------------
constexpr int GT_BLOCKS = 1024;                  // workgroups of a sweep: four per CU
constexpr int GT_MAX_EXPERTS = 1024;

static int gt_lanes(int E) {                     // lanes per row: eight values each up to 128 experts, sixteen above
    int l = 1;
    while (l * (E > 128 ? 16 : 8) < E) l <<= 1;
    return l;
}
static int gt_blocks(long T, int E) {
    const long per = (long)(GT_NT / 64) * (64 / gt_lanes(E));
    return (int)std::max(1L, std::min((long)GT_BLOCKS, (T + per - 1) / per));
}
// one workgroup up to eight rows per group of lanes
static bool gt_one(long T, int E) { return T * gt_lanes(E) <= 8L * GT_ONE_NT; }

struct GateOut {
    float* loss;
    int* counts;
    float* mean_probs;
    int* n_valid;
    void* grad;
    const float *g_loss, *g_mean;
};
struct GateWork { float* p; int* c; int* n; };

template <typename T, int L, int NV, int VEC>
static int gt_run(const GateArgs& a, const GateWork& w, const GateOut& o, bool stats, hipStream_t st) {
    if (stats && gt_one(a.T, a.E)) {
        auto kern = gate_one_kernel<T, L, NV, VEC>;
        const size_t lds = (size_t)(GT_ONE_NT / 64) * L * NV * 8;
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        MV_REQUIRE(e == hipSuccess, (int)e, "gate_one_kernel: cannot raise the LDS limit: %s", hipGetErrorString(e));
        hipLaunchKernelGGL(kern, dim3(1), dim3(GT_ONE_NT), lds, st, a, o.loss, o.counts, o.mean_probs, o.n_valid, (T*)o.grad);
        MV_LAUNCH_CHECK("gate_one_kernel");
        return 0;
    }
    const int nb = gt_blocks(a.T, a.E);
    const GatePartials parts = {w.p, w.c, w.n, nb};
    if (stats) {
        hipLaunchKernelGGL((gate_stats_kernel<T, L, NV, VEC>), dim3(nb), dim3(GT_NT), 0, st, a, w.p, w.c, w.n);
        MV_LAUNCH_CHECK("gate_stats_kernel");
        if (o.grad && (long)nb * a.E <= GT_SMALL_PARTIALS) {
            hipLaunchKernelGGL((gate_grad_kernel<T, L, NV, VEC, true>), dim3(nb), dim3(GT_NT), 0, st, a, parts, o.counts, o.mean_probs,
                               o.n_valid, o.g_loss, o.g_mean, o.loss, (T*)o.grad);
            MV_LAUNCH_CHECK("gate_grad_kernel");
            return 0;
        }
        hipLaunchKernelGGL(gate_reduce_kernel, dim3((a.E + 15) / 16), dim3(1024), 0, st, (const float*)w.p, (const int*)w.c,
                           (const int*)w.n, nb, a.E, o.counts, o.mean_probs, o.n_valid);
        MV_LAUNCH_CHECK("gate_reduce_kernel");
        if (!o.grad) {
            hipLaunchKernelGGL(gate_loss_kernel, dim3(1), dim3(64), 0, st, (const int*)o.counts, (const float*)o.mean_probs,
                               (const int*)o.n_valid, a.E, a.top_k, o.loss);
            MV_LAUNCH_CHECK("gate_loss_kernel");
            return 0;
        }
    }
    hipLaunchKernelGGL((gate_grad_kernel<T, L, NV, VEC, false>), dim3(nb), dim3(GT_NT), 0, st, a, parts, o.counts, o.mean_probs, o.n_valid,
                       o.g_loss, o.g_mean, stats ? o.loss : nullptr, (T*)o.grad);
    MV_LAUNCH_CHECK("gate_grad_kernel");
    return 0;
}

template <typename T, int VEC>
static int gt_dispatch_lanes(const GateArgs& a, const GateWork& w, const GateOut& o, bool stats, hipStream_t st) {
    if (a.E > 128) {
        switch (gt_lanes(a.E)) {
            case 16: return gt_run<T, 16, 16, VEC>(a, w, o, stats, st);
            case 32: return gt_run<T, 32, 16, VEC>(a, w, o, stats, st);
            default: return gt_run<T, 64, 16, VEC>(a, w, o, stats, st);
        }
    }
    switch (gt_lanes(a.E)) {
        case 1: return gt_run<T, 1, 8, VEC>(a, w, o, stats, st);
        case 2: return gt_run<T, 2, 8, VEC>(a, w, o, stats, st);
        case 4: return gt_run<T, 4, 8, VEC>(a, w, o, stats, st);
        case 8: return gt_run<T, 8, 8, VEC>(a, w, o, stats, st);
        default: return gt_run<T, 16, 8, VEC>(a, w, o, stats, st);
    }
}
template <typename T>
static int gt_dispatch(const GateArgs& a, const GateWork& w, const GateOut& o, bool stats, hipStream_t st) {
    // four values per load where every row starts on a multiple of four elements
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(o.grad);
    if (a.E % 4 == 0 && at % (4 * sizeof(T)) == 0) return gt_dispatch_lanes<T, 4>(a, w, o, stats, st);
    return gt_dispatch_lanes<T, 1>(a, w, o, stats, st);
}

static int gt_check(const char* who, const void* logits, long T, int E, int top_k, int dtype) {
    MV_REQUIRE(dtype == MDNVAE_F32 || dtype == MDNVAE_BF16, E_ARG, "%s: unknown element type %d", who, dtype);
    MV_REQUIRE(T >= 0 && T <= 0x7fffffffL, E_ARG, "%s: %ld rows", who, T);
    MV_REQUIRE(E >= 1 && E <= GT_MAX_EXPERTS, E_SHAPE, "%s: %d experts outside [1, %d]", who, E, GT_MAX_EXPERTS);
    MV_REQUIRE(top_k >= 1 && top_k <= E, E_ARG, "%s: top_k = %d outside [1, %d experts]", who, top_k, E);
    MV_REQUIRE(logits || T == 0, E_ARG, "%s: null pointer", who);
    return 0;
}

}  // namespace mdnvae
using namespace mdnvae;

extern "C" size_t mdnvae_gate_balance_workspace_bytes(long T, int E) {
    if (T < 1 || E < 1 || E > GT_MAX_EXPERTS || gt_one(T, E)) return 0;
    return (size_t)gt_blocks(T, E) * ((size_t)E * 8 + 4) + 4;
}

extern "C" int mdnvae_gate_balance(const void* logits, const unsigned char* valid, long T, int E, int top_k, int dtype, void* workspace,
                                   size_t workspace_bytes, float* loss, int* counts, float* mean_probs, int* n_valid, void* grad,
                                   void* stream) {
    const int bad = gt_check("mdnvae_gate_balance", logits, T, E, top_k, dtype);
    if (bad) return bad;
    MV_REQUIRE(loss && counts && mean_probs, E_ARG, "mdnvae_gate_balance: null output");
    const size_t need = mdnvae_gate_balance_workspace_bytes(T, E);
    MV_REQUIRE(workspace_bytes >= need && (workspace || need == 0), E_ARG, "mdnvae_gate_balance: workspace of %zu bytes, %zu are needed",
               workspace_bytes, need);
    MV_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 3u) == 0, E_ALIGN, "mdnvae_gate_balance: workspace must be 4-byte aligned");
    const GateArgs a = {logits, valid, T, E, top_k};
    const size_t nb = need ? (size_t)gt_blocks(T, E) : 0;
    float* p = static_cast<float*>(workspace);
    const GateWork w = {p, reinterpret_cast<int*>(p + nb * E), reinterpret_cast<int*>(p + 2 * nb * E)};
    if (!n_valid && need) n_valid = reinterpret_cast<int*>(p + 2 * nb * E) + nb;
    const GateOut o = {loss, counts, mean_probs, n_valid, grad, nullptr, nullptr};
    return dtype == MDNVAE_F32 ? gt_dispatch<float>(a, w, o, true, (hipStream_t)stream)
                               : gt_dispatch<__bf16>(a, w, o, true, (hipStream_t)stream);
}

extern "C" int mdnvae_gate_balance_bwd(const void* logits, const unsigned char* valid, long T, int E, int top_k, int dtype,
                                       const int* counts, const float* mean_probs, const int* n_valid, const float* g_loss,
                                       const float* g_mean, void* grad, void* stream) {
    const int bad = gt_check("mdnvae_gate_balance_bwd", logits, T, E, top_k, dtype);
    if (bad) return bad;
    if (T == 0) return 0;
    MV_REQUIRE(counts && mean_probs && n_valid && grad, E_ARG, "mdnvae_gate_balance_bwd: null pointer");
    const GateArgs a = {logits, valid, T, E, top_k};
    const GateWork w = {nullptr, nullptr, nullptr};
    const GateOut o = {nullptr, const_cast<int*>(counts), const_cast<float*>(mean_probs), const_cast<int*>(n_valid), grad, g_loss, g_mean};
    return dtype == MDNVAE_F32 ? gt_dispatch<float>(a, w, o, false, (hipStream_t)stream)
                               : gt_dispatch<__bf16>(a, w, o, false, (hipStream_t)stream);
}
