// Group norm with an activation on channels-last maps, forward and backward.
//   x[N, S, C], G groups of Cg = C / G channels, M = S * Cg values per (sample, group):
//     h = (x - mean) * rstd      mean, biased variance over the group's S positions and Cg channels, rstd = 1 / sqrt(var + eps)
//     z = w h + b                y = act(z):  0 z,  1 z * sigmoid(z),  2 z > 0 ? z : slope * z
//   backward, dz = dy act'(z), A[n,c] = sum_s dz, B[n,c] = sum_s dz h:
//     db = sum_n A, dw = sum_n B, s1 = sum_{c in g} w A, s2 = sum_{c in g} w B, dx = rstd (w dz - (s1 + h s2) / M)
// Sums are in fp32, the joins of a group's parts and of the parameters' rows in fp64.  z and h are computed again in the backward pass from x and the
// two statistics of a group, by way of x - mean as in the forward pass: the rounding of mean * rstd in x * rstd - mean * rstd would be one of
// |mean| rstd 2^-24 in h, more than all else where the mean is far from zero.  B = rstd sum dz (x - mean).
//
// Memory bounds all of it: forward x is read and y written, backward x and dy are read and dx written.  A (sample, set of groups) that fits
// the registers of a workgroup is read once, in one launch (gn_slab_*).  A larger one is read twice: parts of a sample's positions give
// partial sums (gn_stats, gn_bwd_sums), a join gives the group's, and a second pass over the map writes the result (gn_apply, gn_bwd_dx).
// Figures below: one MI355X, medians of a kernel trace; a 1 GiB copy reads and writes 5.1 TB/s there, 128 MiB of cached data 8.5 TB/s.
#include "elem.h"

#define ACT_NONE 0
#define ACT_SILU 1
#define ACT_LRELU 2

struct GnArgs {
    const void *x, *dy, *w, *b;
    void *y, *dw, *db;
    float *mean, *rstd;
    long long xs, xr, ds, dr;   // strides of x and dy in elements: between samples, between positions (channels are adjacent)
    int N, S, C, G, Cg, ptype;
    float eps, slope;
};

template <int ACT>
__device__ __forceinline__ float act_fwd(float z, float slope) {
    if (ACT == ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
    if (ACT == ACT_LRELU) return z > 0.f ? z : z * slope;
    return z;
}
// dy * act'(z)
template <int ACT>
__device__ __forceinline__ float act_bwd(float dy, float z, float slope) {
    if (ACT == ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
        return dy * (s * (1.f + z * (1.f - s)));
    }
    if (ACT == ACT_LRELU) return z > 0.f ? dy : dy * slope;
    return dy;
}

// V parameters from channel c of C on, `none` where there are none
template <class E>
__device__ __forceinline__ void load_params(const void* p, int ptype, int c, int C, float none, float (&v)[E::V]) {
    constexpr int V = E::V;
    if (!p) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = none;
    } else if (c + V > C) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = c + k < C ? load_any(p, ptype, c + k) : none;
    } else if (ptype == AG2V_F32) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const u32x4 r = *reinterpret_cast<const u32x4_a4*>((const float*)p + c + k);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k + j] = __uint_as_float(r[j]);
        }
    } else {            // the maps' own type
        E::unpack(load_vec<E>((const typename E::T*)p + c, V), v);
    }
}
// mean and 1 / std of V channels from c on
template <int V>
__device__ __forceinline__ void load_stats(const GnArgs& a, int n, int c, float (&mean)[V], float (&rstd)[V], const float2* coef = nullptr,
                                           float2* cf = nullptr) {
    if (a.Cg % V == 0 && c % V == 0) {
        const int g = n * a.G + c / a.Cg;
        const float m = a.mean[g], r = a.rstd[g];
        const float2 f = coef ? coef[g] : make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            mean[k] = m;
            rstd[k] = r;
            if (coef) cf[k] = f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int g = n * a.G + min(c + k, a.C - 1) / a.Cg;
            mean[k] = a.mean[g];
            rstd[k] = a.rstd[g];
            if (coef) cf[k] = coef[g];
        }
    }
}

// ---------------------------------------------------------------- layout shared by the kernels
// Channels are walked as rows of 16-byte vectors.  `cols` vectors side by side -- a power of two, the ones beyond the slab or tile idle --
// and threads / cols rows at a time: thread t works on vector t % cols of row t / cols, t / cols + rows at a time, ...  Lanes of one wave
// that hold the same vector then meet by shuffles, and what a wave (or, with more than 64 vectors, a row of threads) is left with by LDS:
// rows[slot][cols * per], `slots` of them.
//
// x_j += the same x_j of the other lanes of the wave that hold the same vector
template <int K>
__device__ __forceinline__ void same_vector_sums(float (&x)[K], int cols) {
    for (int o = 32; o >= cols; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) x[k] += __shfl_xor(x[k], o, 64);
}
// out[g] = sum over the slots of group g's columns [g * wg, (g + 1) * wg): 2^llg lanes a group, `threads` lanes in all
__device__ __forceinline__ void share_sums(const float* rows, int slots, int width, int wg, int ng, int llg, int t, int threads, float* out) {
    const int l = t & ((1 << llg) - 1), step = 1 << llg;
    const int dr = step / wg, dc = step - dr * wg;
    for (int g = t >> llg; g < ng; g += threads >> llg) {
        int r = l / wg, c = l - r * wg;
        float s = 0.f;
        while (r < slots) {
            s += rows[r * width + g * wg + c];
            r += dr;
            c += dc;
            if (c >= wg) { c -= wg; ++r; }
        }
        for (int o = step >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (l == 0) out[g] = s;
    }
}
// log2 of the lanes a group gets of `threads`: at most a wave
static int share_lanes(int threads, int ng) {
    int l = 0;
    while (l < 6 && (2 << l) * ng <= threads) ++l;
    return l;
}
static int log2_up(long long v) {
    int l = 0;
    while ((1LL << l) < v) ++l;
    return l;
}

// ---------------------------------------------------------------- one launch: a slab's values stay in registers
// T threads own all S positions of kg adjacent groups of one sample, U vectors a thread, read once: mean, then the squared deviations from
// it, then the result.  blockDim / T slabs a workgroup.  ONE: a thread's vector touches one group (Cg a multiple of the vector, or kg = 1);
// otherwise sums and statistics are per channel.
// 6.0 us for 1 x 64 x 1024 bf16 and for 8 x 64 x 1024 fp32, of which an empty kernel's launch is 2 and the chain load - sum - squares - store
// the rest.  20 us for 8 x 4096 x 256 fp16 in 32 groups, two of them a slab: 1.6 TB/s, bound by its 128 workgroups, which leave half of the CUs without work.
struct GnSlab {
    int T, kg, nsets;                  // threads, groups, sets of groups a sample
    int lc, rows, slots, wg, llg;      // log2 of vectors a row, rows at a time, LDS slots, columns a group there, log2 of lanes a group
    long long nslab;
};

template <class E, int ACT, int U, bool ONE>
__global__ __launch_bounds__(1024) void gn_slab_fwd_kernel(GnArgs a, GnSlab p) {
    extern __shared__ float shm[];
    constexpr int V = E::V, NG = ONE ? 1 : V;        // groups a vector may touch
    const int sub = threadIdx.x / p.T, t = threadIdx.x - sub * p.T, subs = blockDim.x / p.T;
    const int cols = 1 << p.lc, width = cols * NG;
    float* rows = shm + sub * (p.slots * width + 2 * p.kg);
    float* stat = rows + p.slots * width;
    const long long slab = (long long)xcd_remap(blockIdx.x, gridDim.x) * subs + sub;
    const bool live = slab < p.nslab;
    const int n = live ? (int)(slab / p.nsets) : 0, g0 = live ? (int)(slab - (long long)n * p.nsets) * p.kg : 0;
    const int ng = min(p.kg, a.G - g0), c0 = g0 * a.Cg, W = ng * a.Cg;
    const int rs = t >> p.lc, col = t & (cols - 1);
    const bool on = live && col * V < W;
    const int at = W < V ? 0 : min(col * V, W - V), dup = col * V - at;      // (see GnWhere)
    const float inv = 1.f / ((float)a.S * (float)a.Cg);
    const typename E::T* x = (const typename E::T*)a.x + n * a.xs + c0 + at;
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = rs + u * p.rows;
        raw[u] = u32x4{0, 0, 0, 0};
        if (on && r < a.S) raw[u] = load_vec<E>(x + r * a.xr, W);
    }
    float w[V], b[V];
    load_params<E>(a.w, a.ptype, c0 + at, a.C, 1.f, w);
    load_params<E>(a.b, a.ptype, c0 + at, a.C, 0.f, b);
    // per-thread sums to rows[slot][...]
    const auto hand_over = [&](const float (&acc)[V]) {
        float s[NG];
        if (ONE) {
            s[0] = 0.f;
#pragma unroll
            for (int k = 0; k < V; ++k) s[0] += k >= dup && at + k < W ? acc[k] : 0.f;
        } else {
#pragma unroll
            for (int k = 0; k < NG; ++k) s[k] = acc[k];
        }
        same_vector_sums(s, cols);
        if (cols > 64 || (t & 63) < cols) {
            const int slot = cols > 64 ? rs : t >> 6;
#pragma unroll
            for (int k = 0; k < NG; ++k)
                if (ONE || k >= dup) rows[slot * width + (ONE ? col : at + k)] = s[k];
        }
    };
    float acc[V] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float v[V];
        E::unpack(raw[u], v);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += v[k];
    }
    hand_over(acc);
    __syncthreads();
    if (live) share_sums(rows, p.slots, width, p.wg, ng, p.llg, t, p.T, stat);
    __syncthreads();
    float mean[NG];
    int gi[NG];
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        gi[k] = min(ONE ? col / p.wg : (at + k) / a.Cg, ng - 1);
        mean[k] = on ? stat[gi[k]] * inv : 0.f;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.f;
    if (on) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (rs + u * p.rows < a.S) {
                float v[V];
                E::unpack(raw[u], v);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float d = v[k] - mean[k % NG];
                    acc[k] = fmaf(d, d, acc[k]);
                }
            }
    }
    hand_over(acc);
    __syncthreads();
    if (live) share_sums(rows, p.slots, width, p.wg, ng, p.llg, t, p.T, stat + p.kg);
    __syncthreads();
    if (live)
        for (int g = t; g < ng; g += p.T) {
            a.mean[n * a.G + g0 + g] = stat[g] * inv;
            a.rstd[n * a.G + g0 + g] = 1.f / sqrtf(stat[p.kg + g] * inv + a.eps);
        }
    if (!on) return;
    float rstd[NG];
#pragma unroll
    for (int k = 0; k < NG; ++k) rstd[k] = 1.f / sqrtf(stat[p.kg + gi[k]] * inv + a.eps);
#pragma unroll
    for (int k = 0; k < V; ++k) w[k] *= rstd[k % NG];
    typename E::T* y = (typename E::T*)a.y + (long long)n * a.S * a.C + c0 + at;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = rs + u * p.rows;
        if (r < a.S) {
            float v[V];
            E::unpack(raw[u], v);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = act_fwd<ACT>(fmaf(v[k] - mean[k % NG], w[k], b[k]), a.slope);
            store_tail<E>(y + (long long)r * a.C, dup, W, v);
        }
    }
}

// Backward on slabs: x and dy of a slab in registers.  A workgroup keeps its set of groups and walks samples, `walkers` apart, so that the
// parameters' gradients leave it once: ab[walker][C] = (sum dz, sum dz h) over its samples.  Without ONE the statistics are per channel and
// take up to 256 registers a thread; with ONE the bound of 1024 threads keeps them to 128, so that two workgroups of 512 fit a CU (64 x 1024 x 256
// bf16: 58 us with 128 and 82 with 136).  7 to 9 us for 8 x 64 x 1024 fp32 (medians of runs), bound by the chain of loads and joins.
template <class E, int ACT, int U, bool ONE>
__global__ __launch_bounds__(ONE ? 1024 : 512) void gn_slab_bwd_kernel(GnArgs a, GnSlab p, int walkers, float2* ab) {
    extern __shared__ float shm[];
    constexpr int V = E::V, NG = ONE ? 1 : V;
    const int sub = threadIdx.x / p.T, t = threadIdx.x - sub * p.T, subs = blockDim.x / p.T;
    const int cols = 1 << p.lc, width = cols * V, gwidth = cols * NG;
    // two arrays of group sums while walking, one of channel sums at the end
    const int area = p.slots * (ONE ? width : 2 * width);
    float* r1 = shm + sub * (area + 2 * p.kg);
    float* r2 = r1 + p.slots * gwidth;
    float* stat = r1 + area;
    const int blk = xcd_remap(blockIdx.x, gridDim.x), set = blk % p.nsets, walker = blk / p.nsets * subs + sub;
    const int g0 = set * p.kg, ng = min(p.kg, a.G - g0), c0 = g0 * a.Cg, W = ng * a.Cg;
    const int rs = t >> p.lc, col = t & (cols - 1);
    const bool on = col * V < W, writes = cols > 64 || (t & 63) < cols;
    const int at = W < V ? 0 : min(col * V, W - V), dup = col * V - at;      // (see GnWhere)
    const int slot = cols > 64 ? rs : t >> 6;
    const float inv = 1.f / ((float)a.S * (float)a.Cg);
    float w[V], b[V], A[V], B[V];
    int gi[NG];
#pragma unroll
    for (int k = 0; k < NG; ++k) gi[k] = min(ONE ? col / p.wg : (at + k) / a.Cg, ng - 1);
    load_params<E>(a.w, a.ptype, c0 + at, a.C, 1.f, w);
    load_params<E>(a.b, a.ptype, c0 + at, a.C, 0.f, b);
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = B[k] = 0.f;
    for (int n0 = blk / p.nsets * subs; n0 < a.N; n0 += walkers) {
        const int n = n0 + sub;
        const bool live = n < a.N, here = on && live;
        u32x4 rx[U], rd[U];
        const typename E::T* x = (const typename E::T*)a.x + (long long)n * a.xs + c0 + at;
        const typename E::T* dy = (const typename E::T*)a.dy + (long long)n * a.ds + c0 + at;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = rs + u * p.rows;
            rx[u] = rd[u] = u32x4{0, 0, 0, 0};
            if (here && r < a.S) {
                rx[u] = load_vec<E>(x + r * a.xr, W);
                rd[u] = load_vec<E>(dy + r * a.dr, W);
            }
        }
        float mean[NG], rstd[NG], sA[V] = {}, sB[V] = {}, g1[NG] = {}, g2[NG] = {};      // sums of dz, dz h; of w dz, w dz h
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            rstd[k] = here ? a.rstd[(long long)n * a.G + g0 + gi[k]] : 0.f;
            mean[k] = here ? a.mean[(long long)n * a.G + g0 + gi[k]] : 0.f;
        }
        if (here) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (rs + u * p.rows < a.S) {
                    float v[V], d[V];
                    E::unpack(rx[u], v);
                    E::unpack(rd[u], d);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float e = v[k] - mean[k % NG], dz = act_bwd<ACT>(d[k], fmaf(e, w[k] * rstd[k % NG], b[k]), a.slope);
                        sA[k] += dz;
                        sB[k] = fmaf(dz, e, sB[k]);
                    }
                }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                sB[k] *= rstd[k % NG];
                A[k] += sA[k];
                B[k] += sB[k];
                if (k >= dup && at + k < W) {      // (w and b behind W are the next group's)
                    g1[k % NG] = fmaf(w[k], sA[k], g1[k % NG]);
                    g2[k % NG] = fmaf(w[k], sB[k], g2[k % NG]);
                }
            }
        }
        if (a.y) {
            same_vector_sums(g1, cols);
            same_vector_sums(g2, cols);
            if (writes) {
#pragma unroll
                for (int k = 0; k < NG; ++k)
                    if (ONE || k >= dup) {
                        r1[slot * gwidth + (ONE ? col : at + k)] = g1[k];
                        r2[slot * gwidth + (ONE ? col : at + k)] = g2[k];
                    }
            }
            __syncthreads();
            if (live) {
                share_sums(r1, p.slots, gwidth, p.wg, ng, p.llg, t, p.T, stat);
                share_sums(r2, p.slots, gwidth, p.wg, ng, p.llg, t, p.T, stat + p.kg);
            }
            __syncthreads();
        }
        if (here && a.y) {
            typename E::T* dx = (typename E::T*)a.y + (long long)n * a.S * a.C + c0 + at;
            // (the values above are computed again: kept, they would not fit the registers)
#pragma unroll
            for (int u = 0; u < U; ++u) asm volatile("" : "+v"(rx[u]), "+v"(rd[u]));
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                g1[k] = stat[gi[k]] * inv * rstd[k];
                g2[k] = stat[p.kg + gi[k]] * inv * rstd[k];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = rs + u * p.rows;
                if (r < a.S) {
                    float v[V], d[V];
                    E::unpack(rx[u], v);
                    E::unpack(rd[u], d);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float e = v[k] - mean[k % NG], wr = w[k] * rstd[k % NG], dz = act_bwd<ACT>(d[k], fmaf(e, wr, b[k]), a.slope);
                        v[k] = fmaf(-(e * rstd[k % NG]), g2[k % NG], fmaf(dz, wr, -g1[k % NG]));
                    }
                    store_tail<E>(dx + (long long)r * a.C, dup, W, v);
                }
            }
        }
    }
    if (!ab) return;
    // the channels' sums over the workgroup's rows, one array at a time in all of the rows' memory
    same_vector_sums(A, cols);
    same_vector_sums(B, cols);
    for (int half = 0; half < 2; ++half) {
        __syncthreads();
        if (writes) {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (k >= dup) r1[slot * width + at + k] = half ? B[k] : A[k];
        }
        __syncthreads();
        for (int c = t; c < W; c += p.T) {
            float s = 0.f;
            for (int r = 0; r < p.slots; ++r) s += r1[r * width + c];
            (&ab[(long long)walker * a.C + c0 + c].x)[half] = s;
        }
    }
}

// ---------------------------------------------------------------- larger maps: sums of parts, a join, a second pass over the map
// A workgroup owns `len` positions of one sample and a tile of 2^lc vectors of channels.
struct GnParts {
    int tiles, lc, rows, slots, len, P, tg, llg;    // P: parts a sample; tg: tiles a group may touch
};
// The last vector of a row whose width is no multiple of the vector moves back to end with the row, so every load is 16 bytes wide; the `dup`
// elements it shares with the vector before are left out of the sums and the stores.
struct GnWhere {
    int tile, n, q, rs, c0, W, c, dup, lo, hi;      // c: first channel of the thread's vector
    bool on;
};
template <int V>
__device__ __forceinline__ GnWhere where_of(const GnArgs& a, const GnParts& p, int blk) {
    GnWhere i;
    // rows of neighbouring tiles share cache lines: tiles of a part, and neighbouring parts, run on one XCD
    blk = xcd_remap(blk, p.tiles * p.P * a.N);
    i.tile = blk % p.tiles;
    const int np = blk / p.tiles;
    i.n = np / p.P;
    i.q = np - i.n * p.P;
    i.rs = threadIdx.x >> p.lc;
    i.c0 = (i.tile * V) << p.lc;
    i.W = min(V << p.lc, a.C - i.c0);
    const int c = i.c0 + (threadIdx.x & ((1 << p.lc) - 1)) * V;
    i.on = c < a.C;
    i.c = a.C < V ? 0 : min(c, a.C - V);
    i.dup = c - i.c;
    i.lo = i.q * p.len;
    i.hi = min(a.S, i.lo + p.len);
    return i;
}

// Statistics of a part.  A thread sums deviations from the first value it sees of each channel: that value is one of the summed ones, so the
// sum of squares about it is at most (count + 1) times the one about the thread's mean, and nothing cancels that matters, whatever the mean.
// Threads, waves and channels then join pairwise as (count, mean, squares about the mean).
// part[n][g][q * tg + (tile - the group's first tile)] = (count, mean, squares, 0)
// 134 MB (16 x 65536 x 64 bf16) in 34 us, 4.0 TB/s; the joins at the end of every 32 KB are what keeps it below the copy's rate.
template <class E>
__global__ __launch_bounds__(256) void gn_stats_kernel(GnArgs a, GnParts p, float4* part) {
    constexpr int V = E::V, U = 8;
    __shared__ float sm[4 * 64 * V], sq[4 * 64 * V], sn[4];      // [slot][width]
    const GnWhere i = where_of<V>(a, p, blockIdx.x);
    const int cols = 1 << p.lc, width = cols * V;
    const typename E::T* x = (const typename E::T*)a.x + i.n * a.xs + i.c;
    float mean[V] = {}, s[V] = {}, m[V] = {};
    int count = 0;
    if (i.on && i.lo + i.rs < i.hi) {
        for (int r = i.lo + i.rs; r < i.hi; r += U * p.rows) {
            u32x4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * p.rows < i.hi) raw[u] = load_vec<E>(x + (long long)(r + u * p.rows) * a.xr, a.C);
            if (count == 0) E::unpack(raw[0], mean);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * p.rows < i.hi) {
                    float v[V];
                    E::unpack(raw[u], v);
                    ++count;
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float d = v[k] - mean[k];
                        s[k] += d;
                        m[k] = fmaf(d, d, m[k]);
                    }
                }
        }
        const float rc = 1.f / (float)count;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float ds = s[k] * rc, q = fmaf(-s[k], ds, m[k]);
            mean[k] += ds;
            m[k] = q < 0.f ? 0.f : q;
        }
    }
    // lanes with the same vector
    float nn = (float)max(0, (i.hi - i.lo - i.rs + p.rows - 1) / p.rows);
    for (int o = 32; o >= cols; o >>= 1) {
        const float nb = __shfl_xor(nn, o, 64), nt = nn + nb, f = nt > 0.f ? nb / nt : 0.f, nf = nn * f;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float mb = __shfl_xor(mean[k], o, 64), qb = __shfl_xor(m[k], o, 64), d = nt > nn ? mb - mean[k] : 0.f;
            mean[k] = nn > 0.f ? fmaf(d, f, mean[k]) : mb;
            m[k] += qb + d * d * nf;
        }
        nn = nt;
    }
    const int slot = cols > 64 ? i.rs : threadIdx.x >> 6;
    if (cols > 64 || (threadIdx.x & 63) < cols) {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (i.on && k >= i.dup && i.c + k < a.C) {
                sm[slot * width + i.c - i.c0 + k] = mean[k];
                sq[slot * width + i.c - i.c0 + k] = m[k];
            }
        if ((threadIdx.x & (cols - 1)) == 0) sn[slot] = nn;
    }
    __syncthreads();
    // the slots of a channel, to slot 0
    const float rows = (float)(i.hi - i.lo);
    for (int c = threadIdx.x; c < i.W; c += 256) {
        float n = sn[0], mc = sm[c], qc = sq[c];
        for (int w = 1; w < p.slots; ++w) {
            const float nb = sn[w], d = sm[w * width + c] - mc, nt = n + nb;
            if (nb > 0.f) {
                mc = fmaf(d, nb / nt, mc);
                qc += sq[w * width + c] + d * d * (n * nb / nt);
                n = nt;
            }
        }
        sm[c] = mc;
        sq[c] = qc;
    }
    __syncthreads();
    // the channels of a group: 2^llg lanes each
    const int gl = i.c0 / a.Cg, gh = (i.c0 + i.W - 1) / a.Cg, step = 1 << p.llg, l = threadIdx.x & (step - 1);
    for (int g = gl + (threadIdx.x >> p.llg); g <= gh; g += 256 >> p.llg) {
        const int cl = max(g * a.Cg - i.c0, 0), ch = min((g + 1) * a.Cg - i.c0, i.W);
        float t = 0.f, q = 0.f;
        for (int c = cl + l; c < ch; c += step) t += sm[c];
        for (int o = step >> 1; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
        const float gm = t / (float)(ch - cl);
        for (int c = cl + l; c < ch; c += step) {
            const float d = sm[c] - gm;
            q += sq[c] + rows * (d * d);
        }
        for (int o = step >> 1; o > 0; o >>= 1) q += __shfl_xor(q, o, 64);
        if (l == 0)
            part[((long long)i.n * a.G + g) * p.P * p.tg + i.q * p.tg + i.tile - g * a.Cg / (V << p.lc)] =
                make_float4(rows * (float)(ch - cl), gm, q, 0.f);
    }
}

// A wave per (sample, group): the mean of its parts' means, then the squares about it, in fp64.  4.8 us for 512 groups of 256 parts, two
// rounds of loads and shuffles.
template <int V>
__global__ __launch_bounds__(256) void gn_stats_join_kernel(GnArgs a, GnParts p, const float4* part) {
    const int id = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63;
    if (id >= a.N * a.G) return;
    const int g = id % a.G, tw = V << p.lc, tg = ((g + 1) * a.Cg - 1) / tw - g * a.Cg / tw + 1;    // tiles the group touches
    const float4* mine = part + (long long)id * p.P * p.tg;
    const int all = p.P * p.tg;
    double total = 0.0, squares = 0.0;
    // eight parts a lane in flight; the first eight stay for the second sum (a map of one tile has at most 512 parts)
    float4 o[8];
    const auto fetch = [&](int b) {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = b + u * 64 + l;
            o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i < all && (p.tg == 1 || i % p.tg < tg)) o[u] = mine[i];
        }
    };
    for (int b = 0; b < all; b += 512) {
        fetch(b);
#pragma unroll
        for (int u = 0; u < 8; ++u) total += (double)o[u].x * o[u].y;
    }
    const double count = (double)a.S * a.Cg, mean = wave_sum_d(total) / count;
    for (int b = 0; b < all; b += 512) {
        if (all > 512) fetch(b);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const double d = o[u].y - mean;
            squares += o[u].z + d * d * o[u].x;
        }
    }
    squares = wave_sum_d(squares);
    if (l == 0) {
        a.mean[id] = (float)mean;
        a.rstd[id] = (float)(1.0 / sqrt(squares / count + (double)a.eps));
    }
}

// The same for the groups of a workgroup's tile, 2^llg lanes each, to LDS: where the parts are few, every workgroup of the second pass joins
// them itself and a launch is saved.  stat[g - gl] = (mean, 1 / std).
#define GN_JOIN_GROUPS 512
template <int V>
__device__ __forceinline__ int join_here(const GnArgs& a, const GnParts& p, const GnWhere& i, const float4* part, float2* stat) {
    const int first = a.C < V ? 0 : min(i.c0, a.C - V), gl = first / a.Cg, gh = (i.c0 + i.W - 1) / a.Cg, tw = V << p.lc;
    const int step = 1 << p.llg, l = threadIdx.x & (step - 1), all = p.P * p.tg;
    const double inv = 1.0 / ((double)a.S * a.Cg);
    for (int g = gl + (threadIdx.x >> p.llg); g <= gh; g += 256 >> p.llg) {
        const int t0 = g * a.Cg / tw, tg = ((g + 1) * a.Cg - 1) / tw - t0 + 1;
        const float4* mine = part + ((long long)i.n * a.G + g) * all;
        double total = 0.0, squares = 0.0;
        for (int q = l; q < all; q += step)
            if (p.tg == 1 || q % p.tg < tg) total += (double)mine[q].x * mine[q].y;
        for (int o = step >> 1; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
        const double mean = total * inv;
        for (int q = l; q < all; q += step)
            if (p.tg == 1 || q % p.tg < tg) {
                const float4 o = mine[q];
                const double d = o.y - mean;
                squares += o.z + d * d * o.x;
            }
        for (int o = step >> 1; o > 0; o >>= 1) squares += __shfl_xor(squares, o, 64);
        if (l == 0) {
            const float2 r = make_float2((float)mean, (float)(1.0 / sqrt(squares * inv + (double)a.eps)));
            stat[g - gl] = r;
            if (i.q == 0 && t0 == i.tile) {
                a.mean[i.n * a.G + g] = r.x;
                a.rstd[i.n * a.G + g] = r.y;
            }
        }
    }
    __syncthreads();
    return gl;
}

// y.  `part` where the groups' parts are joined here.  268 MB (16 x 65536 x 64 bf16) in 45 us, 6.0 TB/s: memory, half of it from the Infinity
// Cache that the statistics have filled.
template <class E, int ACT, bool NT>
__global__ __launch_bounds__(256) void gn_apply_kernel(GnArgs a, GnParts p, const float4* part) {
    constexpr int V = E::V, U = 4;
    __shared__ float2 stat[GN_JOIN_GROUPS];
    const GnWhere i = where_of<V>(a, p, blockIdx.x);
    const int gl = part ? join_here<V>(a, p, i, part, stat) : 0;
    if (!i.on) return;
    float mean[V], rstd[V], w[V], b[V];
    load_params<E>(a.w, a.ptype, i.c, a.C, 1.f, w);
    load_params<E>(a.b, a.ptype, i.c, a.C, 0.f, b);
    if (part) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float2 st = stat[min(i.c + k, a.C - 1) / a.Cg - gl];
            mean[k] = st.x;
            rstd[k] = st.y;
        }
    } else {
        load_stats<V>(a, i.n, i.c, mean, rstd);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) w[k] *= rstd[k];
    const typename E::T* x = (const typename E::T*)a.x + i.n * a.xs + i.c;
    typename E::T* y = (typename E::T*)a.y + (long long)i.n * a.S * a.C + i.c;
    for (int r = i.lo + i.rs; r < i.hi; r += U * p.rows) {
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * p.rows < i.hi) raw[u] = load_vec<E>(x + (long long)(r + u * p.rows) * a.xr, a.C);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * p.rows < i.hi) {
                float v[V];
                E::unpack(raw[u], v);
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = act_fwd<ACT>(fmaf(v[k] - mean[k], w[k], b[k]), a.slope);
                store_tail<E, NT>(y + (long long)(r + u * p.rows) * a.C, i.dup, a.C, v);
            }
    }
}

// part[n][q][c] = (sum dz, sum dz h) over the part's positions.  268 MB (4 x 65536 x 256 bf16) in 48 us, 5.6 TB/s: memory.
template <class E, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(GnArgs a, GnParts p, float2* part) {
    constexpr int V = E::V, U = 4;
    __shared__ float r1[4 * 64 * V], r2[4 * 64 * V];
    const GnWhere i = where_of<V>(a, p, blockIdx.x);
    const int cols = 1 << p.lc, width = cols * V;
    float A[V] = {}, B[V] = {};
    if (i.on) {
        float mean[V], rstd[V], w[V], b[V];
        load_params<E>(a.w, a.ptype, i.c, a.C, 1.f, w);
        load_params<E>(a.b, a.ptype, i.c, a.C, 0.f, b);
        load_stats<V>(a, i.n, i.c, mean, rstd);
#pragma unroll
        for (int k = 0; k < V; ++k) w[k] *= rstd[k];
        const typename E::T* x = (const typename E::T*)a.x + i.n * a.xs + i.c;
        const typename E::T* dy = (const typename E::T*)a.dy + i.n * a.ds + i.c;
        for (int r = i.lo + i.rs; r < i.hi; r += U * p.rows) {
            u32x4 rx[U], rd[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * p.rows < i.hi) {
                    rx[u] = load_vec<E>(x + (long long)(r + u * p.rows) * a.xr, a.C);
                    rd[u] = load_vec<E>(dy + (long long)(r + u * p.rows) * a.dr, a.C);
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * p.rows < i.hi) {
                    float v[V], d[V];
                    E::unpack(rx[u], v);
                    E::unpack(rd[u], d);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float e = v[k] - mean[k], dz = act_bwd<ACT>(d[k], fmaf(e, w[k], b[k]), a.slope);
                        A[k] += dz;
                        B[k] = fmaf(dz, e, B[k]);
                    }
                }
        }
#pragma unroll
        for (int k = 0; k < V; ++k) B[k] *= rstd[k];
    }
    same_vector_sums(A, cols);
    same_vector_sums(B, cols);
    if (cols > 64 || (threadIdx.x & 63) < cols) {
        const int slot = cols > 64 ? i.rs : threadIdx.x >> 6;
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (i.on && k >= i.dup && i.c + k < a.C) {
                r1[slot * width + i.c - i.c0 + k] = A[k];
                r2[slot * width + i.c - i.c0 + k] = B[k];
            }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < i.W; c += 256) {
        float s = 0.f, t = 0.f;
        for (int r = 0; r < p.slots; ++r) {
            s += r1[r * width + c];
            t += r2[r * width + c];
        }
        part[((long long)i.n * p.P + i.q) * a.C + i.c0 + c] = make_float2(s, t);
    }
}

// `chunks` workgroups per (sample, group): the parts of its channels, in order; ab[n][c], and the (s1 / M, s2 / M) of a workgroup's channels to
// coef[n][g][chunk].  5.2 us for 128 groups of 8 channels in 512 parts.
__global__ __launch_bounds__(256) void gn_bwd_join_kernel(GnArgs a, int P, int lcw, int chunks, const float2* part, float2* ab, float2* coef) {
    __shared__ float2 sh[256];
    const int ng = blockIdx.x / chunks, n = ng / a.G, g = ng - n * a.G;
    const int cw = 1 << lcw, slots = 256 >> lcw, slot = threadIdx.x >> lcw, cl = threadIdx.x & (cw - 1);
    float s1 = 0.f, s2 = 0.f;
    for (long long c0 = (long long)(blockIdx.x - ng * chunks) << lcw; c0 < a.Cg; c0 += (long long)chunks << lcw) {
        const int c = g * a.Cg + (int)c0 + cl;
        float2 v = make_float2(0.f, 0.f);
        if (c0 + cl < a.Cg) {
            const float2* mine = part + (long long)n * P * a.C + c;
            int q = slot;
            for (; q + 3 * slots < P; q += 4 * slots) {
                float2 o[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) o[u] = mine[(long long)(q + u * slots) * a.C];
#pragma unroll
                for (int u = 0; u < 4; ++u) { v.x += o[u].x; v.y += o[u].y; }
            }
            for (; q < P; q += slots) {
                const float2 o = mine[(long long)q * a.C];
                v.x += o.x;
                v.y += o.y;
            }
        }
        sh[threadIdx.x] = v;
        __syncthreads();
        for (int o = slots >> 1; o > 0; o >>= 1) {
            if (slot < o) {
                const float2 q = sh[((slot + o) << lcw) + cl];
                v.x += q.x;
                v.y += q.y;
                sh[threadIdx.x] = v;
            }
            __syncthreads();
        }
        if (slot == 0 && c0 + cl < a.Cg) {
            ab[(long long)n * a.C + c] = v;
            const float w = a.w ? load_any(a.w, a.ptype, c) : 1.f;
            s1 = fmaf(w, v.x, s1);
            s2 = fmaf(w, v.y, s2);
        }
        __syncthreads();
    }
    sh[threadIdx.x] = make_float2(s1, s2);
    __syncthreads();
    if (threadIdx.x < 64) {
        float t1 = 0.f, t2 = 0.f;
        for (int q = threadIdx.x; q < 256; q += 64) { t1 += sh[q].x; t2 += sh[q].y; }
        t1 = wave_sum(t1);
        t2 = wave_sum(t2);
        const float inv = 1.f / ((float)a.S * (float)a.Cg);
        if (threadIdx.x == 0) coef[blockIdx.x] = make_float2(t1 * inv, t2 * inv);
    }
}

// The chunks of a group, a wave each group: coef[n][g].
__global__ __launch_bounds__(256) void gn_bwd_coef_kernel(int groups, int chunks, const float2* chunk, float2* coef) {
    const int id = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= groups) return;
    float t1 = 0.f, t2 = 0.f;
    for (int q = threadIdx.x & 63; q < chunks; q += 64) {
        const float2 o = chunk[(long long)id * chunks + q];
        t1 += o.x;
        t2 += o.y;
    }
    t1 = wave_sum(t1);
    t2 = wave_sum(t2);
    if ((threadIdx.x & 63) == 0) coef[id] = make_float2(t1, t2);
}

// dw, db: 2^lcp channels a workgroup at a time, 256 >> lcp lanes a channel share its `rows` partial sums, eight in flight.  In fp64: each row is the
// sum of a sample or of a walker's samples, and there may be a million of them.
__device__ __forceinline__ void params_of(const GnArgs& a, int blk, int nblk, int lcp, int rows, const float2* ab) {
    __shared__ double2 sh[256];
    const int cl = threadIdx.x & ((1 << lcp) - 1), slot = threadIdx.x >> lcp, slots = 256 >> lcp;
    for (int c0 = blk << lcp; c0 < a.C; c0 += nblk << lcp) {
        const int c = c0 + cl;
        double vx = 0.0, vy = 0.0;
        if (c < a.C)
            for (int r0 = slot; r0 < rows; r0 += 8 * slots) {
                float2 o[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const long long r = r0 + (long long)u * slots;
                    o[u] = r < rows ? ab[r * a.C + c] : make_float2(0.f, 0.f);
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    vx += o[u].x;
                    vy += o[u].y;
                }
            }
        sh[threadIdx.x] = make_double2(vx, vy);
        for (int o = slots >> 1; o > 0; o >>= 1) {
            __syncthreads();
            if (slot < o) {
                const double2 q = sh[threadIdx.x + (o << lcp)];
                vx += q.x;
                vy += q.y;
                sh[threadIdx.x] = make_double2(vx, vy);
            }
        }
        if (slot == 0 && c < a.C) {
            if (a.dw) store_any(a.dw, a.ptype, c, (float)vy);
            if (a.db) store_any(a.db, a.ptype, c, (float)vx);
        }
        __syncthreads();
    }
}
__global__ __launch_bounds__(256) void gn_params_kernel(GnArgs a, int lcp, int rows, const float2* ab) {
    params_of(a, blockIdx.x, gridDim.x, lcp, rows, ab);
}

// dx; the first `pblocks` workgroups sum the parameters' gradients instead.  NT: 1 stores past the caches, 2 loads too.  403 MB (4 x 65536 x 256
// bf16) in 66 us, 6.1 TB/s: memory.
template <class E, int ACT, int NT>
__global__ __launch_bounds__(256) void gn_bwd_dx_kernel(GnArgs a, GnParts p, const float2* coef, int pblocks, int lcp, const float2* ab) {
    constexpr int V = E::V, U = 4;
    if ((int)blockIdx.x < pblocks) {
        params_of(a, blockIdx.x, pblocks, lcp, a.N, ab);
        return;
    }
    const GnWhere i = where_of<V>(a, p, blockIdx.x - pblocks);
    if (!i.on) return;
    float mean[V], rstd[V], w[V], b[V];
    float2 cf[V];
    load_params<E>(a.w, a.ptype, i.c, a.C, 1.f, w);
    load_params<E>(a.b, a.ptype, i.c, a.C, 0.f, b);
    load_stats<V>(a, i.n, i.c, mean, rstd, coef, cf);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        w[k] *= rstd[k];
        cf[k].x *= rstd[k];
        cf[k].y *= rstd[k];
    }
    const typename E::T* x = (const typename E::T*)a.x + i.n * a.xs + i.c;
    const typename E::T* dy = (const typename E::T*)a.dy + i.n * a.ds + i.c;
    typename E::T* dx = (typename E::T*)a.y + (long long)i.n * a.S * a.C + i.c;
    for (int r = i.lo + i.rs; r < i.hi; r += U * p.rows) {
        u32x4 rx[U], rd[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * p.rows < i.hi) {
                rx[u] = load_vec<E, NT == 2>(x + (long long)(r + u * p.rows) * a.xr, a.C);
                rd[u] = load_vec<E, NT == 2>(dy + (long long)(r + u * p.rows) * a.dr, a.C);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * p.rows < i.hi) {
                float v[V], d[V];
                E::unpack(rx[u], v);
                E::unpack(rd[u], d);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float e = v[k] - mean[k], dz = act_bwd<ACT>(d[k], fmaf(e, w[k], b[k]), a.slope);
                    v[k] = fmaf(-(e * rstd[k]), cf[k].y, fmaf(dz, w[k], -cf[k].x));
                }
                store_tail<E, NT != 0>(dx + (long long)(r + u * p.rows) * a.C, i.dup, a.C, v);
            }
    }
}

// ---------------------------------------------------------------- host
static int vec_of(int dtype) { return dtype == AG2V_F32 ? ElemF32::V : ElemBF16::V; }

// A launch takes fewer than 2^32 threads in all.  Batches that need more workgroups go by several launches of `per` samples.
#define GN_SLAB_BLOCKS ((1 << 22) - 1)      // of up to 1024 threads
#define GN_BLOCKS ((1 << 23) - 1)           // of 256, and beside as many again
#define GN_PARAM_BLOCKS (1 << 20)
// Which way (S, C, G) runs, forward or backward, and what N samples need.  Nothing but `per`, the walkers and the workspace depends on N: a sample's
// result is the same, bit for bit, in a batch of any size.
struct GnPlan {
    bool slab, one, join_here;      // one: a vector lies inside one group; join_here: the second pass joins the parts itself
    GnSlab s;
    int U, threads, walkers;
    int per;                         // samples a launch
    size_t lds;
    GnParts p;
    int lcw, chunks;                 // backward: log2 of the channels, and workgroups a group, that join the parts
    long long words, ab, coef, chunk;       // workspace in floats; offsets of ab[][C], coef[N][G] and the chunks' in it
};
// Vectors of a slab at most.  Forward, 8192: 4096 x 256 fp16 in 32 groups, replayed, take 13.6 us (one sample), 19.4 (8) and 92 (64), in parts of the same
// build 15.7, 21.4 and 82; 1961 x 90 fp32 in 6 groups 10.3, 11.3 and 32.5, in parts 10.9, 12.4 and 33.6.  Backward, where x and dy are held, 1024:
// the 2000 vectors of 64 x 2000 x 64 fp16 in 8 groups took 55 us a training pass, 44 in parts, and 24 and 19.5 for one sample.
#define GN_SLAB_FWD 8192
#define GN_SLAB_BWD 1024
#define GN_JOIN_SPLIT 8192
static bool plan_slab(GnPlan& r, int V, int N, int S, int C, int G, bool backward) {
    const int Cg = C / G;
    const auto lcols = [&](int k) { return log2_up(((long long)k * Cg + V - 1) / V); };
    const long long most = backward ? GN_SLAB_BWD : GN_SLAB_FWD;        // vectors a slab
    // Groups of a slab: rows of 64 bytes, so that few slabs share a cache line.  Where what the slabs of a sample read is small enough to stay in an
    // XCD's L2, that does not matter and more workgroups do: 512 vectors are enough then (4 x 1000 x 320 fp16 in 40 groups, forward: one group a slab
    // 7.5 us, four 9.6, eight 13.2; 16 x 100 x 256 fp32 in 64 groups: 6.5, 5.8 and 6.0), or one group of an odd width (2 x 120 x 90 bf16 in 6 groups,
    // training: 16.5 us, two groups 20.2).
    const long long bytes = (long long)S * C * (16 / V) * (backward ? 2 : 1);
    const bool small = bytes <= (1 << 20);
    // Rows of whole vectors at least, where that is not a matter of a few workgroups: 64 x 930 x 298 bf16 in 149 groups took 150 us forward in rows of
    // one group, 4 bytes, and takes 55, 64 x 1500 x 64 fp16 in 32 groups 58 and 17 (one sample 9.6 and 11.1), 64 x 480 x 300 bf16 in 100 groups 80 and
    // 47 (one sample 7.9 and 10.2); but 600 x 8 fp16 in 4 groups 7.3 and 10.
    const bool whole = S > 2048 || (long long)S * C * (16 / V) >= 65536;
    int kg = 1;
    while (kg < G && (long long)kg * Cg < 4 * V && lcols(kg + 1) <= 2 && ((long long)S << lcols(kg + 1)) <= most &&
           !(small && (((long long)S << lcols(kg)) >= 512 || (Cg % V && 4 * Cg >= V)) && (!whole || (long long)kg * Cg >= V)))
        ++kg;
    const int lc = lcols(kg);
    // Narrow rows of a larger map: every cache line would be fetched by many slabs, in pieces (13 x 1085 x 1560 fp16 in 195 groups, one vector a
    // row: 147 us a training pass, 72 us in parts; 11 x 4181 x 45 fp32 in 15 groups, 12 bytes a row: 49 and 37 us).  Forward, rows of whole
    // vectors take one launch and are no slower up to 8 samples (figures at GN_SLAB_FWD).
    if (kg < G && (long long)kg * Cg < V && S > 2048) return false;
    const long long held = (long long)S << lc;
    if (!small && kg < G && !backward && (long long)kg * Cg < 2 * V && Cg % V) return false;
    // Backward they are, beyond 512 vectors in rows of up to 32 bytes also on small maps: 64 x 1024 x 256 bf16 in 32 groups took 87 us a training
    // pass, 71 in parts (one sample 18.8 and 19.1), and 64 x 1000 x 50 fp16 in 10 groups 61 and 46.  Rows of 60 are not: 200 x 90 fp32 in 6 groups
    // 14.3 and 15.6.
    if (kg < G && backward && ((!small && (long long)kg * Cg < 4 * V) || (held > 512 && (long long)kg * Cg <= 2 * V))) return false;
    if (lc > 10 || held > most) return false;
    const bool one = kg == 1 || Cg % V == 0;
    // 512 threads, which meet sooner and leave room for a second workgroup on the CU: 64 x 256 x 1280 bf16 forward took 50 us with 1024 threads and
    // takes 31, 64 x 533 x 608 fp16 59 and 37.  1024 for rows that wide, and where the registers of 512 do not hold the slab and at least three
    // quarters of the lanes work (64 x 1024 x 1280 fp16, 5 vectors in 8 lanes: 134 us, in parts 85).
    const int maxU = backward ? 2 : one ? 8 : 4;
    const bool large = !backward && held > 512 * maxU;
    if (large && ((long long)kg * Cg + V - 1) / V * 4 < 3LL << lc) return false;
    const int maxT = large || (one && lc == 10) ? 1024 : 512;
    int T = 64;
    while (T < maxT && (held > (long long)T * 2 || T < (1 << lc))) T *= 2;
    if (T < (1 << lc)) return false;
    const int rows = T >> lc, U = (S + rows - 1) / rows;
    if (U > maxU) return false;
    r.slab = true;
    r.one = one;
    r.U = U <= 1 ? 1 : U <= 2 ? 2 : U <= 4 ? 4 : 8;
    r.threads = T < 256 ? 256 : T;
    r.s.T = T;
    r.s.kg = kg;
    r.s.nsets = (G + kg - 1) / kg;
    r.s.lc = lc;
    r.s.rows = rows;
    r.s.slots = lc > 6 ? rows : T / 64;
    r.s.wg = kg == 1 && one ? 1 << lc : one ? Cg / V : Cg;
    r.s.llg = share_lanes(T, kg);
    const int subs = r.threads / T;
    r.lds = sizeof(float) * subs * (((size_t)r.s.slots << lc) * (backward ? (one ? V : 2 * V) : (one ? 1 : V)) + 2 * kg);
    if (r.s.nsets > GN_SLAB_BLOCKS || r.lds > 64 * 1024) return false;
    r.per = N;
    if (!backward) {
        const long long per = (long long)GN_SLAB_BLOCKS * subs / r.s.nsets;
        if (per < N) r.per = (int)per;
    } else {                             // (any number of samples in one launch)
        long long wb = ((long long)N + subs - 1) / subs;
        // at most 2048 workgroups, but no walker over 256 samples: it adds them up in fp32
        long long cap = 2048 / r.s.nsets < 1 ? 1 : 2048 / r.s.nsets;
        if (cap * subs * 256 < N) cap = ((long long)N + 256 * subs - 1) / (256 * subs);
        if (wb > cap) wb = cap;
        r.walkers = (int)wb * subs;
        r.words = 2LL * r.walkers * C;
    }
    return true;
}
static GnPlan plan_of(int dtype, int N, int S, int C, int G, bool backward) {
    GnPlan r = {};
    const int V = vec_of(dtype), Cg = C / G;
    if (plan_slab(r, V, N, S, C, G, backward)) return r;
    r = GnPlan();
    GnParts& p = r.p;
    // tiles of 2^lc vectors: the widest, up to a row of 256, that leaves at most an eighth of the lanes idle; 64 bytes (or the row) otherwise
    const long long cvs = ((long long)C + V - 1) / V;
    int lc = log2_up(cvs < 256 ? cvs : 256);
    while (lc > 2 && ((((cvs - 1) >> lc) + 1) << lc) * 8 > cvs * 9) --lc;
    p.lc = lc;
    p.tiles = (int)(((cvs - 1) >> lc) + 1);
    p.rows = 256 >> lc;
    p.slots = lc > 6 ? p.rows : 4;
    // 8 positions a thread; 4 where a sample would have less than 64 workgroups, 2 where less than 32 (1 x 1961 x 90 fp32, 48 workgroups: 22.0 us a
    // training pass with 4, 20.7 with 2; 64 x 1961 x 90 79 and 86); more where it would have over 512 parts, or more workgroups than a launch takes.
    long long P = 0;
    for (long long each = 8; each >= 2; each /= 2) {
        P = (S + each * p.rows - 1) / (each * p.rows);
        if (P * p.tiles >= 8 * each) break;
    }
    if (P > 512) P = 512;
    while (P > 1 && P * p.tiles > GN_BLOCKS) P /= 2;
    p.len = (int)((S + P - 1) / P);
    p.P = (S + p.len - 1) / p.len;
    p.tg = (int)(((long long)Cg - 1) / (V << lc) + 2);
    if (p.tg > p.tiles) p.tg = p.tiles;
    long long per = GN_BLOCKS / ((long long)p.P * p.tiles);
    if (backward) {
        // One workgroup a group; wide groups in many parts take one per 16 channels (more where the parts are few), and a launch more that adds
        // those up: 1 x 65536 x 512 bf16 in one group, 512 parts, 200 us a training pass with one workgroup and 114 so, 4 x 4 x 8192 in one group 49
        // and 23; 65536 x 256 in 32 groups, 4096 sums a group, 70 and 71.
        r.lcw = log2_up(Cg < 256 ? Cg : 256);
        r.chunks = 1;
        if ((long long)Cg * p.P >= GN_JOIN_SPLIT) {
            const int slots = log2_up((p.P + 7) / 8);
            r.lcw = 8 - (slots < 4 ? slots : 4);
            const long long most = GN_BLOCKS / G < 1 ? 1 : GN_BLOCKS / G, chunks = ((long long)Cg + (1 << r.lcw) - 1) >> r.lcw;
            r.chunks = (int)(chunks < most ? chunks : most);
        }
        const long long joins = 2LL * GN_BLOCKS / ((long long)G * r.chunks);
        if (joins < per) per = joins < 1 ? 1 : joins;
        r.per = per < N ? (int)per : N;
        r.ab = 2LL * r.per * p.P * C;
        r.coef = r.ab + 2LL * N * C;
        r.chunk = r.coef + 2LL * r.per * G;
        r.words = r.chunk + (r.chunks > 1 ? 2LL * r.per * G * r.chunks : 0);
    } else {
        r.per = per < N ? (int)per : N;
        const long long per = ((long long)V << lc) / Cg + 2;
        const long long groups = per < G ? per : G;
        p.llg = share_lanes(256, (int)groups);
        r.join_here = groups <= GN_JOIN_GROUPS && groups * p.P * p.tg <= 2048;
        r.words = 4LL * r.per * G * p.P * p.tg;
    }
    return r;
}

// Results that go past the caches: large ones whose rows are whole 64-byte pieces.  Others would reach memory in parts of pieces: 10 x 21888 x
// 150 bf16 forward took 60 us that way and 29 us this way.
template <class E>
static bool past_caches(const GnArgs& a) {
    return (long long)a.N * a.S * a.C * (long long)sizeof(typename E::T) > AG2V_NT_STORE_BYTES && a.C * (long long)sizeof(typename E::T) % 64 == 0;
}

// `count` samples from n0 on
template <class E>
static GnArgs samples_of(const GnArgs& a, int n0, int count) {
    typedef typename E::T T;
    GnArgs b = a;
    b.x = (const T*)a.x + n0 * a.xs;
    if (a.dy) b.dy = (const T*)a.dy + n0 * a.ds;
    if (a.y) b.y = (T*)a.y + (long long)n0 * a.S * a.C;
    b.mean = a.mean + (long long)n0 * a.G;
    b.rstd = a.rstd + (long long)n0 * a.G;
    b.N = a.N - n0 < count ? a.N - n0 : count;
    return b;
}

template <class E, int ACT, bool ONE>
static int run_slab_fwd(const GnArgs& a, const GnPlan& r, hipStream_t st) {
    GnSlab s = r.s;
    s.nslab = (long long)a.N * s.nsets;
    const int subs = r.threads / s.T;
    const dim3 grid(ceil_div(s.nslab, subs)), block(r.threads);
    if (r.U == 1) hipLaunchKernelGGL((gn_slab_fwd_kernel<E, ACT, 1, ONE>), grid, block, r.lds, st, a, s);
    else if (r.U == 2) hipLaunchKernelGGL((gn_slab_fwd_kernel<E, ACT, 2, ONE>), grid, block, r.lds, st, a, s);
    else if (r.U == 4 || !ONE) hipLaunchKernelGGL((gn_slab_fwd_kernel<E, ACT, 4, ONE>), grid, block, r.lds, st, a, s);
    else if constexpr (ONE) hipLaunchKernelGGL((gn_slab_fwd_kernel<E, ACT, 8, true>), grid, block, r.lds, st, a, s);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
template <class E, int ACT, bool ONE>
static int run_slab_bwd(const GnArgs& a, const GnPlan& r, float2* ab, hipStream_t st) {
    const dim3 grid(r.walkers / (r.threads / r.s.T) * r.s.nsets), block(r.threads);
    if (r.U == 1) hipLaunchKernelGGL((gn_slab_bwd_kernel<E, ACT, 1, ONE>), grid, block, r.lds, st, a, r.s, r.walkers, ab);
    else hipLaunchKernelGGL((gn_slab_bwd_kernel<E, ACT, 2, ONE>), grid, block, r.lds, st, a, r.s, r.walkers, ab);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
template <class E, int ACT>
static int run_fwd(const GnArgs& a, const GnPlan& r, bool past, float* ws, hipStream_t st) {
    if (r.slab) return r.one ? run_slab_fwd<E, ACT, true>(a, r, st) : run_slab_fwd<E, ACT, false>(a, r, st);
    const int blocks = a.N * r.p.P * r.p.tiles;
    hipLaunchKernelGGL(gn_stats_kernel<E>, dim3(blocks), dim3(256), 0, st, a, r.p, (float4*)ws);
    AG2V_CHECK_LAUNCH();
    const float4* part = (const float4*)ws;
    if (!r.join_here) {
        hipLaunchKernelGGL(gn_stats_join_kernel<E::V>, dim3(ceil_div((long long)a.N * a.G, 4)), dim3(256), 0, st, a, r.p, part);
        AG2V_CHECK_LAUNCH();
        part = nullptr;
    }
    if (past)
        hipLaunchKernelGGL((gn_apply_kernel<E, ACT, true>), dim3(blocks), dim3(256), 0, st, a, r.p, part);
    else
        hipLaunchKernelGGL((gn_apply_kernel<E, ACT, false>), dim3(blocks), dim3(256), 0, st, a, r.p, part);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
// Workgroups that sum the parameters' gradients, and log2 of the channels each takes at a time: 32, fewer where a channel's lanes would have over 64
// rows each and few channels leave most of the chip without work (8192 x 16 x 16 fp32 in one group, 8192 rows: 61 us a backward pass, 257 with 32
// channels a workgroup and one load in flight).
static int param_blocks(int C, int rows, int& lcp) {
    lcp = 5;
    while (lcp > 0 && rows > 64 * (256 >> lcp) && C >> lcp < 64) --lcp;
    const int blocks = ceil_div(C, 1 << lcp);
    return blocks < GN_PARAM_BLOCKS ? blocks : GN_PARAM_BLOCKS;
}
static int run_params(const GnArgs& a, int rows, const float2* ab, hipStream_t st) {
    int lcp;
    const int blocks = param_blocks(a.C, rows, lcp);
    hipLaunchKernelGGL(gn_params_kernel, dim3(blocks), dim3(256), 0, st, a, lcp, rows, ab);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
// Backward in parts: sums[n][C] of the samples of `a`; dx, and beside it the parameters' gradients where `params`.
template <class E, int ACT>
static int run_bwd_parts(const GnArgs& a, const GnPlan& r, bool past, bool params, float2* sums, float* ws, hipStream_t st) {
    float2 *part = (float2*)ws, *coef = (float2*)(ws + r.coef);
    const int blocks = a.N * r.p.P * r.p.tiles;
    hipLaunchKernelGGL((gn_bwd_sums_kernel<E, ACT>), dim3(blocks), dim3(256), 0, st, a, r.p, part);
    AG2V_CHECK_LAUNCH();
    float2* chunk = r.chunks > 1 ? (float2*)(ws + r.chunk) : coef;
    hipLaunchKernelGGL(gn_bwd_join_kernel, dim3(a.N * a.G * r.chunks), dim3(256), 0, st, a, r.p.P, r.lcw, r.chunks, part, sums, chunk);
    AG2V_CHECK_LAUNCH();
    if (r.chunks > 1) {
        hipLaunchKernelGGL(gn_bwd_coef_kernel, dim3(ceil_div((long long)a.N * a.G, 4)), dim3(256), 0, st, a.N * a.G, r.chunks, chunk, coef);
        AG2V_CHECK_LAUNCH();
    }
    if (!a.y) return params ? run_params(a, a.N, sums, st) : AG2V_OK;
    int lcp = 0;
    const int pblocks = params ? param_blocks(a.C, a.N, lcp) : 0;
    const dim3 grid(blocks + pblocks);
    if (past && r.p.tiles == 1)      // (x and dy together pass the bound of loads; the lines of a tiled row are read twice)
        hipLaunchKernelGGL((gn_bwd_dx_kernel<E, ACT, 2>), grid, dim3(256), 0, st, a, r.p, coef, pblocks, lcp, sums);
    else if (past)
        hipLaunchKernelGGL((gn_bwd_dx_kernel<E, ACT, 1>), grid, dim3(256), 0, st, a, r.p, coef, pblocks, lcp, sums);
    else
        hipLaunchKernelGGL((gn_bwd_dx_kernel<E, ACT, 0>), grid, dim3(256), 0, st, a, r.p, coef, pblocks, lcp, sums);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
template <class E, int ACT>
static int run_bwd(const GnArgs& a, const GnPlan& r, bool past, float* ws, hipStream_t st) {
    const bool params = a.dw || a.db;
    if (r.slab) {
        float2* out = params ? (float2*)ws : nullptr;
        const int rc = r.one ? run_slab_bwd<E, ACT, true>(a, r, out, st) : run_slab_bwd<E, ACT, false>(a, r, out, st);
        return rc != AG2V_OK || !params ? rc : run_params(a, r.walkers, out, st);
    }
    float2* sums = (float2*)(ws + r.ab);
    if (r.per == a.N) return run_bwd_parts<E, ACT>(a, r, past, params, sums, ws, st);
    for (int n0 = 0; n0 < a.N; n0 += r.per) {
        const int rc = run_bwd_parts<E, ACT>(samples_of<E>(a, n0, r.per), r, past, false, sums + (long long)n0 * a.C, ws, st);
        if (rc != AG2V_OK) return rc;
    }
    return params ? run_params(a, a.N, sums, st) : AG2V_OK;
}
template <class E, int ACT>
static int run_act(const GnArgs& a, const GnPlan& r, bool backward, float* ws, hipStream_t st) {
    const bool past = past_caches<E>(a);
    if (backward) return run_bwd<E, ACT>(a, r, past, ws, st);
    for (int n0 = 0; n0 < a.N; n0 += r.per) {
        const int rc = run_fwd<E, ACT>(samples_of<E>(a, n0, r.per), r, past, ws, st);
        if (rc != AG2V_OK) return rc;
    }
    return AG2V_OK;
}
template <class E>
static int run_elem(const GnArgs& a, const GnPlan& r, int act, bool backward, float* ws, hipStream_t st) {
    if (act == ACT_SILU) return run_act<E, ACT_SILU>(a, r, backward, ws, st);
    if (act == ACT_LRELU) return run_act<E, ACT_LRELU>(a, r, backward, ws, st);
    return run_act<E, ACT_NONE>(a, r, backward, ws, st);
}
static int run_any(const GnArgs& a, int dtype, int act, bool backward, float* ws, size_t ws_floats, hipStream_t st) {
    const GnPlan r = plan_of(dtype, a.N, a.S, a.C, a.G, backward);
    if ((r.words && !ws) || ws_floats < (size_t)r.words || ((uintptr_t)ws & 15)) return AG2V_EINVAL;
    if (dtype == AG2V_F32) return run_elem<ElemF32>(a, r, act, backward, ws, st);
    return dtype == AG2V_BF16 ? run_elem<ElemBF16>(a, r, act, backward, ws, st) : run_elem<ElemF16>(a, r, act, backward, ws, st);
}

static bool sizes_ok(int dtype, int ptype, int N, int S, int C, int groups, int act) {
    if (dtype < AG2V_F32 || dtype > AG2V_F16 || ptype < AG2V_F32 || ptype > AG2V_F16 || act < ACT_NONE || act > ACT_LRELU) return false;
    if (ptype != AG2V_F32 && ptype != dtype) return false;
    if (N <= 0 || S <= 0 || C <= 0 || groups <= 0 || C % groups || S >= (1 << 30) || C >= (1 << 30)) return false;
    return (long long)N * groups < (1LL << 24);
}

extern "C" size_t ag2v_group_norm_workspace_floats(int dtype, int N, int S, int C, int groups, int backward) {
    if (!sizes_ok(dtype, AG2V_F32, N, S, C, groups, ACT_NONE)) return 0;
    return (size_t)plan_of(dtype, N, S, C, groups, backward != 0).words;
}
extern "C" int ag2v_group_norm_fwd(int dtype, const void* x, long long x_sample, long long x_row, const void* weight, const void* bias,
                                   int param_dtype, void* y, float* mean, float* rstd, int N, int S, int C, int groups, float eps, int act,
                                   float slope, float* workspace, size_t workspace_floats, void* stream) {
    if (!x || !y || !mean || !rstd || !sizes_ok(dtype, param_dtype, N, S, C, groups, act) || !(eps >= 0.f)) return AG2V_EINVAL;
    GnArgs a = {};
    a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd; a.xs = x_sample; a.xr = x_row;
    a.N = N; a.S = S; a.C = C; a.G = groups; a.Cg = C / groups; a.ptype = param_dtype; a.eps = eps; a.slope = slope;
    return run_any(a, dtype, act, false, workspace, workspace_floats, (hipStream_t)stream);
}
extern "C" int ag2v_group_norm_bwd(int dtype, const void* dy, long long dy_sample, long long dy_row, const void* x, long long x_sample,
                                   long long x_row, const void* weight, const void* bias, int param_dtype, const float* mean,
                                   const float* rstd, void* dx, void* dweight, void* dbias, int N, int S, int C, int groups, int act,
                                   float slope, float* workspace, size_t workspace_floats, void* stream) {
    if (!x || !dy || !mean || !rstd || !sizes_ok(dtype, param_dtype, N, S, C, groups, act)) return AG2V_EINVAL;
    GnArgs a = {};
    a.x = x; a.dy = dy; a.w = weight; a.b = bias; a.y = dx; a.dw = dweight; a.db = dbias; a.mean = (float*)mean; a.rstd = (float*)rstd;
    a.xs = x_sample; a.xr = x_row; a.ds = dy_sample; a.dr = dy_row;
    a.N = N; a.S = S; a.C = C; a.G = groups; a.Cg = C / groups; a.ptype = param_dtype; a.slope = slope;
    return run_any(a, dtype, act, true, workspace, workspace_floats, (hipStream_t)stream);
}
