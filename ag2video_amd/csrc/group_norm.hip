// Group norm with an activation on channels-last maps, forward and backward.
//   x[N, S, C], G groups of Cg = C / G channels, M = S * Cg values per (sample, group):
//     h = (x - mean) * rstd      mean, biased variance over the group's S positions and Cg channels, rstd = 1 / sqrt(var + eps)
//     z = w h + b                y = act(z):  0 z,  1 z * sigmoid(z),  2 z > 0 ? z : slope * z
//   backward, dz = dy act'(z), A[n,c] = sum_s dz, B[n,c] = sum_s dz h:
//     db = sum_n A, dw = sum_n B, s1 = sum_{c in g} w A, s2 = sum_{c in g} w B, dx = rstd (w dz - (s1 + h s2) / M)
// Every sum is in fp32; z and h are computed again in the backward pass from x and the two statistics of a group.
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
    if (ACT == ACT_SILU) return z * __frcp_rn(1.f + __expf(-z));
    if (ACT == ACT_LRELU) return z > 0.f ? z : z * slope;
    return z;
}
// dy * act'(z)
template <int ACT>
__device__ __forceinline__ float act_bwd(float dy, float z, float slope) {
    if (ACT == ACT_SILU) {
        const float s = __frcp_rn(1.f + __expf(-z));
        return dy * (s * (1.f + z * (1.f - s)));
    }
    if (ACT == ACT_LRELU) return z > 0.f ? dy : dy * slope;
    return dy;
}

// ---------------------------------------------------------------- layout shared by the kernels
// A slab of channels (whole groups, or a tile of all channels) is walked as rows of 16-byte vectors: vector `col` of a row, `nv` of its
// elements inside the slab.  Per-thread sums meet in LDS as rows[slot][width]; group g's share is columns [g * wg, (g + 1) * wg) of every
// slot.  A vector lies inside one group where Cg is a multiple of the vector (then one value a thread, wg = vectors a group); elsewhere it
// may span groups, and a thread hands over one value per channel (wg = Cg).
//
// out[g] = sum of group g's share: 2^llg lanes a group, `threads` lanes in all.
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
// lanes a group in share_sums: a power of two, at most a wave
static int share_lanes(int threads, int ng) {
    int l = 0;
    while (l < 6 && (2 << l) * ng <= threads) ++l;
    return l;
}

// ---------------------------------------------------------------- one launch: a slab's values stay in registers
// T threads own all S positions of kg adjacent groups of one sample: U vectors a thread, read once.  Mean, then the squared deviations
// from it, then the result.  blockDim / T slabs a workgroup.
struct GnSlab {
    int T, kg, nsets, CVw, RS, llg;   // threads, groups, sets of groups a sample, vectors a row, rows at a time, log2 of lanes a group
    long long nslab;
};

template <class E, int ACT, int U, bool ONE>
__global__ __launch_bounds__(1024) void gn_slab_fwd_kernel(GnArgs a, GnSlab p) {
    extern __shared__ float shm[];
    constexpr int V = E::V, NG = ONE ? 1 : V;        // groups a vector may touch
    const int sub = threadIdx.x / p.T, t = threadIdx.x - sub * p.T, subs = blockDim.x / p.T;
    const int width = ONE ? p.CVw : p.CVw * V, wg = ONE ? p.CVw / p.kg : a.Cg;
    float* rows = shm + sub * (p.RS * width + 2 * p.kg);
    float* stat = rows + p.RS * width;
    const long long slab = (long long)xcd_remap(blockIdx.x, gridDim.x) * subs + sub;
    const bool live = slab < p.nslab;
    const int n = live ? (int)(slab / p.nsets) : 0, g0 = live ? (int)(slab - (long long)n * p.nsets) * p.kg : 0;
    const int ng = min(p.kg, a.G - g0), c0 = g0 * a.Cg, W = ng * a.Cg;
    const int rs = t / p.CVw, col = t - rs * p.CVw, nv = min(V, W - col * V);
    const bool on = live && rs < p.RS && nv > 0;
    const float inv = 1.f / ((float)a.S * (float)a.Cg);
    const typename E::T* x = (const typename E::T*)a.x + n * a.xs + c0 + col * V;
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = rs + u * p.RS;
        raw[u] = u32x4{0, 0, 0, 0};
        if (on && r < a.S) raw[u] = load_vec<E>(x + r * a.xr, nv);
    }
    float acc[V] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float v[V];
        E::unpack(raw[u], v);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += v[k];
    }
    auto hand_over = [&]() {
        if (!on) return;
        if (ONE) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < V; ++k) s += acc[k];
            rows[rs * width + col] = s;
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) rows[rs * width + col * V + k] = acc[k];
        }
    };
    hand_over();
    __syncthreads();
    if (live) share_sums(rows, p.RS, width, wg, ng, p.llg, t, p.T, stat);
    __syncthreads();
    float mean[NG];
    int gi[NG];
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        gi[k] = min(ONE ? col / wg : (col * V + k) / a.Cg, ng - 1);
        mean[k] = on ? stat[gi[k]] * inv : 0.f;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (rs + u * p.RS < a.S) {
            float v[V];
            E::unpack(raw[u], v);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = v[k] - mean[k % NG];
                acc[k] = fmaf(d, d, acc[k]);
            }
        }
    }
    __syncthreads();
    hand_over();
    __syncthreads();
    if (live) share_sums(rows, p.RS, width, wg, ng, p.llg, t, p.T, stat + p.kg);
    __syncthreads();
    if (live && t < ng) {
        a.mean[n * a.G + g0 + t] = stat[t] * inv;
        a.rstd[n * a.G + g0 + t] = 1.f / sqrtf(stat[p.kg + t] * inv + a.eps);
    }
    if (!on) return;
    float w[V], b[V], rstd[NG];
#pragma unroll
    for (int k = 0; k < NG; ++k) rstd[k] = 1.f / sqrtf(stat[p.kg + gi[k]] * inv + a.eps);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = c0 + col * V + k;
        w[k] = (a.w && k < nv ? load_any(a.w, a.ptype, c) : 1.f) * rstd[k % NG];
        b[k] = a.b && k < nv ? load_any(a.b, a.ptype, c) : 0.f;
    }
    typename E::T* y = (typename E::T*)a.y + (long long)n * a.S * a.C + c0 + col * V;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = rs + u * p.RS;
        if (r < a.S) {
            float v[V];
            E::unpack(raw[u], v);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = act_fwd<ACT>(fmaf(v[k] - mean[k % NG], w[k], b[k]), a.slope);
            store_vec<E>(y + (long long)r * a.C, nv, v);
        }
    }
}

// Backward on slabs: x and dy of a slab in registers.  A workgroup keeps its set of groups and walks samples, `walkers` apart, so that the
// parameters' gradients leave it once: ab[walker][C] = (sum dz, sum dz h) over its samples.  Vectors that span groups hold statistics per
// channel and half as many rows (512 threads, 256 registers each).
template <class E, int ACT, int U, bool ONE>
__global__ __launch_bounds__(ONE ? 1024 : 512) void gn_slab_bwd_kernel(GnArgs a, GnSlab p, int walkers, float2* ab) {
    extern __shared__ float shm[];
    constexpr int V = E::V, NG = ONE ? 1 : V;
    const int sub = threadIdx.x / p.T, t = threadIdx.x - sub * p.T, subs = blockDim.x / p.T;
    const int width = p.CVw * V, swidth = ONE ? p.CVw : width, wg = ONE ? p.CVw / p.kg : a.Cg;
    const int area = p.RS * (ONE ? width : 2 * width);           // two arrays of group sums while walking, one of channel sums at the end
    float* r1 = shm + sub * (area + 2 * p.kg);
    float* r2 = r1 + p.RS * swidth;
    float* stat = r1 + area;
    const int blk = xcd_remap(blockIdx.x, gridDim.x), set = blk % p.nsets, walker = blk / p.nsets * subs + sub;
    const int g0 = set * p.kg, ng = min(p.kg, a.G - g0), c0 = g0 * a.Cg, W = ng * a.Cg;
    const int rs = t / p.CVw, col = t - rs * p.CVw, nv = min(V, W - col * V);
    const bool on = rs < p.RS && nv > 0;
    const float inv = 1.f / ((float)a.S * (float)a.Cg);
    float w[V], b[V], A[V], B[V];
    int gi[NG];
#pragma unroll
    for (int k = 0; k < NG; ++k) gi[k] = min(ONE ? col / wg : (col * V + k) / a.Cg, ng - 1);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = c0 + col * V + k;
        w[k] = a.w && on && k < nv ? load_any(a.w, a.ptype, c) : 1.f;
        b[k] = a.b && on && k < nv ? load_any(a.b, a.ptype, c) : 0.f;
        A[k] = B[k] = 0.f;
    }
    for (int n0 = blk / p.nsets * subs; n0 < a.N; n0 += walkers) {
        const int n = n0 + sub;
        const bool live = n < a.N, here = on && live;
        u32x4 rx[U], rd[U];
        const typename E::T* x = (const typename E::T*)a.x + (long long)n * a.xs + c0 + col * V;
        const typename E::T* dy = (const typename E::T*)a.dy + (long long)n * a.ds + c0 + col * V;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = rs + u * p.RS;
            rx[u] = rd[u] = u32x4{0, 0, 0, 0};
            if (here && r < a.S) {
                rx[u] = load_vec<E>(x + r * a.xr, nv);
                rd[u] = load_vec<E>(dy + r * a.dr, nv);
            }
        }
        float mean[NG], rstd[NG], g1[NG] = {}, g2[NG] = {};     // g1, g2: sums of w dz and w dz h
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            mean[k] = here ? a.mean[(long long)n * a.G + g0 + gi[k]] : 0.f;
            rstd[k] = here ? a.rstd[(long long)n * a.G + g0 + gi[k]] : 0.f;
        }
        if (here) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (rs + u * p.RS < a.S) {
                    float v[V], d[V];
                    E::unpack(rx[u], v);
                    E::unpack(rd[u], d);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float h = (v[k] - mean[k % NG]) * rstd[k % NG], dz = act_bwd<ACT>(d[k], fmaf(h, w[k], b[k]), a.slope), e = w[k] * dz;
                        A[k] += dz;
                        B[k] = fmaf(dz, h, B[k]);
                        g1[k % NG] += e;
                        g2[k % NG] = fmaf(e, h, g2[k % NG]);
                    }
                }
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                r1[rs * swidth + (ONE ? col : col * V + k)] = g1[k];
                r2[rs * swidth + (ONE ? col : col * V + k)] = g2[k];
            }
        }
        __syncthreads();
        if (live && a.y) {
            share_sums(r1, p.RS, swidth, wg, ng, p.llg, t, p.T, stat);
            share_sums(r2, p.RS, swidth, wg, ng, p.llg, t, p.T, stat + p.kg);
        }
        __syncthreads();
        if (here && a.y) {
            typename E::T* dx = (typename E::T*)a.y + (long long)n * a.S * a.C + c0 + col * V;
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                g1[k] = stat[gi[k]] * inv;
                g2[k] = stat[p.kg + gi[k]] * inv;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = rs + u * p.RS;
                if (r < a.S) {
                    float v[V], d[V];
                    E::unpack(rx[u], v);
                    E::unpack(rd[u], d);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float h = (v[k] - mean[k % NG]) * rstd[k % NG], dz = act_bwd<ACT>(d[k], fmaf(h, w[k], b[k]), a.slope);
                        v[k] = rstd[k % NG] * (w[k] * dz - g1[k % NG] - h * g2[k % NG]);
                    }
                    store_vec<E>(dx + (long long)r * a.C, nv, v);
                }
            }
        }
    }
    if (!ab) return;
    // the channels' sums over the workgroup's rows, one array at a time in all of the rows' memory
    for (int half = 0; half < 2; ++half) {
        __syncthreads();
        if (on) {
#pragma unroll
            for (int k = 0; k < V; ++k) r1[rs * width + col * V + k] = half ? B[k] : A[k];
        }
        __syncthreads();
        for (int c = t; c < W; c += p.T) {
            float s = 0.f;
            for (int r = 0; r < p.RS; ++r) s += r1[r * width + c];
            (&ab[(long long)walker * a.C + c0 + c].x)[half] = s;
        }
    }
}

// ---------------------------------------------------------------- larger maps: sums of parts, a join, a second pass over the map
// A workgroup owns `rows` positions of one sample and a tile of CVt vectors of channels.
struct GnParts {
    int tiles, CVt, RS, rows, P, llg;    // P: parts a sample
};

// Every thread sums deviations from the first value it sees of each channel.  That value is one of the summed ones, so the sum of squares
// about it is at most (count + 1) times the one about the thread's mean: nothing cancels that matters, whatever the mean is.
// part[n][p * tiles + tile][g] = (count, mean, sum of squares about it)
template <class E>
__global__ __launch_bounds__(256) void gn_stats_kernel(GnArgs a, GnParts p, float* part) {
    __shared__ float r1[256 * E::V], r2[256 * E::V];
    __shared__ float gs[2][256];
    constexpr int V = E::V, U = 8;
    const int tile = blockIdx.x % p.tiles, np = blockIdx.x / p.tiles, n = np / p.P, q = np - n * p.P;
    const int rs = threadIdx.x / p.CVt, col = threadIdx.x - rs * p.CVt, c0 = tile * p.CVt * V, W = min(p.CVt * V, a.C - c0);
    const int nv = min(V, W - col * V);
    const bool on = rs < p.RS && nv > 0;
    const int lo = q * p.rows, hi = min(a.S, lo + p.rows);
    const typename E::T* x = (const typename E::T*)a.x + n * a.xs + c0 + col * V;
    float x0[V] = {}, s[V] = {}, m[V] = {};
    int cnt = 0;
    if (on && lo + rs < hi) {
        E::unpack(load_vec<E>(x + (lo + rs) * a.xr, nv), x0);
        for (int r = lo + rs; r < hi; r += U * p.RS) {
            u32x4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * p.RS < hi) raw[u] = load_vec<E>(x + (long long)(r + u * p.RS) * a.xr, nv);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * p.RS < hi) {
                    float v[V];
                    E::unpack(raw[u], v);
                    ++cnt;
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float d = v[k] - x0[k];
                        s[k] += d;
                        m[k] = fmaf(d, d, m[k]);
                    }
                }
        }
    }
    // per channel and slot: mean and squares about it; then the groups' means, then the squares about those
    const int width = p.CVt * V;
    float mean[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const float ds = cnt ? s[k] / (float)cnt : 0.f;
        mean[k] = x0[k] + ds;
        const float m2 = m[k] - s[k] * ds;
        m[k] = m2 < 0.f ? 0.f : m2;
        if (on) r1[rs * width + col * V + k] = mean[k] * (float)cnt;
    }
    __syncthreads();
    // groups whose channels lie (partly) in this tile
    const int gl = c0 / a.Cg, gh = (c0 + W - 1) / a.Cg;
    for (int g0 = gl; g0 <= gh; g0 += 256) {
        const int ng = min(256, gh - g0 + 1);
        // lanes a group: all threads shared over the groups, a power of two within a wave
        const int llg = p.llg, step = 1 << llg, l = threadIdx.x & (step - 1);
        for (int round = 0; round < 2; ++round) {
            for (int g = threadIdx.x >> llg; g < ng; g += 256 >> llg) {
                const int cl = max((g0 + g) * a.Cg - c0, 0), wg = min((g0 + g + 1) * a.Cg - c0, W) - cl;
                float t = 0.f;
                for (int e = l; e < p.RS * wg; e += step) {
                    const int r = e / wg, c = e - r * wg;
                    t += (round ? r2 : r1)[r * width + cl + c];
                }
                for (int o = step >> 1; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
                if (l == 0) gs[round][g] = t;
            }
            __syncthreads();
            if (round == 0) {
                const int slots = min(p.RS, hi - lo);
                const float rows = (float)(hi - lo);
                if (on && rs < slots) {
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const int g = (c0 + col * V + k) / a.Cg - g0;
                        if (k < nv && g >= 0 && g < ng) {
                            const int cl = max((g0 + g) * a.Cg - c0, 0), wg = min((g0 + g + 1) * a.Cg - c0, W) - cl;
                            const float d = mean[k] - gs[0][g] / (rows * (float)wg);
                            r2[rs * width + col * V + k] = fmaf(d * d, (float)cnt, m[k]);
                        }
                    }
                } else if (on) {
#pragma unroll
                    for (int k = 0; k < V; ++k) r2[rs * width + col * V + k] = 0.f;
                }
                __syncthreads();
            }
        }
        for (int g = threadIdx.x; g < ng; g += 256) {
            const int cl = max((g0 + g) * a.Cg - c0, 0), wg = min((g0 + g + 1) * a.Cg - c0, W) - cl;
            const float count = (float)(hi - lo) * (float)wg;
            float* o = part + (((long long)n * p.P + q) * p.tiles + tile) * a.G * 3 + (long long)(g0 + g) * 3;
            o[0] = count;
            o[1] = gs[0][g] / count;
            o[2] = gs[1][g];
        }
        __syncthreads();
    }
    for (int g = threadIdx.x; g < a.G; g += 256)
        if (g < gl || g > gh) part[((((long long)n * p.P + q) * p.tiles + tile) * a.G + g) * 3] = 0.f;
}

// A wave per (sample, group): the parts' means and squares joined pairwise, in fp64.
__global__ __launch_bounds__(256) void gn_stats_join_kernel(GnArgs a, int parts, const float* part) {
    const int ngroups = a.N * a.G, id = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63;
    if (id >= ngroups) return;
    const int n = id / a.G, g = id - n * a.G;
    double cnt = 0.0, mean = 0.0, m2 = 0.0;
    auto join = [&](double cb, double mb, double qb) {
        if (cb == 0.0) return;
        const double c = cnt + cb, d = mb - mean;
        mean += d * (cb / c);
        m2 += qb + d * d * (cnt * cb / c);
        cnt = c;
    };
    for (int i = l; i < parts; i += 64) {
        const float* o = part + (((long long)n * parts + i) * a.G + g) * 3;
        join(o[0], o[1], o[2]);
    }
    for (int o = 32; o > 0; o >>= 1) {
        const double cb = __shfl_xor(cnt, o, 64), mb = __shfl_xor(mean, o, 64), qb = __shfl_xor(m2, o, 64);
        // both partners form the same pair in the same order
        if (l & o) {
            const double c1 = cnt, m1 = mean, q1 = m2;
            cnt = cb; mean = mb; m2 = qb;
            join(c1, m1, q1);
        } else {
            join(cb, mb, qb);
        }
    }
    if (l == 0) {
        a.mean[id] = (float)mean;
        a.rstd[id] = (float)(1.0 / sqrt(m2 / cnt + (double)a.eps));
    }
}

template <class E, int ACT>
__global__ __launch_bounds__(256) void gn_apply_kernel(GnArgs a, GnParts p) {
    constexpr int V = E::V, U = 4;
    const int tile = blockIdx.x % p.tiles, np = blockIdx.x / p.tiles, n = np / p.P, q = np - n * p.P;
    const int rs = threadIdx.x / p.CVt, col = threadIdx.x - rs * p.CVt, c0 = tile * p.CVt * V, W = min(p.CVt * V, a.C - c0);
    const int nv = min(V, W - col * V), lo = q * p.rows, hi = min(a.S, lo + p.rows);
    if (rs >= p.RS || nv <= 0) return;
    float mean[V], w[V], b[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = min(c0 + col * V + k, a.C - 1), g = n * a.G + c / a.Cg;
        mean[k] = a.mean[g];
        w[k] = (a.w ? load_any(a.w, a.ptype, c) : 1.f) * a.rstd[g];
        b[k] = a.b ? load_any(a.b, a.ptype, c) : 0.f;
    }
    const typename E::T* x = (const typename E::T*)a.x + n * a.xs + c0 + col * V;
    typename E::T* y = (typename E::T*)a.y + (long long)n * a.S * a.C + c0 + col * V;
    for (int r = lo + rs; r < hi; r += U * p.RS) {
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * p.RS < hi) raw[u] = load_vec<E>(x + (long long)(r + u * p.RS) * a.xr, nv);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * p.RS < hi) {
                float v[V];
                E::unpack(raw[u], v);
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = act_fwd<ACT>(fmaf(v[k] - mean[k], w[k], b[k]), a.slope);
                store_vec<E>(y + (long long)(r + u * p.RS) * a.C, nv, v);
            }
    }
}

// part[n][p][c] = (sum dz, sum dz h) over the part's positions
template <class E, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(GnArgs a, GnParts p, float2* part) {
    __shared__ float r1[256 * E::V], r2[256 * E::V];
    constexpr int V = E::V, U = 4;
    const int tile = blockIdx.x % p.tiles, np = blockIdx.x / p.tiles, n = np / p.P, q = np - n * p.P;
    const int rs = threadIdx.x / p.CVt, col = threadIdx.x - rs * p.CVt, c0 = tile * p.CVt * V, W = min(p.CVt * V, a.C - c0);
    const int nv = min(V, W - col * V), lo = q * p.rows, hi = min(a.S, lo + p.rows);
    const bool on = rs < p.RS && nv > 0;
    float A[V] = {}, B[V] = {};
    if (on) {
        float mean[V], rstd[V], w[V], b[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = min(c0 + col * V + k, a.C - 1), g = n * a.G + c / a.Cg;
            mean[k] = a.mean[g];
            rstd[k] = a.rstd[g];
            w[k] = a.w ? load_any(a.w, a.ptype, c) : 1.f;
            b[k] = a.b ? load_any(a.b, a.ptype, c) : 0.f;
        }
        const typename E::T* x = (const typename E::T*)a.x + n * a.xs + c0 + col * V;
        const typename E::T* dy = (const typename E::T*)a.dy + n * a.ds + c0 + col * V;
        for (int r = lo + rs; r < hi; r += U * p.RS) {
            u32x4 rx[U], rd[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * p.RS < hi) {
                    rx[u] = load_vec<E>(x + (long long)(r + u * p.RS) * a.xr, nv);
                    rd[u] = load_vec<E>(dy + (long long)(r + u * p.RS) * a.dr, nv);
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * p.RS < hi) {
                    float v[V], d[V];
                    E::unpack(rx[u], v);
                    E::unpack(rd[u], d);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float h = (v[k] - mean[k]) * rstd[k], dz = act_bwd<ACT>(d[k], fmaf(h, w[k], b[k]), a.slope);
                        A[k] += dz;
                        B[k] = fmaf(dz, h, B[k]);
                    }
                }
        }
    }
    const int width = p.CVt * V;
    if (on) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            r1[rs * width + col * V + k] = A[k];
            r2[rs * width + col * V + k] = B[k];
        }
    }
    __syncthreads();
    // lanes share a channel's slots where channels are few
    const int step = 1 << p.llg, l = threadIdx.x & (step - 1);
    for (int c = threadIdx.x >> p.llg; c < W; c += 256 >> p.llg) {
        float s = 0.f, t = 0.f;
        for (int r = l; r < p.RS; r += step) {
            s += r1[r * width + c];
            t += r2[r * width + c];
        }
        for (int o = step >> 1; o > 0; o >>= 1) {
            s += __shfl_xor(s, o, 64);
            t += __shfl_xor(t, o, 64);
        }
        if (l == 0) part[((long long)n * p.P + q) * a.C + c0 + c] = make_float2(s, t);
    }
}

// A workgroup per (sample, group): the parts of its channels, in order; ab[n][c], and the group's (s1 / M, s2 / M) to coef[n][g].
__global__ __launch_bounds__(256) void gn_bwd_join_kernel(GnArgs a, int P, int lcw, const float2* part, float2* ab, float2* coef) {
    __shared__ float2 sh[256];
    const int n = blockIdx.x / a.G, g = blockIdx.x - n * a.G;
    const int cw = 1 << lcw, slots = 256 >> lcw, slot = threadIdx.x >> lcw, cl = threadIdx.x & (cw - 1);
    float s1 = 0.f, s2 = 0.f;
    for (int c0 = 0; c0 < a.Cg; c0 += cw) {
        const int c = g * a.Cg + c0 + cl;
        float2 v = make_float2(0.f, 0.f);
        if (c0 + cl < a.Cg)
            for (int q = slot; q < P; q += slots) {
                const float2 o = part[((long long)n * P + q) * a.C + c];
                v.x += o.x;
                v.y += o.y;
            }
        sh[threadIdx.x] = v;
        __syncthreads();
        if (slot == 0 && c0 + cl < a.Cg) {
            for (int q = 1; q < slots; ++q) {
                const float2 o = sh[(q << lcw) + cl];
                v.x += o.x;
                v.y += o.y;
            }
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

template <class E, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_dx_kernel(GnArgs a, GnParts p, const float2* coef) {
    constexpr int V = E::V, U = 4;
    const int tile = blockIdx.x % p.tiles, np = blockIdx.x / p.tiles, n = np / p.P, q = np - n * p.P;
    const int rs = threadIdx.x / p.CVt, col = threadIdx.x - rs * p.CVt, c0 = tile * p.CVt * V, W = min(p.CVt * V, a.C - c0);
    const int nv = min(V, W - col * V), lo = q * p.rows, hi = min(a.S, lo + p.rows);
    if (rs >= p.RS || nv <= 0) return;
    float mean[V], rstd[V], w[V], b[V], s1[V], s2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = min(c0 + col * V + k, a.C - 1), g = n * a.G + c / a.Cg;
        mean[k] = a.mean[g];
        rstd[k] = a.rstd[g];
        w[k] = a.w ? load_any(a.w, a.ptype, c) : 1.f;
        b[k] = a.b ? load_any(a.b, a.ptype, c) : 0.f;
        s1[k] = coef[g].x;
        s2[k] = coef[g].y;
    }
    const typename E::T* x = (const typename E::T*)a.x + n * a.xs + c0 + col * V;
    const typename E::T* dy = (const typename E::T*)a.dy + n * a.ds + c0 + col * V;
    typename E::T* dx = (typename E::T*)a.y + (long long)n * a.S * a.C + c0 + col * V;
    for (int r = lo + rs; r < hi; r += U * p.RS) {
        u32x4 rx[U], rd[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * p.RS < hi) {
                rx[u] = load_vec<E>(x + (long long)(r + u * p.RS) * a.xr, nv);
                rd[u] = load_vec<E>(dy + (long long)(r + u * p.RS) * a.dr, nv);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * p.RS < hi) {
                float v[V], d[V];
                E::unpack(rx[u], v);
                E::unpack(rd[u], d);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float h = (v[k] - mean[k]) * rstd[k], dz = act_bwd<ACT>(d[k], fmaf(h, w[k], b[k]), a.slope);
                    v[k] = rstd[k] * (w[k] * dz - s1[k] - h * s2[k]);
                }
                store_vec<E>(dx + (long long)(r + u * p.RS) * a.C, nv, v);
            }
    }
}

// dw, db: 32 channels a workgroup, 8 lanes a channel share its `rows` partial sums.
__global__ __launch_bounds__(256) void gn_params_kernel(GnArgs a, int rows, const float2* ab) {
    __shared__ float2 sh[256];
    const int cl = threadIdx.x & 31, slot = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
    float2 v = make_float2(0.f, 0.f);
    if (c < a.C)
        for (int r = slot; r < rows; r += 8) {
            const float2 o = ab[(long long)r * a.C + c];
            v.x += o.x;
            v.y += o.y;
        }
    sh[threadIdx.x] = v;
    __syncthreads();
    if (slot == 0 && c < a.C) {
        for (int q = 1; q < 8; ++q) {
            v.x += sh[q * 32 + cl].x;
            v.y += sh[q * 32 + cl].y;
        }
        if (a.dw) store_any(a.dw, a.ptype, c, v.y);
        if (a.db) store_any(a.db, a.ptype, c, v.x);
    }
}

// ---------------------------------------------------------------- host
static int vec_of(int dtype) { return dtype == AG2V_F32 ? ElemF32::V : ElemBF16::V; }

// Which way (N, S, C, G) runs, forward or backward.
struct GnPlan {
    bool slab, one;                  // one: a vector lies inside one group
    GnSlab s;
    int U, threads, blocks, walkers;
    size_t lds;
    GnParts p;
    long long words, ab, coef;       // workspace in floats; offsets of ab[][C] and coef[N][G] in it
};
static GnPlan plan_of(int dtype, int N, int S, int C, int G, bool backward) {
    GnPlan r = {};
    const int V = vec_of(dtype), Cg = C / G;
    const bool one = Cg % V == 0;
    const int maxT = backward && !one ? 512 : 1024, maxU = !backward ? 8 : one ? 4 : 2;
    // groups of a slab: rows of 128 bytes where that fits, so that slabs share no cache line
    int kg = 1;
    auto vecs = [&](int k) { return ((long long)k * Cg + V - 1) / V; };
    while (kg < G && vecs(kg) < 128 / 16 && (long long)S * vecs(kg + 1) <= maxT * maxU) ++kg;
    const long long cv = vecs(kg), total = (long long)S * cv;
    if (cv <= maxT && total <= (long long)maxT * maxU) {
        int T = 64;
        while (T < maxT && ((long long)T * (maxU < 4 ? maxU : 4) < total || T < cv)) T *= 2;
        const int RS = T / (int)cv;
        const int U = (S + RS - 1) / RS;
        if (U <= maxU) {
            r.slab = true;
            r.s.T = T;
            r.s.kg = kg;
            r.s.nsets = (G + kg - 1) / kg;
            r.s.CVw = (int)cv;
            r.s.RS = RS;
            r.s.llg = share_lanes(T, kg);
            r.one = one;
            r.s.nslab = (long long)N * r.s.nsets;
            r.U = U <= 1 ? 1 : U <= 2 ? 2 : U <= 4 ? 4 : 8;
            r.threads = T < 256 ? 256 : T;
            const int subs = r.threads / T, width = (int)cv * (one && !backward ? 1 : V);
            r.lds = sizeof(float) * subs * ((backward && !one ? 2 : 1) * (size_t)RS * width + 2 * kg);
            if (!backward) {
                const long long b = (r.s.nslab + subs - 1) / subs;
                if (b >= (1LL << 22)) { r.slab = false; } else r.blocks = (int)b;
            } else {
                long long wb = ((long long)N + subs - 1) / subs;
                const long long most = 2048 / r.s.nsets < 1 ? 1 : 2048 / r.s.nsets;
                if (wb > most) wb = most;
                r.walkers = (int)wb * subs;
                if (wb * r.s.nsets >= (1LL << 22)) r.slab = false; else r.blocks = (int)(wb * r.s.nsets);
                r.words = 2LL * r.walkers * C;
            }
            if (r.lds > 64 * 1024) r.slab = false;
            if (r.slab) return r;
        }
    }
    r = GnPlan();
    GnParts& p = r.p;
    const long long cvs = ((long long)C + V - 1) / V;
    p.tiles = (int)((cvs + 255) / 256);
    p.CVt = (int)((cvs + p.tiles - 1) / p.tiles);
    p.RS = 256 / p.CVt;
    // 8 positions a thread, more where a sample would have over 512 parts.  By the sample's own sizes alone: its result is the same, bit for
    // bit, in a batch of any size.
    long long P = (S + 8LL * p.RS - 1) / (8LL * p.RS);
    if (P > 512) P = 512;
    p.rows = (int)((S + P - 1) / P);
    p.P = (S + p.rows - 1) / p.rows;
    if (backward) {
        p.llg = share_lanes(256, p.CVt * V);
        r.ab = 2LL * N * p.P * C;
        r.coef = r.ab + 2LL * N * C;
        r.words = r.coef + 2LL * N * G;
    } else {
        const long long per = ((long long)p.CVt * V + Cg - 1) / Cg + 1;
        p.llg = share_lanes(256, (int)(per < G ? per : G));
        r.words = 3LL * N * p.P * p.tiles * G;
    }
    return r;
}

template <class E, int ACT, bool ONE>
static int run_slab_fwd(const GnArgs& a, const GnPlan& r, hipStream_t st) {
    const dim3 grid(r.blocks), block(r.threads);
    if (r.U == 1) hipLaunchKernelGGL((gn_slab_fwd_kernel<E, ACT, 1, ONE>), grid, block, r.lds, st, a, r.s);
    else if (r.U == 2) hipLaunchKernelGGL((gn_slab_fwd_kernel<E, ACT, 2, ONE>), grid, block, r.lds, st, a, r.s);
    else if (r.U == 4) hipLaunchKernelGGL((gn_slab_fwd_kernel<E, ACT, 4, ONE>), grid, block, r.lds, st, a, r.s);
    else hipLaunchKernelGGL((gn_slab_fwd_kernel<E, ACT, 8, ONE>), grid, block, r.lds, st, a, r.s);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
template <class E, int ACT, bool ONE>
static int run_slab_bwd(const GnArgs& a, const GnPlan& r, float2* ab, hipStream_t st) {
    const dim3 grid(r.blocks), block(r.threads);
    if (r.U == 1) hipLaunchKernelGGL((gn_slab_bwd_kernel<E, ACT, 1, ONE>), grid, block, r.lds, st, a, r.s, r.walkers, ab);
    else if (r.U == 2 || !ONE) hipLaunchKernelGGL((gn_slab_bwd_kernel<E, ACT, 2, ONE>), grid, block, r.lds, st, a, r.s, r.walkers, ab);
    else if constexpr (ONE) hipLaunchKernelGGL((gn_slab_bwd_kernel<E, ACT, 4, true>), grid, block, r.lds, st, a, r.s, r.walkers, ab);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
template <class E, int ACT>
static int run_fwd(const GnArgs& a, const GnPlan& r, float* ws, hipStream_t st) {
    if (r.slab) return r.one ? run_slab_fwd<E, ACT, true>(a, r, st) : run_slab_fwd<E, ACT, false>(a, r, st);
    const int blocks = a.N * r.p.P * r.p.tiles;
    hipLaunchKernelGGL(gn_stats_kernel<E>, dim3(blocks), dim3(256), 0, st, a, r.p, ws);
    AG2V_CHECK_LAUNCH();
    hipLaunchKernelGGL(gn_stats_join_kernel, dim3(ceil_div((long long)a.N * a.G, 4)), dim3(256), 0, st, a, r.p.P * r.p.tiles, ws);
    AG2V_CHECK_LAUNCH();
    hipLaunchKernelGGL((gn_apply_kernel<E, ACT>), dim3(blocks), dim3(256), 0, st, a, r.p);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}
template <class E, int ACT>
static int run_bwd(const GnArgs& a, const GnPlan& r, float* ws, hipStream_t st) {
    const bool params = a.dw || a.db;
    int rows = a.N;
    const float2* ab = (const float2*)ws;
    if (r.slab) {
        float2* out = params ? (float2*)ws : nullptr;
        const int rc = r.one ? run_slab_bwd<E, ACT, true>(a, r, out, st) : run_slab_bwd<E, ACT, false>(a, r, out, st);
        if (rc != AG2V_OK) return rc;
        rows = r.walkers;
    } else {
        float2 *part = (float2*)ws, *sums = (float2*)(ws + r.ab), *coef = (float2*)(ws + r.coef);
        const int blocks = a.N * r.p.P * r.p.tiles;
        hipLaunchKernelGGL((gn_bwd_sums_kernel<E, ACT>), dim3(blocks), dim3(256), 0, st, a, r.p, part);
        AG2V_CHECK_LAUNCH();
        int lcw = 0;
        while (lcw < 8 && (1 << lcw) < a.Cg) ++lcw;
        hipLaunchKernelGGL(gn_bwd_join_kernel, dim3(a.N * a.G), dim3(256), 0, st, a, r.p.P, lcw, part, sums, coef);
        AG2V_CHECK_LAUNCH();
        if (a.y) hipLaunchKernelGGL((gn_bwd_dx_kernel<E, ACT>), dim3(blocks), dim3(256), 0, st, a, r.p, coef);
        AG2V_CHECK_LAUNCH();
        ab = sums;
    }
    if (params) {
        hipLaunchKernelGGL(gn_params_kernel, dim3(ceil_div(a.C, 32)), dim3(256), 0, st, a, rows, ab);
        AG2V_CHECK_LAUNCH();
    }
    return AG2V_OK;
}
template <class E>
static int run_elem(const GnArgs& a, const GnPlan& r, int act, bool backward, float* ws, hipStream_t st) {
    if (act == ACT_SILU) return backward ? run_bwd<E, ACT_SILU>(a, r, ws, st) : run_fwd<E, ACT_SILU>(a, r, ws, st);
    if (act == ACT_LRELU) return backward ? run_bwd<E, ACT_LRELU>(a, r, ws, st) : run_fwd<E, ACT_LRELU>(a, r, ws, st);
    return backward ? run_bwd<E, ACT_NONE>(a, r, ws, st) : run_fwd<E, ACT_NONE>(a, r, ws, st);
}
static int run_any(const GnArgs& a, int dtype, int act, bool backward, float* ws, size_t ws_floats, hipStream_t st) {
    const GnPlan r = plan_of(dtype, a.N, a.S, a.C, a.G, backward);
    if ((r.words && !ws) || ws_floats < (size_t)r.words || ((uintptr_t)ws & 7)) return AG2V_EINVAL;
    if (!r.slab && (long long)a.N * r.p.P * r.p.tiles >= (1LL << 24)) return AG2V_EINVAL;
    if (dtype == AG2V_F32) return run_elem<ElemF32>(a, r, act, backward, ws, st);
    return dtype == AG2V_BF16 ? run_elem<ElemBF16>(a, r, act, backward, ws, st) : run_elem<ElemF16>(a, r, act, backward, ws, st);
}

static bool sizes_ok(int dtype, int ptype, int N, int S, int C, int groups, int act) {
    if (dtype < AG2V_F32 || dtype > AG2V_F16 || ptype < AG2V_F32 || ptype > AG2V_F16 || act < ACT_NONE || act > ACT_LRELU) return false;
    if (N <= 0 || S <= 0 || C <= 0 || groups <= 0 || C % groups) return false;
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
