// Embedding lookup with scaling, and its gradient by sorted tokens.
//   out[i, :] = scale * table[idx_i, :]          dtable[v, :] = scale * sum over {i : idx_i = v} of dout[i, :]
// A token outside [0, V) reads nothing: its row of the output is NaN, and it takes part in no sum; neither does padding_idx.  Products
// and sums are in fp32 and rounded once.
//
// Both directions move memory and compute nothing to speak of: the lookup reads n rows (from the caches, where tokens repeat) and writes
// n rows; the gradient reads n rows and writes V.
//
// The gradient, by sizes:
//   few rows, few tokens    one launch: a workgroup per row of the table picks its tokens out of all n (embed_pick_kernel);
//   few rows                one workgroup sorts a tile of tokens in LDS and sums its rows by token; a second launch adds the tiles' sums
//                           (embed_tile_kernel, embed_tile_join_kernel);
//   up to RANK_MAX tokens   a token's place in the sorted order is the number of tokens before it: n^2 compares, spread over the whole
//                           chip in ONE launch that also clears the table's gradient (embed_rank_kernel);
//   more                    a stable radix sort, 9 bits a pass, two launches a pass (embed_hist_kernel, embed_scatter_kernel).
// After a sort of all tokens, embed_sum_kernel walks equal shares of the sorted order -- a long run of one token costs no more than many short ones --
// and writes every row whose tokens lie inside one workgroup's share; embed_join_kernel adds the rest up, in order.  No atomics on
// floating-point values: equal calls give equal bits.
// Figures below: one MI355X, medians of a kernel trace; a 1 GiB copy reads and writes 5.1 TB/s there.
#include "elem.h"

__device__ __forceinline__ long long token_at(const void* idx, int wide, long long stride, long long i) {
    return wide ? ((const long long*)idx)[i * stride] : (long long)((const int*)idx)[i * stride];
}
// sort key of a token: V for the ones that take part in no sum
__device__ __forceinline__ int key_at(const void* idx, int wide, long long stride, long long i, int V, int pad) {
    const long long v = token_at(idx, wide, stride, i);
    return v >= 0 && v < V && v != pad ? (int)v : V;
}

// The last vector of a row whose width is no multiple of V ends with the row: the elements it shares with the vector before are written
// twice, with the same bits.  They are sums in one order and one product, and the product is rounded to fp32 before the conversion (the
// compiler would fuse the two for some elements of a vector and not for others).
template <class E, bool NT = false>
__device__ __forceinline__ void store_row(typename E::T* p, int width, const float (&x)[E::V]) {
    float v[E::V];
#pragma unroll
    for (int k = 0; k < E::V; ++k) {
        v[k] = x[k];
        asm volatile("" : "+v"(v[k]));
    }
    store_vec<E, NT>(p, width, v);
}

// acc of group 0 += acc of all other groups of 2^lsh lanes, pairwise; sh: V floats a thread.  All threads of the workgroup.
template <int V, int THREADS>
__device__ __forceinline__ void join_groups(float (&acc)[V], float* sh, int lsh) {
    const int grp = threadIdx.x >> lsh;
#pragma unroll
    for (int k = 0; k < V; ++k) sh[k * THREADS + threadIdx.x] = acc[k];
    for (int o = (THREADS >> lsh) >> 1; o > 0; o >>= 1) {
        __syncthreads();
        if (grp < o) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                acc[k] += sh[k * THREADS + threadIdx.x + (o << lsh)];
                sh[k * THREADS + threadIdx.x] = acc[k];
            }
        }
    }
}

// ---------------------------------------------------------------- lookup
// 2^lsh lanes a row, 16 bytes a lane, four rows in flight a thread.  The last vector of a row whose width is no multiple of the vector
// moves back to end with the row (store_row).  134 MB of 27 words' rows (bf16, 128 wide) in 23 us, 5.8 TB/s written: memory.  102 MB of 50001 words'
// (fp16, 389 wide) in 27 us: the rows' reads, which the caches serve in part, come on top.  Ten rows in 2.0 us: the launch.
template <class E, bool NT>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* __restrict__ idx, int wide, long long istride,
                                                        const typename E::T* __restrict__ table, long long tstride,
                                                        typename E::T* __restrict__ out, long long n, int V, int D, float scale, int lsh) {
    constexpr int U = 4;
    const int lane = threadIdx.x & ((1 << lsh) - 1), grp = threadIdx.x >> lsh, ng = 256 >> lsh;
    for (long long i0 = (long long)blockIdx.x * ng * U + grp; i0 < n; i0 += (long long)gridDim.x * ng * U) {
        long long row[U];
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long i = i0 + u * ng;
            const long long v = i < n ? token_at(idx, wide, istride, i) : 0;
            in[u] = v >= 0 && v < V;
            row[u] = (in[u] ? v : 0) * tstride;
        }
        for (int c0 = lane * E::V; c0 < D; c0 += E::V << lsh) {
            const int c = D < E::V ? 0 : min(c0, D - E::V);
            u32x4 r[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * ng < n) r[u] = load_vec<E>(table + row[u] + c, D);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float v[E::V];
                E::unpack(r[u], v);
#pragma unroll
                for (int k = 0; k < E::V; ++k) v[k] = in[u] ? v[k] * scale : __builtin_nanf("");
                if (i0 + u * ng < n) store_row<E, NT>(out + (i0 + u * ng) * D + c, D, v);
            }
        }
    }
}

// ---------------------------------------------------------------- gradient: one launch for few rows and few tokens
// 1280 tokens of 24 words, 128 fp32: 5.0 us, bound by the chain tokens - list - rows - join.
#define PICK_MAX 2048
#define PICK_THREADS 1024
template <class E>
__global__ __launch_bounds__(PICK_THREADS) void embed_pick_kernel(const void* __restrict__ idx, int wide, long long istride,
                                                         const typename E::T* __restrict__ dout, long long dstride,
                                                         typename E::T* __restrict__ dtable, int n, int V, int D, float scale, int pad, int lsh) {
    constexpr int W = PICK_THREADS / 64, U = 8;
    __shared__ int list[PICK_MAX], found[W];
    __shared__ float part[PICK_THREADS * E::V];
    const int v = blockIdx.x % V, slice = blockIdx.x / V;
    const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63;
    // each wave finds the tokens of its share; their places in the list follow from the waves before
    const int share_n = (n + W - 1) / W, lo = wave * share_n, hi = min(n, lo + share_n);      // at most 128
    unsigned long long m[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int i = lo + q * 64 + wl;
        m[q] = __ballot(i < hi && key_at(idx, wide, istride, i, V, pad) == v);
    }
    if (wl == 0) found[wave] = __popcll(m[0]) + __popcll(m[1]);
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        before += w < wave ? found[w] : 0;
        total += found[w];
    }
    const unsigned long long below = (1ull << wl) - 1;
    if ((m[0] >> wl) & 1) list[before + __popcll(m[0] & below)] = lo + wl;
    if ((m[1] >> wl) & 1) list[before + __popcll(m[0]) + __popcll(m[1] & below)] = lo + 64 + wl;
    __syncthreads();
    const int lane = threadIdx.x & ((1 << lsh) - 1), grp = threadIdx.x >> lsh, ng = PICK_THREADS >> lsh;
    const int c0 = (slice << lsh) * E::V + lane * E::V, c = D < E::V ? 0 : min(c0, D - E::V);
    const int share = (total + ng - 1) / ng, e1 = min(total, (grp + 1) * share);
    float acc[E::V] = {};
    if (c0 < D)
        for (int e = grp * share; e < e1; e += U) {
            u32x4 r[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (e + u < e1) r[u] = load_vec<E>(dout + list[e + u] * dstride + c, D);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (e + u < e1) {
                    float x[E::V];
                    E::unpack(r[u], x);
#pragma unroll
                    for (int k = 0; k < E::V; ++k) acc[k] += x[k];
                }
        }
    join_groups<E::V, PICK_THREADS>(acc, part, lsh);
    if (grp == 0 && c0 < D) {
#pragma unroll
        for (int k = 0; k < E::V; ++k) acc[k] *= scale;
        store_row<E>(dtable + (long long)v * D + c, D, acc);
    }
}

// V of the D floats at p
template <int V>
__device__ __forceinline__ void load_part(const float* p, int D, float (&v)[V]) {
    if (D >= V) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const u32x4 r = *reinterpret_cast<const u32x4_a4*>(p + k);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k + j] = __uint_as_float(r[j]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = k < D ? p[k] : 0.f;
    }
}
template <int V>
__device__ __forceinline__ void store_part(float* p, int D, const float (&v)[V]) {
    if (D >= V) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            u32x4 r;
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = __float_as_uint(v[k + j]);
            *reinterpret_cast<u32x4_a4*>(p + k) = r;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < D) p[k] = v[k];
    }
}

// ---------------------------------------------------------------- gradient: tiles of tokens, for few rows
// A workgroup sorts T tokens by counting (ranks within a wave by matching the keys' bits over ballots, then over waves), its groups of lanes
// walk equal shares of the sorted tile as in embed_sum_kernel below, and the sum of each token that occurs goes to part[tile][token][:],
// count[tile][token] says how often it does.  No pass over the tokens but this one.  131072 tokens of 27 words, 128 fp32 (67 MB): 22.6 us, 3.0 TB/s,
// and 4.1 us for the join; 2 workgroups of 32 groups a CU have eight rows a group in flight, and the sort (some 4 us) is not hidden.
#define TILE_THREADS 512
#define TILE_MIN 512
#define TILE_MAX 2048
#define TILE_BITS 9
// More tiles than this are joined by 1024 threads in groups of 16 lanes, fewer by 256 in groups of up to 64: 5 tiles of 89 rows, 1400 wide, took
// 27 us a training pass so and 40 the other way; 256 tiles of 27 rows, 128 wide, 4.1 us a join and 5.4 in wider groups.
#define TILE_JOIN_WIDE 64
struct TileArgs {
    const void *idx, *dout;
    void* dtable;
    int* count;
    float* part;
    long long istride, dstride;
    int wide, n, V, D, pad, lsh, jlsh, T, bits, tiles;
    float scale;
};
template <class E, bool NT>
__global__ __launch_bounds__(TILE_THREADS) void embed_tile_kernel(TileArgs a) {
    constexpr int U = 8, PER = TILE_MAX / TILE_THREADS, W = TILE_THREADS / 64, DIG = 1 << TILE_BITS;
    static_assert(DIG == TILE_THREADS, "a thread scans one key");
    __shared__ int cnt[W][DIG], wsum[W], flags[TILE_THREADS / 8];
    __shared__ unsigned short skey[TILE_MAX], spos[TILE_MAX];
    __shared__ float head[TILE_THREADS * E::V];
    const int tile = blockIdx.x % a.tiles, slice = blockIdx.x / a.tiles, t0 = tile * a.T;
    const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63, rounds = a.T / TILE_THREADS, own = a.T / W;
#pragma unroll
    for (int w = 0; w < W; ++w) cnt[w][threadIdx.x] = 0;
    int key[PER], rank[PER];
#pragma unroll
    for (int q = 0; q < PER; ++q)
        if (q < rounds) {
            const int i = t0 + wave * own + q * 64 + wl;
            key[q] = i < a.n ? key_at(a.idx, a.wide, a.istride, i, a.V, a.pad) : a.V;
        }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < PER; ++q)
        if (q < rounds) {
            unsigned long long m = ~0ull;
            for (int b = 0; b < a.bits; ++b) {
                const bool bit = (key[q] >> b) & 1;
                const unsigned long long same = __ballot(bit);
                m &= bit ? same : ~same;
            }
            const int lower = __popcll(m & ((1ull << wl) - 1)), seen = cnt[wave][key[q]];
            __builtin_amdgcn_wave_barrier();
            if (lower == 0) cnt[wave][key[q]] = seen + __popcll(m);
            __builtin_amdgcn_wave_barrier();
            rank[q] = seen + lower;
        }
    __syncthreads();
    // exclusive sums over keys, then waves
    {
        const int d = threadIdx.x;
        int c[W], all = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            c[w] = cnt[w][d];
            all += c[w];
        }
        if (slice == 0 && d < a.V) a.count[tile * a.V + d] = all;
        int scan = all;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(scan, o, 64);
            if (wl >= o) scan += up;
        }
        if (wl == 63) wsum[wave] = scan;
        __syncthreads();
        for (int w = 0; w < wave; ++w) scan += wsum[w];
        int run = scan - all;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            cnt[w][d] = run;
            run += c[w];
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < PER; ++q)
        if (q < rounds) {
            const int at = cnt[wave][key[q]] + rank[q];
            skey[at] = (unsigned short)key[q];
            spos[at] = (unsigned short)(wave * own + q * 64 + wl);
        }
    __syncthreads();
    const int lane = threadIdx.x & ((1 << a.lsh) - 1), grp = threadIdx.x >> a.lsh, ng = TILE_THREADS >> a.lsh, L = a.T / ng;
    const int c0 = ((slice << a.lsh) + lane) * E::V, c = a.D < E::V ? 0 : min(c0, a.D - E::V);
    const bool mine = c0 < a.D;
    const typename E::T* dout = (const typename E::T*)a.dout + (long long)t0 * a.dstride + c;
    float* part = a.part + (long long)tile * a.V * a.D + c;
    const int e0 = grp * L, e1 = e0 + L;
    int cur = skey[e0], flag = e0 > 0 && skey[e0 - 1] == cur ? 1 : 0;      // (see embed_sum_kernel)
    bool began_before = flag;
    const int next = e1 < a.T ? skey[e1] : -1;
    float acc[E::V] = {};
    const auto finish = [&]() {
        if (began_before) {
#pragma unroll
            for (int k = 0; k < E::V; ++k) head[k * TILE_THREADS + threadIdx.x] = acc[k];
        } else if (cur != a.V && mine) {
            store_part<E::V>(part + (long long)cur * a.D, a.D, acc);
        }
    };
    for (int e = e0; e < e1; e += U) {
        int k8[U];
        u32x4 r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k8[u] = skey[e + u];
            if (k8[u] != a.V && mine) r[u] = load_vec<E, NT>(dout + spos[e + u] * a.dstride, a.D);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k8[u] != cur) {
                finish();
                cur = k8[u];
                began_before = false;
#pragma unroll
                for (int k = 0; k < E::V; ++k) acc[k] = 0.f;
            }
            if (k8[u] != a.V && mine) {
                float x[E::V];
                E::unpack(r[u], x);
#pragma unroll
                for (int k = 0; k < E::V; ++k) acc[k] += x[k];
            }
        }
    }
    if (next != cur || began_before) finish();
    if (next == cur) flag |= began_before ? 2 : 4;
    if (lane == 0) flags[grp] = flag;
    __syncthreads();
    if ((flag & 4) && cur != a.V && mine) {
        for (int g = grp + 1; g < ng; ++g) {
#pragma unroll
            for (int k = 0; k < E::V; ++k) acc[k] += head[k * TILE_THREADS + (g << a.lsh) + lane];
            if (!(flags[g] & 2)) break;
        }
        store_part<E::V>(part + (long long)cur * a.D, a.D, acc);
    }
}

// dtable[v] = scale * the tiles' sums of token v, in order: 2^jlsh lanes a row, the tiles shared over the groups of lanes.
template <class E, int THREADS>
__global__ __launch_bounds__(THREADS) void embed_tile_join_kernel(TileArgs a) {
    constexpr int U = 8;
    __shared__ float sh[THREADS * E::V];
    const int v = blockIdx.x % a.V, slice = blockIdx.x / a.V;
    const int lane = threadIdx.x & ((1 << a.jlsh) - 1), grp = threadIdx.x >> a.jlsh, ng = THREADS >> a.jlsh;
    const int c0 = ((slice << a.jlsh) + lane) * E::V, c = a.D < E::V ? 0 : min(c0, a.D - E::V);
    const int share = (a.tiles + ng - 1) / ng, q1 = min(a.tiles, (grp + 1) * share);
    float acc[E::V] = {};
    if (c0 < a.D)
        for (int q = grp * share; q < q1; q += U) {
            bool in[U];
            float x[U][E::V];
#pragma unroll
            for (int u = 0; u < U; ++u) in[u] = q + u < q1 && a.count[(q + u) * a.V + v] > 0;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (in[u]) load_part<E::V>(a.part + ((long long)(q + u) * a.V + v) * a.D + c, a.D, x[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (in[u]) {
#pragma unroll
                    for (int k = 0; k < E::V; ++k) acc[k] += x[u][k];
                }
        }
    join_groups<E::V, THREADS>(acc, sh, a.jlsh);
    if (grp == 0 && c0 < a.D) {
#pragma unroll
        for (int k = 0; k < E::V; ++k) acc[k] *= a.scale;
        store_row<E>((typename E::T*)a.dtable + (long long)v * a.D + c, a.D, acc);
    }
}

// ---------------------------------------------------------------- gradient: clearing the table (rows that no token names)
__device__ __forceinline__ void clear_share(char* p, long long bytes, int blk, int nblk) {
    const long long vecs = bytes >> 4, from = (long long)blk * blockDim.x + threadIdx.x, step = (long long)nblk * blockDim.x;
    const u32x4 z = {0, 0, 0, 0};
    if (bytes > AG2V_NT_STORE_BYTES)
        for (long long i = from; i < vecs; i += step) __builtin_nontemporal_store(z, reinterpret_cast<u32x4_a2*>(p) + i);
    else
        for (long long i = from; i < vecs; i += step) reinterpret_cast<u32x4_a2*>(p)[i] = z;
    if (blk == 0)
        for (long long i = (vecs << 4) + threadIdx.x * 2; i < bytes; i += blockDim.x * 2) *reinterpret_cast<unsigned short*>(p + i) = 0;
}

// ---------------------------------------------------------------- gradient: the order by counting
// Workgroup b ranks tokens [i0, i0 + 32), i0 = 32 b: rank_i = #{j : k_j < k_i} + #{j < i : k_j = k_i}.  All keys go to LDS; a lane holds k_i
// (lanes t and t + 32 the same one) and walks its share of j, four broadcast keys a read, a compare and an add with carry each: 2 n^2 / 64
// vector instructions over the whole chip.  Before i0 equal keys count (k_j < k_i + 1), behind the 32 they do not; the 32 themselves are
// compared with their positions.  Workgroups beyond the ranking ones clear the table's gradient.  8192 tokens and a table of 64 MB: 16 us, of
// which the clearing alone is about 10.
#define RANK_MAX 8192
#define RANK_T 32
#define RANK_THREADS 1024
__global__ __launch_bounds__(RANK_THREADS) void embed_rank_kernel(const void* __restrict__ idx, int wide, long long istride, int* __restrict__ skey,
                                                                  int* __restrict__ order, int n, int V, int pad, int rank_blocks, char* clear,
                                                                  long long clear_bytes) {
    if ((int)blockIdx.x >= rank_blocks) {
        clear_share(clear, clear_bytes, blockIdx.x - rank_blocks, gridDim.x - rank_blocks);
        return;
    }
    __shared__ __align__(16) int keys[RANK_MAX];
    const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63, i0 = blockIdx.x * RANK_T, t = wl & (RANK_T - 1);
    const int n4 = (n + 3) & ~3;
    for (int j = threadIdx.x; j < n4; j += RANK_THREADS) keys[j] = j < n ? key_at(idx, wide, istride, j, V, pad) : 0x7fffffff;
    __syncthreads();
    const int ki = i0 + t < n ? keys[i0 + t] : 0;
    // 32 shares of j, in fours: wave w's lanes below 32 take share 2 w, the others share 2 w + 1
    const int fours = n4 >> 2, share = (fours + 31) >> 5, q0 = (2 * wave + (wl >> 5)) * share, q1 = min(fours, q0 + share);
    const int qa = i0 >> 2, qb = (i0 + RANK_T) >> 2;
    int cnt = 0;
    const auto walk = [&](int from, int to, int limit) {      // keys below `limit` among fours [from, to)
#pragma unroll 8
        for (int q = from; q < to; ++q) {
            const int4 k = *reinterpret_cast<const int4*>(keys + 4 * q);
            cnt += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
        }
    };
    walk(q0, min(q1, qa), ki + 1);
    walk(max(q0, qb), q1, ki);
    for (int q = max(q0, qa); q < min(q1, qb); ++q)
        for (int e = 0; e < 4; ++e) {
            const int j = 4 * q + e, k = keys[j];
            cnt += k < ki || (k == ki && j < i0 + t);
        }
    cnt += __shfl_xor(cnt, 32, 64);
    __syncthreads();
    if (wl < RANK_T) keys[wave * RANK_T + wl] = cnt;
    __syncthreads();
    if (threadIdx.x < RANK_T && i0 + t < n) {
        int r = 0;
#pragma unroll
        for (int w = 0; w < RANK_THREADS / 64; ++w) r += keys[w * RANK_T + t];
        skey[r] = ki;
        order[r] = i0 + t;
    }
}

// ---------------------------------------------------------------- gradient: the order by radix passes
// A pass sorts by `bits` <= 9 bits of the key, stably.  Each workgroup owns `rounds` * 2048 consecutive entries.  hist: how often each digit
// occurs in each workgroup's share, counts[workgroup][digit].  scatter: a workgroup reads all counts, which gives where its entries of
// each digit begin, ranks its entries (within a wave by matching digits over ballots, then over waves, then over rounds) and writes them.
// 131071 tokens: hist 4.0 us (7.5 with a table of 39 MB to clear), scatter 10.9: the chain counts - scan - ranks - stores, twice for
// 50001 words.  Tiles of 1024 tokens or 4096 were slower (12 and 13 us a scatter).
#define RADIX_BITS 9
#define RADIX_N (1 << RADIX_BITS)
#define RADIX_THREADS 512
#define RADIX_TILE 2048
#define RADIX_BLOCKS 128
struct RadixSrc {
    const void* idx;          // first pass: the tokens
    int wide, V, pad;
    long long istride;
    const int *key, *pos;     // later passes
};
__device__ __forceinline__ int radix_key(const RadixSrc& s, int e) { return s.key ? s.key[e] : key_at(s.idx, s.wide, s.istride, e, s.V, s.pad); }

__global__ __launch_bounds__(RADIX_THREADS) void embed_hist_kernel(RadixSrc s, int n, int shift, int bits, int rounds, int nb, int* __restrict__ counts,
                                                                   char* clear, long long clear_bytes) {
    if ((int)blockIdx.x >= nb) {
        clear_share(clear, clear_bytes, blockIdx.x - nb, gridDim.x - nb);
        return;
    }
    __shared__ int h[RADIX_N];
    h[threadIdx.x] = 0;
    __syncthreads();
    const int mask = (1 << bits) - 1;
    const long long lo = (long long)blockIdx.x * rounds * RADIX_TILE, hi = min((long long)n, lo + (long long)rounds * RADIX_TILE);
    for (long long e = lo + threadIdx.x; e < hi; e += RADIX_THREADS)
        atomicAdd(&h[(radix_key(s, (int)e) >> shift) & mask], 1);          // whole numbers: any order, one result
    __syncthreads();
    counts[blockIdx.x * RADIX_N + threadIdx.x] = h[threadIdx.x];
}

__global__ __launch_bounds__(RADIX_THREADS) void embed_scatter_kernel(RadixSrc s, int n, int shift, int bits, int rounds, int nb,
                                                                      const int* __restrict__ counts, int* __restrict__ okey, int* __restrict__ opos) {
    constexpr int W = RADIX_THREADS / 64, PER = RADIX_TILE / RADIX_THREADS;
    __shared__ int cnt[W][RADIX_N], base[RADIX_N], wsum[W];
    const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63, mask = (1 << bits) - 1, d = threadIdx.x;
    int key[PER], pos[PER], rank[PER];
    const auto fetch = [&](int r) {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const long long e = ((long long)blockIdx.x * rounds + r) * RADIX_TILE + wave * (64 * PER) + q * 64 + wl;
            key[q] = e < n ? radix_key(s, (int)e) : 0;
            pos[q] = e < n ? (s.pos ? s.pos[e] : (int)e) : 0;
        }
    };
    fetch(0);
    // where this workgroup's entries of digit d begin: all entries of smaller digits, then those of d in earlier workgroups
    int before = 0, total = 0;
    for (int b0 = 0; b0 < nb; b0 += 32) {
        int c[32];
#pragma unroll
        for (int u = 0; u < 32; ++u) c[u] = b0 + u < nb ? counts[(b0 + u) * RADIX_N + d] : 0;
#pragma unroll
        for (int u = 0; u < 32; ++u) {
            total += c[u];
            before += b0 + u < (int)blockIdx.x ? c[u] : 0;
        }
    }
    int scan = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(scan, o, 64);
        if (wl >= o) scan += up;
    }
    if (wl == 63) wsum[wave] = scan;
    __syncthreads();
    for (int w = 0; w < wave; ++w) scan += wsum[w];
    base[d] = scan - total + before;
    for (int r = 0; r < rounds; ++r) {
#pragma unroll
        for (int w = 0; w < W; ++w) cnt[w][d] = 0;
        __syncthreads();
        const long long e0 = ((long long)blockIdx.x * rounds + r) * RADIX_TILE + wave * (64 * PER);
        if (r) fetch(r);
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const bool in = e0 + q * 64 + wl < n;
            const int dig = (key[q] >> shift) & mask;
            unsigned long long m = __ballot(in);
            for (int b = 0; b < bits; ++b) {
                const bool bit = (dig >> b) & 1;
                const unsigned long long same = __ballot(bit);
                m &= bit ? same : ~same;
            }
            const int lower = __popcll(m & ((1ull << wl) - 1));
            int seen = 0;
            if (in) seen = cnt[wave][dig];
            __builtin_amdgcn_wave_barrier();
            if (in && lower == 0) cnt[wave][dig] = seen + __popcll(m);
            __builtin_amdgcn_wave_barrier();
            rank[q] = seen + lower;
        }
        __syncthreads();
        int run = base[d];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int c = cnt[w][d];
            cnt[w][d] = run;
            run += c;
        }
        base[d] = run;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < PER; ++q)
            if (e0 + q * 64 + wl < n) {
                const int at = cnt[wave][(key[q] >> shift) & mask] + rank[q];
                okey[at] = key[q];
                opos[at] = pos[q];
            }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- gradient: sums over the sorted order
// A group of 2^lsh lanes walks L sorted entries, eight rows in flight.  A segment (the entries of one token) that begins and ends in its
// share goes to the table at once.  The end of one that began earlier goes to LDS (head), and the group where a segment begins and goes on
// adds the heads behind its own part.  flags: 1 the share begins inside a segment, 2 which fills it and goes on, 4 a segment begins in the
// share and goes on.  What began before the workgroup or goes on behind it goes to part[0 / 1][workgroup][:] for embed_join_kernel.
// 102 MB of rows (131071 x 389 fp16, in the order of 50001 words) in 33 us and 21 MB written, 3.7 TB/s: rows of 778 bytes in no order.
struct SumArgs {
    const int *skey, *order;
    const void* dout;
    void* dtable;
    float* part;
    long long dstride;
    int n, V, D, lsh, L, nblk;
    float scale;
};
template <class E, bool NT>
__global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs a) {
    constexpr int U = 8;
    __shared__ float head[256 * E::V];
    __shared__ int flags[32];
    const int lane = threadIdx.x & ((1 << a.lsh) - 1), grp = threadIdx.x >> a.lsh, ng = 256 >> a.lsh;
    const int blk = blockIdx.x % a.nblk, slice = blockIdx.x / a.nblk;
    const int c0 = ((slice << a.lsh) + lane) * E::V, c = a.D < E::V ? 0 : min(c0, a.D - E::V);
    const bool mine = c0 < a.D;
    const typename E::T* dout = (const typename E::T*)a.dout + c;
    typename E::T* dtable = (typename E::T*)a.dtable + c;
    const long long e0 = ((long long)blk * ng + grp) * a.L, e1 = min((long long)a.n, e0 + a.L);
    int cur = a.V, flag = 0;
    float acc[E::V] = {};
    if (e0 < e1) {
        cur = a.skey[e0];
        bool began_before = e0 > 0 && a.skey[e0 - 1] == cur;
        const int next = e1 < a.n ? a.skey[e1] : -1;
        flag = began_before ? 1 : 0;
        const auto finish = [&]() {          // the segment `cur` ends here, or the share does
            if (began_before) {
#pragma unroll
                for (int k = 0; k < E::V; ++k) head[k * 256 + threadIdx.x] = acc[k];
            } else if (cur != a.V && mine) {
                float v[E::V];
#pragma unroll
                for (int k = 0; k < E::V; ++k) v[k] = acc[k] * a.scale;
                store_row<E>(dtable + (long long)cur * a.D, a.D, v);
            }
        };
        for (long long e = e0; e < e1; e += U) {
            int key[U], pos[U];
#pragma unroll
            for (int q = 0; q < U / 4; ++q) {
                const int4 k4 = *reinterpret_cast<const int4*>(a.skey + e + 4 * q), p4 = *reinterpret_cast<const int4*>(a.order + e + 4 * q);
                key[4 * q] = k4.x; key[4 * q + 1] = k4.y; key[4 * q + 2] = k4.z; key[4 * q + 3] = k4.w;
                pos[4 * q] = p4.x; pos[4 * q + 1] = p4.y; pos[4 * q + 2] = p4.z; pos[4 * q + 3] = p4.w;
            }
            u32x4 r[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (e + u < e1 && key[u] != a.V && mine) r[u] = load_vec<E, NT>(dout + pos[u] * a.dstride, a.D);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (e + u < e1) {
                    if (key[u] != cur) {
                        finish();
                        cur = key[u];
                        began_before = false;
#pragma unroll
                        for (int k = 0; k < E::V; ++k) acc[k] = 0.f;
                    }
                    if (key[u] != a.V && mine) {
                        float x[E::V];
                        E::unpack(r[u], x);
#pragma unroll
                        for (int k = 0; k < E::V; ++k) acc[k] += x[k];
                    }
                }
        }
        if (next != cur || began_before) finish();
        if (next == cur) flag |= began_before ? 2 : 4;
    }
    if (lane == 0) flags[grp] = flag;
    __syncthreads();
    if (!mine) return;
    float* part = a.part + (long long)blk * a.D + c;
    // group g's head onto x; whether the segment goes on behind it
    const auto add_head = [&](float (&x)[E::V], int g) {
#pragma unroll
        for (int k = 0; k < E::V; ++k) x[k] += head[k * 256 + (g << a.lsh) + lane];
        return (flags[g] & 2) != 0;
    };
    if (flag & 4) {
        bool open = true;
        for (int g = grp + 1; open && g < ng; ++g) open = add_head(acc, g);
        if (open) {
            store_part<E::V>(part + (long long)a.nblk * a.D, a.D, acc);
        } else if (cur != a.V) {
#pragma unroll
            for (int k = 0; k < E::V; ++k) acc[k] *= a.scale;
            store_row<E>(dtable + (long long)cur * a.D, a.D, acc);
        }
    }
    if (grp == 0 && (flag & 1)) {
        float x[E::V] = {};
        bool open = true;
        for (int g = 0; open && g < ng; ++g) open = add_head(x, g);
        store_part<E::V>(part, a.D, x);
    }
}

// The segments that cross workgroups of embed_sum_kernel: the workgroup where one begins adds its tail and the heads behind it.  8.6 us where the
// longest has 8400 tokens, 5 us else: five loads that wait for each other.
template <class E>
__global__ __launch_bounds__(256) void embed_join_kernel(SumArgs a) {
    __shared__ float sh[256 * E::V];
    const int blk = blockIdx.x % a.nblk, slice = blockIdx.x / a.nblk, ng = 256 >> a.lsh;
    const long long B = (long long)ng * a.L, s = blk * B, t = min((long long)a.n, s + B) - 1;
    if (t + 1 >= a.n) return;
    const int key = a.skey[t];
    if (key == a.V || a.skey[t + 1] != key) return;
    if (a.skey[s] == key && s > 0 && a.skey[s - 1] == key) return;       // began earlier
    int m = 0;                                                           // workgroups behind this one that the segment reaches
    for (int q = blk + 1;; q += 256) {
        const int k = __syncthreads_count(q + (int)threadIdx.x < a.nblk && a.skey[(q + (int)threadIdx.x) * B] == key);
        m += k;
        if (k < 256) break;
    }
    const int lane = threadIdx.x & ((1 << a.lsh) - 1), grp = threadIdx.x >> a.lsh;
    const int c0 = ((slice << a.lsh) + lane) * E::V, c = a.D < E::V ? 0 : min(c0, a.D - E::V);
    const int share = (m + ng - 1) / ng, q0 = min(m, grp * share), q1 = min(m, q0 + share);
    const float* heads = a.part + (long long)(blk + 1) * a.D + c;
    float acc[E::V] = {};
    if (c0 < a.D) {
        for (int q = q0; q < q1; q += 8) {
            float x[8][E::V];
#pragma unroll
            for (int u = 0; u < 8; ++u) load_part<E::V>(heads + (long long)min(q + u, q1 - 1) * a.D, a.D, x[u]);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (q + u < q1) {
#pragma unroll
                    for (int k = 0; k < E::V; ++k) acc[k] += x[u][k];
                }
        }
    }
    join_groups<E::V, 256>(acc, sh, a.lsh);
    if (grp == 0 && c0 < a.D) {
        const float* tail = a.part + (long long)a.nblk * a.D + (long long)blk * a.D + c;
        float v[E::V];
        load_part<E::V>(tail, a.D, v);
#pragma unroll
        for (int k = 0; k < E::V; ++k) v[k] = (v[k] + acc[k]) * a.scale;
        store_row<E>((typename E::T*)a.dtable + (long long)key * a.D + c, a.D, v);
    }
}

// ---------------------------------------------------------------- host
static bool embed_ok(int dtype, int idx_bytes, long long n, long long V, int D) {
    return dtype >= AG2V_F32 && dtype <= AG2V_F16 && (idx_bytes == 4 || idx_bytes == 8) && n > 0 && n < (1LL << 31) &&
           V > 0 && V < (1LL << 31) - 1 && D > 0 && D < (1 << 30);
}
static int log2_up(long long v) {
    int l = 0;
    while ((1LL << l) < v) ++l;
    return l;
}
static int vec_of(int dtype) { return dtype == AG2V_F32 ? ElemF32::V : ElemBF16::V; }

#define MOST_BLOCKS (1LL << 24)     // a launch takes fewer than 2^32 threads: fewer workgroups of 256 than this
// How the gradient of (n, V, D) runs.
struct EmbedPlan {
    bool pick, tile, rank;
    int lsh, slices, L, nblk;       // sums
    int jlsh, jslices;              // join of tiles
    int T, tiles, bits, passes, rounds, nb;   // tiles; radix
    long long npad, words;          // workspace: sorted keys and positions, their ping-pong, counts, parts
};
static EmbedPlan plan_of(int dtype, long long n, long long V, int D) {
    EmbedPlan p = {};
    const long long cv = ((long long)D + vec_of(dtype) - 1) / vec_of(dtype);
    p.lsh = log2_up(cv < 64 ? cv : 64);
    if (p.lsh < 3) p.lsh = 3;       // at most 32 groups a workgroup
    p.slices = (int)((cv + (1 << p.lsh) - 1) >> p.lsh);
    // One workgroup may get all n tokens: at most 64 rows a group of lanes then (2156 equal tokens of 136 fp16 took 64 us in groups of 8 times as
    // many rows, 18 us by ranks).  Every row costs a workgroup: 2000 tokens of 64 fp32, lookup and gradient, take 12.4 us with 1024 rows (by
    // ranks 16.9) and 18.9 with 2048 (17.1).
    p.pick = n <= 64LL * (PICK_THREADS >> p.lsh) && n <= PICK_MAX && V * p.slices <= 1024;
    if (p.pick) return p;
    // about 256 tiles, at most 512, whose sums (fp32, V rows a tile) are at most a quarter of the bytes of the rows summed: 131072 tokens of 27
    // words, 128 wide, take 23 us so and 33 us by a radix pass; 524288 of 256 words in fp16, half the rows' bytes, 72 and 55 us.  The keys 0 .. V
    // have a counter each in LDS
    p.T = TILE_MIN;
    while (p.T < TILE_MAX && n >= 512LL * p.T) p.T *= 2;
    // (rows so wide that their slices would pass what a launch holds go the other way)
    const long long slices16 = (cv + 15) >> 4;
    p.tile = V * 16 <= (dtype == AG2V_F32 ? 4 : 2) * p.T && V < 1 << TILE_BITS && n <= 512LL * TILE_MAX && slices16 * V < MOST_BLOCKS / 4 &&
             slices16 * ((n + p.T - 1) / p.T) < MOST_BLOCKS / 4;
    if (p.tile) {
        p.jlsh = p.lsh;
        p.jslices = p.slices;
        if (p.lsh > 4) {                // 16 lanes a row: shares of 16 tokens at least, and more workgroups
            p.lsh = 4;
            p.slices = (int)slices16;
        }
        p.tiles = (int)((n + p.T - 1) / p.T);
        if (p.tiles > TILE_JOIN_WIDE) {
            p.jlsh = p.lsh;
            p.jslices = p.slices;
        }
        p.bits = log2_up(V + 1);
        p.words = ((long long)p.tiles * V + 3) / 4 * 4 + (long long)p.tiles * V * D;
        return p;
    }
    // counting takes 6.2 us for 2156 tokens, 10.5 for 5849, 25 for 11925; a radix pass 12: one pass (V < 512) is faster from 6000 tokens on,
    // two or more from about 11000
    p.rank = n <= (V < RADIX_N ? RANK_MAX * 3 / 4 : RANK_MAX);
    // entries a group walks: enough groups for 4096 waves, 8 .. 64 (for 2048 waves 131072 rows of 389 fp16 take 49 us and not 37; for 8192 the join
    // of their longest segment 14 us and not 8.6); more only where the workgroups' parts would pass 16384, or the workgroups what a launch holds
    const int ng = 256 >> p.lsh;
    long long L = (n * p.slices << p.lsh) / 64 / 4096;
    L = L < 8 ? 8 : L > 64 ? 64 : 1LL << (log2_up(L + 1) - 1);
    while ((n + ng * L - 1) / (ng * L) > 16384 || (n + ng * L - 1) / (ng * L) * p.slices >= MOST_BLOCKS) L *= 2;
    p.L = (int)L;
    p.nblk = (int)((n + ng * L - 1) / (ng * L));
    p.npad = (n + 63) / 64 * 64;
    p.words = 2 * p.npad + 2LL * p.nblk * D;
    if (!p.rank) {
        const int all = log2_up(V + 1);      // keys 0 .. V
        p.passes = (all + RADIX_BITS - 1) / RADIX_BITS;
        p.bits = (all + p.passes - 1) / p.passes;
        const long long tiles = (n + RADIX_TILE - 1) / RADIX_TILE;
        p.rounds = (int)((tiles + RADIX_BLOCKS - 1) / RADIX_BLOCKS);
        p.nb = (int)((tiles + p.rounds - 1) / p.rounds);
        p.words += (p.passes > 1 ? 2 * p.npad : 0) + (long long)RADIX_N * p.nb;
    }
    return p;
}

template <class E>
static int run_fwd(const void* idx, int idx_bytes, long long istride, const void* table, long long tstride, void* out, long long n, int V, int D,
                   float scale, hipStream_t st) {
    const long long cv = ((long long)D + E::V - 1) / E::V;
    const int lsh = log2_up(cv < 64 ? cv : 64), rows = (256 >> lsh) * 4;
    const long long blocks = (n + rows - 1) / rows;
    const dim3 grid((int)(blocks < (1 << 20) ? blocks : (1 << 20)));
    if (n * D * (long long)sizeof(typename E::T) > AG2V_NT_STORE_BYTES)
        hipLaunchKernelGGL((embed_fwd_kernel<E, true>), grid, dim3(256), 0, st, idx, idx_bytes == 8, istride, (const typename E::T*)table, tstride,
                           (typename E::T*)out, n, V, D, scale, lsh);
    else
        hipLaunchKernelGGL((embed_fwd_kernel<E, false>), grid, dim3(256), 0, st, idx, idx_bytes == 8, istride, (const typename E::T*)table, tstride,
                           (typename E::T*)out, n, V, D, scale, lsh);
    AG2V_CHECK_LAUNCH();
    return AG2V_OK;
}

template <class E>
static int run_bwd(const EmbedPlan& p, const void* idx, int wide, long long istride, const void* dout, long long dstride, void* dtable, int n, int V,
                   int D, float scale, int pad, float* workspace, hipStream_t st) {
    if (p.pick) {
        hipLaunchKernelGGL(embed_pick_kernel<E>, dim3(V * p.slices), dim3(PICK_THREADS), 0, st, idx, wide, istride, (const typename E::T*)dout, dstride,
                           (typename E::T*)dtable, n, V, D, scale, pad, p.lsh);
        AG2V_CHECK_LAUNCH();
        return AG2V_OK;
    }
    if (p.tile) {
        int* count = (int*)workspace;
        const TileArgs t = {idx, dout, dtable, count, workspace + ((long long)p.tiles * V + 3) / 4 * 4, istride, dstride, wide, n, V, D, pad,
                            p.lsh, p.jlsh, p.T, p.bits, p.tiles, scale};
        if ((long long)n * D * (long long)sizeof(typename E::T) > AG2V_NT_LOAD_BYTES)
            hipLaunchKernelGGL((embed_tile_kernel<E, true>), dim3(p.tiles * p.slices), dim3(TILE_THREADS), 0, st, t);
        else
            hipLaunchKernelGGL((embed_tile_kernel<E, false>), dim3(p.tiles * p.slices), dim3(TILE_THREADS), 0, st, t);
        AG2V_CHECK_LAUNCH();
        if (p.tiles > TILE_JOIN_WIDE)
            hipLaunchKernelGGL((embed_tile_join_kernel<E, 1024>), dim3(V * p.jslices), dim3(1024), 0, st, t);
        else
            hipLaunchKernelGGL((embed_tile_join_kernel<E, 256>), dim3(V * p.jslices), dim3(256), 0, st, t);
        AG2V_CHECK_LAUNCH();
        return AG2V_OK;
    }
    int *skey = (int*)workspace, *order = skey + p.npad;
    const long long bytes = (long long)V * D * (long long)sizeof(typename E::T);
    // one vector a thread: workgroups that walk the table write it slower (4000 tokens of 131072 words, 1024 bf16: 64 us a training pass, 84 with
    // 1024 workgroups)
    const int threads = p.rank ? RANK_THREADS : RADIX_THREADS;
    const long long cb = (bytes / 16 + threads - 1) / threads;
    const int clearers = cb < 1 ? 1 : cb < 65536 ? (int)cb : 65536;
    SumArgs a = {skey, order, dout, dtable, (float*)(order + p.npad), dstride, n, V, D, p.lsh, p.L, p.nblk, scale};
    if (p.rank) {
        const int rank_blocks = ceil_div(n, RANK_T);
        hipLaunchKernelGGL(embed_rank_kernel, dim3(rank_blocks + clearers), dim3(RANK_THREADS), 0, st, idx, wide, istride, skey, order, n, V,
                           pad, rank_blocks, (char*)dtable, bytes);
        AG2V_CHECK_LAUNCH();
    } else {
        int* counts = (int*)(a.part + 2LL * p.nblk * D);
        int *key2 = counts + (long long)RADIX_N * p.nb, *pos2 = key2 + p.npad;
        RadixSrc s = {idx, wide, V, pad, istride, nullptr, nullptr};
        for (int q = 0; q < p.passes; ++q) {
            const bool last = ((p.passes - 1 - q) & 1) == 0;         // the last pass writes skey / order, the passes before it in turn
            int *ok = last ? skey : key2, *op = last ? order : pos2;
            hipLaunchKernelGGL(embed_hist_kernel, dim3(p.nb + (q == 0 ? clearers : 0)), dim3(RADIX_THREADS), 0, st, s, n, q * p.bits, p.bits, p.rounds,
                               p.nb, counts, (char*)dtable, bytes);
            AG2V_CHECK_LAUNCH();
            hipLaunchKernelGGL(embed_scatter_kernel, dim3(p.nb), dim3(RADIX_THREADS), 0, st, s, n, q * p.bits, p.bits, p.rounds, p.nb, counts, ok, op);
            AG2V_CHECK_LAUNCH();
            s.key = ok;
            s.pos = op;
        }
    }
    if ((long long)n * D * (long long)sizeof(typename E::T) > AG2V_NT_LOAD_BYTES)
        hipLaunchKernelGGL((embed_sum_kernel<E, true>), dim3(p.nblk * p.slices), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((embed_sum_kernel<E, false>), dim3(p.nblk * p.slices), dim3(256), 0, st, a);
    AG2V_CHECK_LAUNCH();
    if (p.nblk > 1) {
        hipLaunchKernelGGL(embed_join_kernel<E>, dim3(p.nblk * p.slices), dim3(256), 0, st, a);
        AG2V_CHECK_LAUNCH();
    }
    return AG2V_OK;
}

extern "C" size_t ag2v_embed_bwd_workspace_floats(int dtype, long long n, long long V, int D) {
    return embed_ok(dtype, 8, n, V, D) ? (size_t)plan_of(dtype, n, V, D).words : 0;
}
extern "C" int ag2v_embed_fwd(int dtype, const void* idx, int idx_bytes, long long idx_stride, const void* table, long long table_stride,
                              void* out, long long n, long long V, int D, float scale, void* stream) {
    if (!idx || !table || !out || !embed_ok(dtype, idx_bytes, n, V, D) || table_stride < D) return AG2V_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AG2V_F32) return run_fwd<ElemF32>(idx, idx_bytes, idx_stride, table, table_stride, out, n, (int)V, D, scale, st);
    if (dtype == AG2V_BF16) return run_fwd<ElemBF16>(idx, idx_bytes, idx_stride, table, table_stride, out, n, (int)V, D, scale, st);
    return run_fwd<ElemF16>(idx, idx_bytes, idx_stride, table, table_stride, out, n, (int)V, D, scale, st);
}
extern "C" int ag2v_embed_bwd(int dtype, const void* idx, int idx_bytes, long long idx_stride, const void* dout, long long dout_stride,
                              void* dtable, long long n, long long V, int D, float scale, long long padding_idx, float* workspace,
                              size_t workspace_floats, void* stream) {
    if (!idx || !dout || !dtable || !embed_ok(dtype, idx_bytes, n, V, D)) return AG2V_EINVAL;
    const EmbedPlan p = plan_of(dtype, n, V, D);
    if ((p.words && !workspace) || workspace_floats < (size_t)p.words || ((uintptr_t)workspace & 15)) return AG2V_EINVAL;
    const int wide = idx_bytes == 8, pad = padding_idx >= 0 && padding_idx < V ? (int)padding_idx : -1;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AG2V_F32)
        return run_bwd<ElemF32>(p, idx, wide, idx_stride, dout, dout_stride, dtable, (int)n, (int)V, D, scale, pad, workspace, st);
    if (dtype == AG2V_BF16)
        return run_bwd<ElemBF16>(p, idx, wide, idx_stride, dout, dout_stride, dtable, (int)n, (int)V, D, scale, pad, workspace, st);
    return run_bwd<ElemF16>(p, idx, wide, idx_stride, dout, dout_stride, dtable, (int)n, (int)V, D, scale, pad, workspace, st);
}
