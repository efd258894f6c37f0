// moe_sort.cu -- (token, expert) pairs sorted by expert and back, as operators of their own:
// the sort, the copy of every pair's token row into expert order (plain, or quantised to MXFP4
// on the way), the weighted sum back per token, and the gradients of both copies. No reference
// counterpart (the reference visits a token's experts one after another,
// src/core/k3_ops.c:630-645); the order of a token's sum is the reference's.
//
// With pairs p = t*topk + j:
//     pos[p]  = off[idx[p]] + #{q < p : idx[q] = idx[p]}       (stable counting sort)
//     rows[pos[t][j]] = x[t]                                    permute
//     dx[t]   = sum_j drows[pos[t][j]]                          its gradient
//     out[t]  = sum_j wt[t][j] * y[pos[t][j]]                   unpermute
//     dy[pos[t][j]] = wt[t][j] * dout[t],  dwt[t][j] = <dout[t], y[pos[t][j]]>
// Sums run in the order of j in fp32, each result is rounded once. Every output element has one
// writer, so no result depends on the order in which blocks run.
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "mx4_quant.cuh"

namespace k3c {

namespace {

// ------------------------------------------------------------------ sort
constexpr int SORT_TH = 1024;
constexpr int SORT_WARPS = SORT_TH / 32;
constexpr int SORT_ONE = 8;                       // rounds of 32 pairs a warp, when one block takes all pairs
constexpr int SORT_MANY = 2;                      // and when several do, per pass
constexpr int SORT_SUB = SORT_MANY * SORT_TH;     // pairs of a pass
constexpr int SORT_BLOCKS = 128;                  // blocks at most: every one reads all blocks' counts
constexpr int SORT_EMAX = 2048;

__device__ __forceinline__ int expert_of(const int *idx, int p, int P, int E) {
    if (p >= P) return -1;
    const int e = __ldg(idx + p);
    return (unsigned)e < (unsigned)E ? e : -1;
}

// Exclusive prefix sums of v over the block's threads; all: their total. warp_tot: SORT_WARPS ints.
__device__ __forceinline__ int block_prefix(int v, int &all, int *warp_tot) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) warp_tot[warp] = inc;
    __syncthreads();
    const int t = warp_tot[lane];                 // every warp sums the warps' totals itself
    int ti = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, ti, o);
        if (lane >= o) ti += u;
    }
    all = __shfl_sync(0xffffffffu, ti, 31);
    const int pre = __shfl_sync(0xffffffffu, ti - t, warp);
    __syncthreads();                              // warp_tot may be written again
    return pre + inc - v;
}

// A warp's pairs of one pass: 32 * R of them side by side from p0 on. count() adds the warp's counts
// per expert into its own row `mine` of the table; after the table's columns have been turned
// into first ranks, place() gives each pair its rank: earlier rounds through `mine`, lower lanes
// with the same expert by one match per round. No atomics, and a stable order.
template <int R>
struct WarpPairs {
    int ex[R];
    uint32_t same[R];
    __device__ __forceinline__ void count(uint16_t *mine, const int *idx, int p0, int hi, int E) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < R; r++) ex[r] = expert_of(idx, p0 + 32 * r + lane, hi, E);
#pragma unroll
        for (int r = 0; r < R; r++) {
            same[r] = __match_any_sync(0xffffffffu, ex[r]);
            if (ex[r] >= 0 && (same[r] & ((1u << lane) - 1u)) == 0) mine[ex[r]] += (uint16_t)__popc(same[r]);
            __syncwarp();
        }
    }
    __device__ __forceinline__ void place(uint16_t *mine, const int *base, int *pos, int *pair, int p0, int hi) {
        const int lane = threadIdx.x & 31;
        const uint32_t below = (1u << lane) - 1u;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int p = p0 + 32 * r + lane;
            int row = -1;
            if (ex[r] >= 0) row = base[ex[r]] + mine[ex[r]] + __popc(same[r] & below);
            __syncwarp();
            if (ex[r] >= 0 && (same[r] & below) == 0) mine[ex[r]] += (uint16_t)__popc(same[r]);
            __syncwarp();
            if (p < hi) {
                pos[p] = row;
                if (row >= 0) pair[row] = p;
            }
        }
    }
};

// Column e of the table [warps][E] from counts to first ranks; returns its sum.
__device__ __forceinline__ int column_ranks(uint16_t *wh, int warps, int E, int e) {
    int at = 0;
#pragma unroll 4
    for (int w = 0; w < warps; w++) {
        const int c = wh[w * E + e];
        wh[w * E + e] = (uint16_t)at;
        at += c;
    }
    return at;
}

// All pairs in one block (at most SORT_ONE * SORT_TH): warps = those that have any. Bound by its
// launch and five barriers: 3.6 us for 128 pairs and 384 experts, 7.2 for 6216 and 48.
__global__ void __launch_bounds__(SORT_TH) k_sort_one(int *__restrict__ pos, int *__restrict__ pair, int *__restrict__ off,
                                                      const int *__restrict__ idx, int P, int E, int warps) {
    extern __shared__ int sort_sm[];
    int *base = sort_sm;                                       // [E] first row of each expert
    uint16_t *wh = reinterpret_cast<uint16_t *>(base + E);     // [warps][E]
    __shared__ int warp_tot[SORT_WARPS];
    const int tid = threadIdx.x, warp = tid >> 5;
    for (int i = tid; i < (warps * E + 1) / 2; i += SORT_TH) reinterpret_cast<uint32_t *>(wh)[i] = 0;
    __syncthreads();
    WarpPairs<SORT_ONE> mine;
    uint16_t *row = wh + warp * E;
    const int p0 = warp * (SORT_ONE * 32);
    if (warp < warps) mine.count(row, idx, p0, P, E);
    __syncthreads();
    int run = 0;
    for (int e0 = 0; e0 < E; e0 += SORT_TH) {
        const int e = e0 + tid, n = e < E ? column_ranks(wh, warps, E, e) : 0;
        int all;
        const int first = run + block_prefix(n, all, warp_tot);
        if (e < E) base[e] = off[e] = first;
        run += all;
    }
    if (tid == 0) off[E] = run;
    for (int r = run + tid; r < P; r += SORT_TH) pair[r] = -1;   // rows behind the last pair
    __syncthreads();
    if (warp < warps) mine.place(row, base, pos, pair, p0, P);
}

// Counts of a block's pairs per expert: cnt[block][E].
__global__ void __launch_bounds__(SORT_TH) k_sort_count(int *__restrict__ cnt, const int *__restrict__ idx, int P,
                                                        int E, int chunk) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ int sort_sm[];
    for (int e = threadIdx.x; e < E; e += SORT_TH) sort_sm[e] = 0;
    __syncthreads();
    const int lo = blockIdx.x * chunk, hi = min(P - lo, chunk) + lo;
    for (int p = lo + threadIdx.x; p < hi; p += SORT_TH) {
        const int e = expert_of(idx, p, P, E);
        if (e >= 0) atomicAdd(&sort_sm[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += SORT_TH) cnt[(size_t)blockIdx.x * E + e] = sort_sm[e];
}

// Each block finds its experts' next free rows from all blocks' counts and places its chunk,
// SORT_SUB pairs at a time. A programmatic dependent of k_sort_count: the first pass's matching
// needs only idx, which was there before that kernel began. 32768 pairs, 384 experts: 8.1 us for both.
__global__ void __launch_bounds__(SORT_TH) k_sort_place(int *__restrict__ pos, int *__restrict__ pair,
                                                        int *__restrict__ off, const int *__restrict__ idx,
                                                        const int *cnt, int P, int E, int chunk) {
    extern __shared__ int sort_sm[];
    int *base = sort_sm;                                       // [E] next free row of each expert
    uint16_t *wh = reinterpret_cast<uint16_t *>(base + E);     // [SORT_WARPS][E]
    __shared__ int warp_tot[SORT_WARPS];
    const int tid = threadIdx.x, warp = tid >> 5, nblk = gridDim.x;
    const int lo = blockIdx.x * chunk, hi = min(P - lo, chunk) + lo;
    uint16_t *row = wh + warp * E;
    WarpPairs<SORT_MANY> mine;
    auto first_half = [&](int s0) {
        for (int i = tid; i < SORT_WARPS * E / 2; i += SORT_TH) reinterpret_cast<uint32_t *>(wh)[i] = 0;
        __syncthreads();
        mine.count(row, idx, s0 + warp * (SORT_MANY * 32), hi, E);
    };
    first_half(lo);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int run = 0;
    for (int e0 = 0; e0 < E; e0 += SORT_TH) {
        const int e = e0 + tid;
        int n = 0, before = 0;
        if (e < E) {
#pragma unroll 8
            for (int b = 0; b < nblk; b++) {
                const int c = __ldcg(cnt + (size_t)b * E + e);
                before += b < (int)blockIdx.x ? c : 0;
                n += c;
            }
        }
        int all;
        const int first = run + block_prefix(n, all, warp_tot);
        if (e < E) {
            base[e] = first + before;
            if (blockIdx.x == 0) off[e] = first;
        }
        run += all;
    }
    if (blockIdx.x == 0 && tid == 0) off[E] = run;
    for (int r = lo + tid; r < hi; r += SORT_TH)   // rows behind the last pair
        if (r >= run) pair[r] = -1;
    for (int s0 = lo; s0 < hi; s0 += SORT_SUB) {
        if (s0 != lo) first_half(s0);
        __syncthreads();
        for (int e = tid; e < E; e += SORT_TH) column_ranks(wh, SORT_WARPS, E, e);
        __syncthreads();
        mine.place(row, base, pos, pair, s0 + warp * (SORT_MANY * 32), hi);
        __syncthreads();
        // the last warp's running ranks are the pass's counts
        for (int e = tid; e < E; e += SORT_TH) base[e] += wh[(SORT_WARPS - 1) * E + e];
        __syncthreads();
    }
}

// ------------------------------------------------------------------ elements
// 16 bytes of T as floats and back; V elements.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int V = 4;
    static __device__ __forceinline__ void get(const uint4 &u, float (&f)[4]) {
        f[0] = __uint_as_float(u.x);
        f[1] = __uint_as_float(u.y);
        f[2] = __uint_as_float(u.z);
        f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 put(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ float back(float v) { return v; }
};
template <>
struct Vec<uint16_t> {   // bf16 bits
    static constexpr int V = 8;
    static __device__ __forceinline__ void get(const uint4 &u, float (&f)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
        return make_uint4(f32x2_to_bf16x2(f[0], f[1]), f32x2_to_bf16x2(f[2], f[3]), f32x2_to_bf16x2(f[4], f[5]),
                          f32x2_to_bf16x2(f[6], f[7]));
    }
    static __device__ __forceinline__ float one(uint16_t v) { return bf16_bits_to_f32(v); }
    static __device__ __forceinline__ uint16_t back(float v) { return (uint16_t)(f32x2_to_bf16x2(v, 0.0f) & 0xFFFFu); }
};

__device__ __forceinline__ uint4 ld16(const void *p) { return ldg_nc_v4(p); }
// Past L1, but with L2's ordinary policy: a later kernel reads what is written here.
__device__ __forceinline__ void st16(void *p, const uint4 &v) {
    asm volatile("st.global.L1::no_allocate.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}

constexpr int PM_TH = 512;   // threads of a block at most
// Rows on no 16-byte boundary move element by element, so many per thread and round (32768 rows of
// 7167 bf16 summed to 4096: 175 us, 202 with one at a time). Bound by the number of loads and stores: 2 bytes
// each where aligned rows of 7168 move 16 in 78 us; in fp32 (3583 and 3584 wide) 99 and 80.
constexpr int PM_U = 4, UB_U = 2;

// A token's pairs that have a row, in the order of j: rows, j and weights in shared memory, so that
// the loops below run over those pairs alone with several loads in flight (an expert-parallel
// rank holds one pair in eight). A row outside [0, P) counts as none.
struct TokenRows {
    int row[K3_MAX_TOPK], j[K3_MAX_TOPK];
    float w[K3_MAX_TOPK];
    int n;
};
__device__ __forceinline__ int token_rows(TokenRows &s, const int *__restrict__ pos, const float *__restrict__ wt,
                                          size_t p0, int P, int topk) {
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int n = 0;
        for (int j0 = 0; j0 < topk; j0 += 32) {
            const int j = j0 + lane, r = j < topk ? __ldg(pos + p0 + j) : -1;
            const float w = wt && j < topk ? __ldg(wt + p0 + j) : 1.0f;
            const bool on = (unsigned)r < (unsigned)P;
            const uint32_t m = __ballot_sync(0xffffffffu, on);
            if (on) {
                const int at = n + __popc(m & ((1u << lane) - 1u));
                s.row[at] = r;
                s.j[at] = j;
                s.w[at] = w;
            }
            n += __popc(m);
        }
        if (lane == 0) s.n = n;
    }
    __syncthreads();
    return s.n;
}

// ------------------------------------------------------------------ permute
// Block (t, h): 16-byte chunks of token t, read once and stored into the token's rows. Bound by HBM,
// nearly all of it writes: 4096 x 8 rows of 14 KB in 88 us, 6.0 TB/s.
template <typename T, bool VEC>
__global__ void __launch_bounds__(PM_TH) k_permute(T *__restrict__ rows, const T *__restrict__ x, int64_t ldx,
                                                   const int *__restrict__ pos, int P, int topk, int H) {
    __shared__ TokenRows s;
    const int t = blockIdx.x;
    const T *xr = x + (size_t)t * ldx;
    const int m = token_rows(s, pos, nullptr, (size_t)t * topk, P, topk);
    if (!m) return;
    if constexpr (VEC) {
        constexpr int V = Vec<T>::V;
        const int n = H / V, stride = gridDim.y * blockDim.x;
        for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < n; c += stride) {
            const uint4 v = ld16(xr + (size_t)c * V);
#pragma unroll 4
            for (int j = 0; j < m; j++) st16(rows + (size_t)s.row[j] * H + (size_t)c * V, v);
        }
    } else {
        const int th = blockDim.x;
        for (int c0 = blockIdx.y * th * PM_U + threadIdx.x; c0 < H; c0 += gridDim.y * th * PM_U) {
            T v[PM_U];
#pragma unroll
            for (int i = 0; i < PM_U; i++)
                if (c0 + i * th < H) v[i] = xr[c0 + i * th];
            for (int j = 0; j < m; j++) {
                T *r = rows + (size_t)s.row[j] * H;
#pragma unroll
                for (int i = 0; i < PM_U; i++)
                    if (c0 + i * th < H) r[c0 + i * th] = v[i];
            }
        }
    }
}

// ------------------------------------------------------------------ sums back per token
// out[t] = sum_j w_j y[pos[t][j]]; wt NULL: w_j = 1 (the gradient of the permute). Eight rows'
// loads are in flight before the first is added; the additions keep the order of j. Bound by HBM:
// 4096 x 8 rows of 14 KB in 80 us, 6.6 TB/s.
constexpr int GS_JB = 8;
template <typename T, typename O, bool VEC>
__global__ void __launch_bounds__(PM_TH) k_gather_sum(O *__restrict__ out, const T *__restrict__ y,
                                                      const float *__restrict__ wt, const int *__restrict__ pos, int P,
                                                      int topk, int H) {
    __shared__ TokenRows s;
    const int t = blockIdx.x;
    const int m = token_rows(s, pos, wt, (size_t)t * topk, P, topk);
    if constexpr (VEC) {
        constexpr int V = Vec<T>::V, VO = Vec<O>::V;
        const int n = H / V, stride = gridDim.y * blockDim.x;
        for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < n; c += stride) {
            float acc[V];
#pragma unroll
            for (int i = 0; i < V; i++) acc[i] = 0.0f;
            for (int j0 = 0; j0 < m; j0 += GS_JB) {
                uint4 u[GS_JB];
#pragma unroll
                for (int q = 0; q < GS_JB; q++)
                    if (j0 + q < m) u[q] = ld16(y + (size_t)s.row[j0 + q] * H + (size_t)c * V);
#pragma unroll
                for (int q = 0; q < GS_JB; q++)
                    if (j0 + q < m) {
                        const float w = s.w[j0 + q];
                        float f[V];
                        Vec<T>::get(u[q], f);
#pragma unroll
                        for (int i = 0; i < V; i++) acc[i] = __fadd_rn(acc[i], __fmul_rn(w, f[i]));
                    }
            }
            O *o = out + (size_t)t * H + (size_t)c * V;
            if constexpr (VO == V) {
                st16(o, Vec<O>::put(acc));
            } else if constexpr (VO < V) {   // bf16 rows, fp32 sums: two stores
#pragma unroll
                for (int h = 0; h < V / VO; h++) {
                    float part[VO];
#pragma unroll
                    for (int i = 0; i < VO; i++) part[i] = acc[h * VO + i];
                    st16(o + h * VO, Vec<O>::put(part));
                }
            } else {                         // fp32 rows, bf16 sums: half a store
                *reinterpret_cast<uint2 *>(o) = make_uint2(f32x2_to_bf16x2(acc[0], acc[1]), f32x2_to_bf16x2(acc[2], acc[3]));
            }
        }
    } else {
        const int th = blockDim.x;
        for (int c0 = blockIdx.y * th * PM_U + threadIdx.x; c0 < H; c0 += gridDim.y * th * PM_U) {
            float acc[PM_U];
#pragma unroll
            for (int i = 0; i < PM_U; i++) acc[i] = 0.0f;
            for (int j0 = 0; j0 < m; j0 += GS_JB) {
                T u[GS_JB][PM_U];
#pragma unroll
                for (int q = 0; q < GS_JB; q++) {
                    const T *r = y + (size_t)s.row[j0 + q < m ? j0 + q : 0] * H;
#pragma unroll
                    for (int i = 0; i < PM_U; i++)
                        if (j0 + q < m && c0 + i * th < H) u[q][i] = r[c0 + i * th];
                }
#pragma unroll
                for (int q = 0; q < GS_JB; q++)
                    if (j0 + q < m) {
                        const float w = s.w[j0 + q];
#pragma unroll
                        for (int i = 0; i < PM_U; i++) acc[i] = __fadd_rn(acc[i], __fmul_rn(w, Vec<T>::one(u[q][i])));
                    }
            }
#pragma unroll
            for (int i = 0; i < PM_U; i++)
                if (c0 + i * th < H) out[(size_t)t * H + c0 + i * th] = Vec<O>::back(acc[i]);
        }
    }
}

// ------------------------------------------------------------------ unpermute's gradients
// One block per token: dout[t] is read once per batch of UB_JB pairs, each pair's y row once; the
// products for dwt are summed per thread in fp32, then across the block in a fixed tree. Bound by
// HBM: 4096 x 8 rows of 14 KB in 156 us, 6.4 TB/s.
constexpr int UB_JB = 8;
template <typename T, typename D, bool VEC>
__global__ void __launch_bounds__(PM_TH) k_unpermute_bwd(T *__restrict__ dy, float *__restrict__ dwt,
                                                         const D *__restrict__ dout, const T *__restrict__ y,
                                                         const float *__restrict__ wt, const int *__restrict__ pos,
                                                         int P, int topk, int H) {
    __shared__ float part[PM_TH / 32][UB_JB];
    __shared__ TokenRows s;
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t p0 = (size_t)t * topk;
    const D *dr = dout + (size_t)t * H;
    const int m = token_rows(s, pos, wt, p0, P, topk);
    // pairs without a row: their products are all absent
    if (dwt)
        for (int j = threadIdx.x; j < topk; j += blockDim.x) {
            const int r = __ldg(pos + p0 + j);
            if ((unsigned)r >= (unsigned)P) dwt[p0 + j] = 0.0f;
        }
    for (int j0 = 0; j0 < m; j0 += UB_JB) {
        const int jn = min(UB_JB, m - j0);
        float dot[UB_JB];
#pragma unroll
        for (int q = 0; q < UB_JB; q++) dot[q] = 0.0f;
        if constexpr (VEC) {
            constexpr int V = Vec<T>::V, VD = Vec<D>::V;
            for (int c = threadIdx.x; c < H / V; c += blockDim.x) {
                float d[V];
                if constexpr (VD == V) {
                    Vec<D>::get(ld16(dr + (size_t)c * V), d);
                } else if constexpr (VD > V) {   // bf16 dout, fp32 rows: half a load
                    const uint2 u = *reinterpret_cast<const uint2 *>(dr + (size_t)c * V);
                    d[0] = __uint_as_float(u.x << 16);
                    d[1] = __uint_as_float(u.x & 0xFFFF0000u);
                    d[2] = __uint_as_float(u.y << 16);
                    d[3] = __uint_as_float(u.y & 0xFFFF0000u);
                } else {                         // fp32 dout, bf16 rows: two loads
#pragma unroll
                    for (int h = 0; h < V / VD; h++) {
                        float g[VD];
                        Vec<D>::get(ld16(dr + (size_t)c * V + h * VD), g);
#pragma unroll
                        for (int i = 0; i < VD; i++) d[h * VD + i] = g[i];
                    }
                }
#pragma unroll
                for (int q0 = 0; q0 < UB_JB; q0 += 4) {
                    uint4 u[4];
                    if (dwt) {
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            if (q0 + q < jn) u[q] = ld16(y + (size_t)s.row[j0 + q0 + q] * H + (size_t)c * V);
                    }
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int a = q0 + q;
                        if (a >= jn) continue;
                        float f[V];
                        if (dwt) {
                            Vec<T>::get(u[q], f);
#pragma unroll
                            for (int i = 0; i < V; i++) dot[a] = fmaf(d[i], f[i], dot[a]);
                        }
                        if (dy) {
                            const float w = s.w[j0 + a];
#pragma unroll
                            for (int i = 0; i < V; i++) f[i] = w * d[i];
                            st16(dy + (size_t)s.row[j0 + a] * H + (size_t)c * V, Vec<T>::put(f));
                        }
                    }
                }
            }
        } else {
            constexpr int U = UB_U;
            const int th = blockDim.x;
            for (int c0 = threadIdx.x; c0 < H; c0 += th * U) {
                float d[U];
                T f[UB_JB][U];
#pragma unroll
                for (int i = 0; i < U; i++) d[i] = c0 + i * th < H ? Vec<D>::one(dr[c0 + i * th]) : 0.0f;
                if (dwt) {
#pragma unroll
                    for (int q = 0; q < UB_JB; q++) {
                        const T *r = y + (size_t)s.row[j0 + (q < jn ? q : 0)] * H;
#pragma unroll
                        for (int i = 0; i < U; i++)
                            if (q < jn && c0 + i * th < H) f[q][i] = r[c0 + i * th];
                    }
                }
#pragma unroll
                for (int q = 0; q < UB_JB; q++) {
                    if (q >= jn) continue;
                    T *r = dy + (size_t)s.row[j0 + q] * H;
                    const float w = s.w[j0 + q];
#pragma unroll
                    for (int i = 0; i < U; i++)
                        if (c0 + i * th < H) {
                            if (dwt) dot[q] = fmaf(d[i], Vec<T>::one(f[q][i]), dot[q]);
                            if (dy) r[c0 + i * th] = Vec<T>::back(w * d[i]);
                        }
                }
            }
        }
        if (dwt) {
#pragma unroll
            for (int q = 0; q < UB_JB; q++) {
                const float v = warp_sum(dot[q]);
                if (lane == 0) part[warp][q] = v;
            }
            __syncthreads();
            if ((int)threadIdx.x < jn) {
                float v = 0.0f;
                for (int w2 = 0; w2 < (int)blockDim.x / 32; w2++) v += part[w2][threadIdx.x];
                dwt[p0 + s.j[j0 + threadIdx.x]] = v;
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------ quantising permute
// One thread per 32-element group of a token: read and quantised once, its 16 bytes of codes
// and its scale byte stored into each of the token's rows. Bound by HBM: 4096 x 8 rows of 7168 in
// 32 us, 5.8 TB/s (the permute and a quantisation of its rows: 88 + 93), 66 us with x on odd addresses.
template <typename T>
__global__ void __launch_bounds__(PM_TH) k_permute_mx4(uint8_t *__restrict__ packed, uint8_t *__restrict__ scales,
                                                       const T *__restrict__ x, int64_t ldx,
                                                       const int *__restrict__ pos, int P, int topk, int H, int vec) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ TokenRows s;
    const int t = blockIdx.x, G = H / 32;
    const int m = token_rows(s, pos, nullptr, (size_t)t * topk, P, topk);
    if (!m) return;
    for (int g = blockIdx.y * blockDim.x + threadIdx.x; g < G; g += gridDim.y * blockDim.x) {
        float v[32];
        mx4_load32(v, x + (size_t)t * ldx + (size_t)g * 32, 32, vec);
        uint4 codes;
        const uint8_t sb = mx4_quant32(v, codes);
        for (int j = 0; j < m; j++) {
            const int r = s.row[j];
            *reinterpret_cast<uint4 *>(packed + (size_t)r * (H / 2) + (size_t)g * 16) = codes;
            scales[(size_t)r * G + g] = sb;
        }
    }
}

// ------------------------------------------------------------------ host side
bool al16(const void *p) { return ((uintptr_t)p & 15) == 0; }
bool known(int dt) { return dt == K3C_F32 || dt == K3C_BF16; }
size_t size_of(int dt) { return dt == K3C_F32 ? 4 : 2; }

// Grid and block for ntok rows of `units` pieces: blocks along a row while there are fewer than two
// per SM, and threads so that each takes the same number of pieces (rows of 14 KB: 448 threads
// move 8 copies of 4096 tokens in 87 us, 256 in 91, 128 in 95).
struct Shape {
    dim3 grid, block;
};
Shape row_shape(int ntok, int units, bool split) {
    int gy = split ? (2 * 148 + ntok - 1) / ntok : 1;
    const int most = (units + 127) / 128;
    gy = gy > most ? most : gy;
    const int per = (units + gy - 1) / gy, rounds = (per + PM_TH - 1) / PM_TH;
    const int th = ((per + rounds - 1) / rounds + 31) / 32 * 32;
    return {dim3(ntok, gy), dim3(th)};
}

int check_pairs(const char *what, int ntok, int topk, int hidden) {
    if (ntok < 0 || topk < 1 || topk > K3_MAX_TOPK || hidden < 1 || hidden > 1 << 28)
        return set_error(K3C_EINVAL, "%s: ntok=%d topk=%d (1..%d) hidden=%d", what, ntok, topk, K3_MAX_TOPK, hidden);
    if ((int64_t)ntok * topk > 0x7FFFFFFF - 2 * SORT_BLOCKS * SORT_SUB)
        return set_error(K3C_EINVAL, "%s: %d x %d pairs exceed 32 bits", what, ntok, topk);
    return K3C_OK;
}

// One block as far as its warps' registers reach: a second launch costs more than the other SMs
// save. Beyond that, blocks of one pass or more.
int sort_blocks(int64_t P) {
    if (P <= SORT_ONE * SORT_TH) return 1;
    const int64_t n = (P + SORT_SUB - 1) / SORT_SUB;
    return (int)(n < SORT_BLOCKS ? n : SORT_BLOCKS);
}

template <typename T, typename O>
int run_gather(O *out, const T *y, const float *wt, const int *pos, int ntok, int topk, int H, cudaStream_t s) {
    const bool vec = al16(y) && al16(out) && H % Vec<T>::V == 0 && H % Vec<O>::V == 0;
    const Shape g = row_shape(ntok, vec ? H / Vec<T>::V : (H + PM_U - 1) / PM_U, true);
    if (vec) k_gather_sum<T, O, true><<<g.grid, g.block, 0, s>>>(out, y, wt, pos, ntok * topk, topk, H);
    else k_gather_sum<T, O, false><<<g.grid, g.block, 0, s>>>(out, y, wt, pos, ntok * topk, topk, H);
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

template <typename T, typename D>
int run_unpermute_bwd(T *dy, float *dwt, const D *dout, const T *y, const float *wt, const int *pos, int ntok, int topk,
                      int H, cudaStream_t s) {
    const bool vec = al16(y) && al16(dy) && al16(dout) && H % Vec<T>::V == 0 && H % Vec<D>::V == 0;
    const Shape g = row_shape(ntok, vec ? H / Vec<T>::V : (H + UB_U - 1) / UB_U, false);   // one block per token: it sums dwt
    if (vec) k_unpermute_bwd<T, D, true><<<g.grid, g.block, 0, s>>>(dy, dwt, dout, y, wt, pos, ntok * topk, topk, H);
    else k_unpermute_bwd<T, D, false><<<g.grid, g.block, 0, s>>>(dy, dwt, dout, y, wt, pos, ntok * topk, topk, H);
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

}  // namespace
}  // namespace k3c

using namespace k3c;

extern "C" size_t k3c_moe_sort_scratch(int ntok, int topk, int n_experts) {
    if (ntok <= 0 || topk <= 0 || n_experts <= 0) return 0;
    const int nb = sort_blocks((int64_t)ntok * topk);
    return nb == 1 ? 0 : (size_t)nb * n_experts * sizeof(int);
}

extern "C" int k3c_moe_sort(int *pos, int *pair, int *off, const int *idx, int ntok, int topk, int n_experts,
                            void *scratch, size_t scratch_bytes, k3c_stream_t stream) {
    clear_error();
    K3C_TRY(check_pairs("moe_sort", ntok, topk, 1));
    if (n_experts < 1 || n_experts > SORT_EMAX)
        return set_error(K3C_EINVAL, "moe_sort: n_experts=%d (1..%d)", n_experts, SORT_EMAX);
    if (!off || (ntok && (!pos || !pair || !idx))) return set_error(K3C_EINVAL, "moe_sort: NULL array");
    const size_t need = k3c_moe_sort_scratch(ntok, topk, n_experts);
    if (need && (!scratch || scratch_bytes < need || ((uintptr_t)scratch & 3)))
        return set_error(K3C_EINVAL, "moe_sort: scratch of %zu bytes, %zu needed (4-byte aligned)", scratch_bytes, need);
    cudaStream_t s = (cudaStream_t)stream;
    const int P = ntok * topk, nblk = sort_blocks(P);
    static bool attr_of[64] = {};
    bool &attr = attr_of[cur_dev()];
    if (!attr) {
        const int most = SORT_EMAX * (int)(sizeof(int) + SORT_WARPS * sizeof(uint16_t));
        K3C_TRY_CUDA(cudaFuncSetAttribute(k_sort_one, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        K3C_TRY_CUDA(cudaFuncSetAttribute(k_sort_place, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        attr = true;
    }
    auto table = [&](int warps) { return (size_t)n_experts * sizeof(int) + ((size_t)n_experts * warps + 1) / 2 * 4; };
    if (nblk == 1) {
        const int warps = (P + SORT_ONE * 32 - 1) / (SORT_ONE * 32);
        k_sort_one<<<1, SORT_TH, table(warps), s>>>(pos, pair, off, idx, P, n_experts, warps);
        K3C_CHECK_LAUNCH();
        return K3C_OK;
    }
    const int64_t n = ((int64_t)P + SORT_SUB - 1) / SORT_SUB;
    const int chunk = (int)((n + nblk - 1) / nblk) * SORT_SUB;
    k_sort_count<<<nblk, SORT_TH, n_experts * sizeof(int), s>>>((int *)scratch, idx, P, n_experts, chunk);
    K3C_CHECK_LAUNCH();
    K3C_TRY_CUDA(launch_pdl(k_sort_place, dim3(nblk), dim3(SORT_TH), table(SORT_WARPS), s, pos, pair, off, idx,
                            (const int *)scratch, P, n_experts, chunk));
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

extern "C" int k3c_moe_permute(void *rows, const void *x, int dtype, int64_t ldx, const int *pos, int ntok, int topk,
                               int hidden, k3c_stream_t stream) {
    clear_error();
    K3C_TRY(check_pairs("moe_permute", ntok, topk, hidden));
    if (!known(dtype) || ldx < hidden) return set_error(K3C_EINVAL, "moe_permute: dtype=%d ldx=%lld", dtype, (long long)ldx);
    if (!ntok) return K3C_OK;
    if (!rows || !x || !pos) return set_error(K3C_EINVAL, "moe_permute: NULL array");
    cudaStream_t s = (cudaStream_t)stream;
    const int V = dtype == K3C_F32 ? 4 : 8, P = ntok * topk;
    const bool vec = al16(rows) && al16(x) && hidden % V == 0 && ldx % V == 0;
    const Shape g = row_shape(ntok, vec ? hidden / V : (hidden + PM_U - 1) / PM_U, true);
    if (dtype == K3C_F32) {
        if (vec) k_permute<float, true><<<g.grid, g.block, 0, s>>>((float *)rows, (const float *)x, ldx, pos, P, topk, hidden);
        else k_permute<float, false><<<g.grid, g.block, 0, s>>>((float *)rows, (const float *)x, ldx, pos, P, topk, hidden);
    } else {
        if (vec) k_permute<uint16_t, true><<<g.grid, g.block, 0, s>>>((uint16_t *)rows, (const uint16_t *)x, ldx, pos, P, topk, hidden);
        else k_permute<uint16_t, false><<<g.grid, g.block, 0, s>>>((uint16_t *)rows, (const uint16_t *)x, ldx, pos, P, topk, hidden);
    }
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

extern "C" int k3c_moe_permute_bwd(void *dx, const void *drows, int dtype, const int *pos, int ntok, int topk, int hidden,
                                   k3c_stream_t stream) {
    clear_error();
    K3C_TRY(check_pairs("moe_permute_bwd", ntok, topk, hidden));
    if (!known(dtype)) return set_error(K3C_EINVAL, "moe_permute_bwd: dtype=%d", dtype);
    if (!ntok) return K3C_OK;
    if (!dx || !drows || !pos) return set_error(K3C_EINVAL, "moe_permute_bwd: NULL array");
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == K3C_F32) return run_gather((float *)dx, (const float *)drows, nullptr, pos, ntok, topk, hidden, s);
    return run_gather((uint16_t *)dx, (const uint16_t *)drows, nullptr, pos, ntok, topk, hidden, s);
}

extern "C" int k3c_moe_permute_mxfp4(uint8_t *packed, uint8_t *scales, const void *x, int x_dtype, int64_t ldx,
                                     const int *pos, int ntok, int topk, int hidden, k3c_stream_t stream) {
    clear_error();
    K3C_TRY(check_pairs("moe_permute_mxfp4", ntok, topk, hidden));
    if (!known(x_dtype) || ldx < hidden || hidden % 32)
        return set_error(K3C_EINVAL, "moe_permute_mxfp4: dtype=%d ldx=%lld hidden=%d (a multiple of 32)", x_dtype,
                         (long long)ldx, hidden);
    if (!ntok) return K3C_OK;
    if (!packed || !scales || !x || !pos) return set_error(K3C_EINVAL, "moe_permute_mxfp4: NULL array");
    if (!al16(packed)) return set_error(K3C_EINVAL, "moe_permute_mxfp4: packed must be 16-byte aligned");
    cudaStream_t s = (cudaStream_t)stream;
    const Shape g = row_shape(ntok, hidden / 32, true);
    const int vec = al16(x) && (ldx * size_of(x_dtype)) % 16 == 0;
    if (x_dtype == K3C_F32)
        k_permute_mx4<<<g.grid, g.block, 0, s>>>(packed, scales, (const float *)x, ldx, pos, ntok * topk, topk, hidden, vec);
    else
        k_permute_mx4<<<g.grid, g.block, 0, s>>>(packed, scales, (const uint16_t *)x, ldx, pos, ntok * topk, topk, hidden, vec);
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

extern "C" int k3c_moe_unpermute(void *out, int out_dtype, const void *y, int y_dtype, const float *wt, const int *pos,
                                 int ntok, int topk, int hidden, k3c_stream_t stream) {
    clear_error();
    K3C_TRY(check_pairs("moe_unpermute", ntok, topk, hidden));
    if (!known(out_dtype) || !known(y_dtype))
        return set_error(K3C_EINVAL, "moe_unpermute: out_dtype=%d y_dtype=%d", out_dtype, y_dtype);
    if (!ntok) return K3C_OK;
    if (!out || !y || !wt || !pos) return set_error(K3C_EINVAL, "moe_unpermute: NULL array");
    cudaStream_t s = (cudaStream_t)stream;
    if (y_dtype == K3C_F32) {
        if (out_dtype == K3C_F32) return run_gather((float *)out, (const float *)y, wt, pos, ntok, topk, hidden, s);
        return run_gather((uint16_t *)out, (const float *)y, wt, pos, ntok, topk, hidden, s);
    }
    if (out_dtype == K3C_F32) return run_gather((float *)out, (const uint16_t *)y, wt, pos, ntok, topk, hidden, s);
    return run_gather((uint16_t *)out, (const uint16_t *)y, wt, pos, ntok, topk, hidden, s);
}

extern "C" int k3c_moe_unpermute_bwd(void *dy, float *dwt, const void *dout, int out_dtype, const void *y, int y_dtype,
                                     const float *wt, const int *pos, int ntok, int topk, int hidden,
                                     k3c_stream_t stream) {
    clear_error();
    K3C_TRY(check_pairs("moe_unpermute_bwd", ntok, topk, hidden));
    if (!known(out_dtype) || !known(y_dtype))
        return set_error(K3C_EINVAL, "moe_unpermute_bwd: out_dtype=%d y_dtype=%d", out_dtype, y_dtype);
    if (!ntok || (!dy && !dwt)) return K3C_OK;
    if (!dout || !wt || !pos || (dwt && !y)) return set_error(K3C_EINVAL, "moe_unpermute_bwd: NULL array");
    cudaStream_t s = (cudaStream_t)stream;
    if (y_dtype == K3C_F32) {
        if (out_dtype == K3C_F32)
            return run_unpermute_bwd((float *)dy, dwt, (const float *)dout, (const float *)y, wt, pos, ntok, topk, hidden, s);
        return run_unpermute_bwd((float *)dy, dwt, (const uint16_t *)dout, (const float *)y, wt, pos, ntok, topk, hidden, s);
    }
    if (out_dtype == K3C_F32)
        return run_unpermute_bwd((uint16_t *)dy, dwt, (const float *)dout, (const uint16_t *)y, wt, pos, ntok, topk, hidden, s);
    return run_unpermute_bwd((uint16_t *)dy, dwt, (const uint16_t *)dout, (const uint16_t *)y, wt, pos, ntok, topk, hidden, s);
}
