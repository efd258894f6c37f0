// mxfp4_mm.cu -- MXFP4 quantisation, the product of two MXFP4 matrices, and the product's
// gradient with respect to its activations. No reference counterpart (the reference multiplies
// fp32 activations with packed weights, src/core/k3_ops.c:1363-1768); the packed formats are the
// reference's (E2M1 nibbles, low nibble even; one E8M0 byte per 32 elements).
//
//   quant   x -> (codes [rows][in/2], scales [rows][ceil(in/32)])            mx4_quant.cuh
//   pack    a weight's scales re-ordered into 512-byte atoms of 128 rows x 4 groups, which
//           tcgen05.cp copies to TMEM as they are; scale 255 (the reference: skip the group)
//           becomes zero codes under scale 127, as in the pool format
//   mm      y[r][o] = sum_i A[r][i] W_g[o][i]: E2M1 x E2M1 on tcgen05.mma kind::mxf4 with both
//           block scales applied by the MMA, fp32 accumulation, one rounding to y's type.
//           Rows [off[g], off[g+1]) of A multiply matrix g (grouped by expert), or all rows
//           one matrix.
//   mm_bwd  dA[r][i] = sum_o dY[r][o] W_g[o][i]: the contraction runs over W's rows, which the
//           4-bit MMA cannot read (it wants the contracted index contiguous), so W tiles are
//           widened to bf16 in shared memory (exact: two significant bits and a power of two)
//           and multiplied by kind::f16, fp32 accumulation.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdlib.h>

#include <type_traits>

#include "common.cuh"
#include "mx4_quant.cuh"
#include "tc_common.cuh"
#include "tc_host.cuh"

namespace k3c {

namespace {

constexpr int MX_DIM = 0x7FFFFFFF - 1023;   // rows and columns at most: sums with a tile's stay within 32 bits
constexpr int MX_GMAX = 1024;   // groups of a product: with more, the largest tiles' shared memory would not hold the Plan

static __device__ int g_mx_err;

// One lane of a converged warp. The compiler knows a branch on elect.sync to be taken by one
// thread; behind `lane == 0` it guards every tcgen05 and TMA instruction's uniform operands
// against several (~100 cycles an instruction: the copy and MMA loops below ran 3x slower).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ------------------------------------------------------------------ quantisation
// Rows of whole groups on 16-byte boundaries: four lanes share a group, so that a warp's loads and
// stores are contiguous (with a lane per group, 64 bytes apart, L1 was 72% busy and DRAM 56%).
// Bound by HBM: 8192 x 7168 bf16 in 24.3 us, 6.1 TB/s.
// QUANT_U pieces of 8 elements per thread, all loaded first. DENSE: rows lie side by side.
constexpr int QUANT_U = 4;
template <typename T, bool DENSE>
__global__ void __launch_bounds__(256) k_mx4_quant(uint8_t *__restrict__ packed, uint8_t *__restrict__ scales,
                                                   const T *__restrict__ x, int64_t ldx, int rows, int in) {
    grid_dep_launch();
    constexpr int L = sizeof(T) / 2;             // 16-byte loads per piece
    const size_t per = in / 8, n = (size_t)rows * per;
    for (size_t b0 = (size_t)blockIdx.x * (256 * QUANT_U); b0 < n; b0 += (size_t)gridDim.x * (256 * QUANT_U)) {   // whole blocks
        const size_t i0 = b0 + threadIdx.x;
        uint4 u[QUANT_U][L];
#pragma unroll
        for (int k = 0; k < QUANT_U; k++) {
            const size_t i = i0 + 256 * k;
            if (i < n) {
                const T *src = DENSE ? x + i * 8 : x + (i / per) * ldx + (i % per) * 8;
#pragma unroll
                for (int l = 0; l < L; l++) u[k][l] = ldg_nc_v4(src + 8 / L * l);
            }
        }
#pragma unroll
        for (int k = 0; k < QUANT_U; k++) {
            const size_t i = i0 + 256 * k;
            float f[8];   // of a piece past the end: nothing is stored
            if constexpr (L == 1) {
                const uint32_t w[4] = {u[k][0].x, u[k][0].y, u[k][0].z, u[k][0].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    f[2 * j] = __uint_as_float(w[j] << 16);
                    f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
                }
            } else {
#pragma unroll
                for (int l = 0; l < L; l++) {
                    f[4 * l] = __uint_as_float(u[k][l].x);
                    f[4 * l + 1] = __uint_as_float(u[k][l].y);
                    f[4 * l + 2] = __uint_as_float(u[k][l].z);
                    f[4 * l + 3] = __uint_as_float(u[k][l].w);
                }
            }
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(f[j]) & 0x7FFFFFFFu);
            // n and the strides are multiples of four pieces: a group's lanes are all here or all not
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (i >= n) continue;
            const uint32_t byte = mx4_scale_byte(top);
            const float m = mx4_multiplier(byte);
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] *= m;
            reinterpret_cast<uint32_t *>(packed)[i] = byte == 255 ? 0u : f32x8_to_e2m1(f);
            if ((threadIdx.x & 3) == 0) scales[i / 4] = (uint8_t)byte;
        }
    }
}

// Any other rows: one thread per group. Bound by its loads of single elements and stores of single bytes:
// 8192 x 7168 bf16 on odd addresses 128 us (1.2 TB/s), 8192 x 7166 134.
template <typename T>
__global__ void __launch_bounds__(256) k_mx4_quant_any(uint8_t *__restrict__ packed, uint8_t *__restrict__ scales,
                                                       const T *__restrict__ x, int64_t ldx, int rows, int in) {
    grid_dep_launch();
    const int G = (in + 31) / 32;
    const size_t n = (size_t)rows * G;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t r = i / G;
        const int g = (int)(i - r * G), left = min(32, in - 32 * g);
        float v[32];
        mx4_load32(v, x + r * ldx + (size_t)g * 32, left, 0);
        uint4 c;
        scales[i] = mx4_quant32(v, c);
        uint8_t *d = packed + r * (in / 2) + (size_t)g * 16;
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int b = 0; b < 16; b++)
            if (2 * b < left) d[b] = (uint8_t)(w[b >> 2] >> (8 * (b & 3)));
    }
}

// An epilogue's wait for its item's sums. They take as long as the item's K blocks do, 0.2 to 0.6 us each: 10 s for a
// gradient over 2^31 weight rows, so the limit grows with them (with the other waits' 2 s that
// gradient was NaN from 430 million rows on).
__device__ __forceinline__ bool wait_for_sums(uint64_t *bar, uint32_t parity, int *err, int code, int k_blocks) {
    return tc::mbar_wait_ns(bar, parity, err, code, tc::kWaitLimitNs + 2000ull * (uint32_t)k_blocks);
}

// Byte of row m (0..127), group g (0..3) in a scale atom.
__device__ __forceinline__ int sf_byte(int m, int g) { return 16 * (m & 31) + 4 * (m >> 5) + g; }

// One thread per group of the padded matrix: scale byte into its atom, codes copied (packed and
// codes may be the same array). Done once per weight: 48 matrices of 4096 x 7168 in 260 us, 5.8 TB/s.
__global__ void __launch_bounds__(256) k_mx4_pack(uint8_t *codes, uint8_t *__restrict__ atoms, const uint8_t *packed,
                                                  const uint8_t *__restrict__ scales, int n_mats, int rows, int in) {
    const int G = in / 32, RA = (rows + 127) / 128, KA = (in + 127) / 128;
    const size_t per = (size_t)RA * 128 * KA * 4, n = per * n_mats;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t m = i / per, q = i - m * per;
        const int r = (int)(q / (KA * 4)), g = (int)(q % (KA * 4));
        uint8_t sb = 127;
        if (r < rows && g < G) {
            const size_t row = m * rows + r;
            sb = scales[row * G + g];
            uint4 c = *reinterpret_cast<const uint4 *>(packed + row * (in / 2) + (size_t)g * 16);
            if (sb == 255) {
                c = make_uint4(0, 0, 0, 0);
                sb = 127;
            }
            *reinterpret_cast<uint4 *>(codes + row * (in / 2) + (size_t)g * 16) = c;
        }
        atoms[((m * RA + r / 128) * KA + g / 4) * 512 + sf_byte(r & 127, g & 3)] = sb;
    }
}

// ------------------------------------------------------------------ work items
// Groups own consecutive rows; an item is one row tile of one group x one column tile.
struct Item {
    int mat;         // matrix index, -1: none (the rows' results are zeros)
    int row0, n;     // first row, rows of the tile
    int nt;          // column tile
};

// The groups' tiles, in shared memory: group g has row tiles tile[g] .. tile[g+1] - 1.
struct Plan {
    int tile[MX_GMAX + 1], warp_tot[32];
};

// Group g's first row; its rows end before group g + 1's. Offsets cannot leave the rows.
__device__ __forceinline__ int first_of(const int *off, int g, int M) {
    return off ? min(max(__ldg(off + g), 0), M) : g ? M : 0;
}

// Row tiles of at most `tile` rows that n_groups groups of M rows can have together.
__host__ __device__ __forceinline__ int64_t most_tiles(int M, int n_groups, int tile) {
    return (int64_t)M / tile + (n_groups < M ? n_groups : M);
}

// Filled by all THREADS of the block; returns the number of row tiles. Ascending offsets have no more than
// most_tiles of them. Offsets that descend in places can name the same rows again and again (0, M, 0, M, ...: 512
// times M), more tiles than 32 bits count and items than the launch was checked for: tiles past
// most_tiles are left out, so that every sum here and in a Walk stays within what the host has checked.
template <int THREADS>
__device__ int plan_tiles(Plan &pl, const int *off, int G, int M, int rows) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (!off) {
        const int n = (M + rows - 1) / rows;
        if (tid == 0) {
            pl.tile[0] = 0;
            pl.tile[1] = n;
        }
        __syncthreads();
        return n;
    }
    const int most = (int)most_tiles(M, G, rows);
    int run = 0;
    for (int g0 = 0; g0 < G; g0 += THREADS) {
        const int g = g0 + tid;
        const int n = g < G ? (max(first_of(off, g + 1, M) - first_of(off, g, M), 0) + rows - 1) / rows : 0;
        int inc = n;   // n < 2^25: a warp's sum stays below 2^30
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) pl.warp_tot[warp] = inc;
        __syncthreads();
        int pre = run, all = run;
#pragma unroll
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) pre = min(pre + pl.warp_tot[w], most);
            all = min(all + pl.warp_tot[w], most);
        }
        if (g < G) pl.tile[g] = min(pre + inc - n, most);
        run = all;
        __syncthreads();
    }
    if (tid == 0) pl.tile[G] = run;
    __syncthreads();
    return run;
}

// Items of a group run through its row tiles first, MX_RB of them at a time, so that the CTAs
// working side by side share W tiles and a bounded set of A rows in L2. A Walk turns ascending
// item numbers into items; it keeps the group at hand, since a search with its divisions (1500
// cycles for one thread) at every item left the copies that far behind.
constexpr int MX_RB = 16;
struct Walk {
    const Plan &pl;
    const int *off, *mat_of;
    int M, n_mats, G, NTL, rows;
    int g = -1, lo = 0, hi = 0;    // items lo .. hi - 1 belong to group g
    int mt = 0, f0 = 0, f1 = 0, mat = -1;
    __device__ __forceinline__ Item at(int it) {
        if (it >= hi) {
            int a = g + 1, b = G;   // tile[a] * NTL <= it < tile[b] * NTL
            while (b - a > 1) {
                const int c = (a + b) >> 1;
                if (pl.tile[c] * NTL <= it) a = c;
                else b = c;
            }
            g = a;
            mt = pl.tile[g + 1] - pl.tile[g];
            lo = pl.tile[g] * NTL;
            hi = pl.tile[g + 1] * NTL;
            f0 = first_of(off, g, M);
            f1 = first_of(off, g + 1, M);
            mat = mat_of ? __ldg(mat_of + g) : g;
            if (mat < 0 || mat >= n_mats) mat = -1;
        }
        int i = it - lo, m = 0, mb = mt;
        if (mt > MX_RB) {
            const int b = i / (MX_RB * NTL);
            m = MX_RB * b;
            mb = min(MX_RB, mt - m);
            i -= m * NTL;
        }
        Item x;
        x.mat = mat;
        x.nt = mb == 1 ? i : i / mb;
        m += i - x.nt * mb;
        x.row0 = f0 + m * rows;
        x.n = min(rows, f1 - x.row0);
        return x;
    }
};

struct MxArgs {
    void *y;
    int64_t ldy;
    int y_bf16, vec;             // vec: rows of y start on 16-byte boundaries
    int M, N, K, G, NTL;         // A [M][K], W [N][K]
    const int *off, *mat_of;
    int n_mats;
    const uint8_t *as;           // A's scales [M][K/32]
    const uint8_t *atoms;        // W's scale atoms, atom_stride bytes per matrix
    size_t atom_stride;
    int *err;
};

// 32 * NC columns of 32 rows (a warp's share of the accumulator, a row per lane) to y: staged in 2 KB of
// shared memory, 64 bytes of a row at a time with the 16-byte pieces rotated by the row, and stored
// by four lanes per row, 8 rows x 64 bytes a store. rows: valid rows of the 32; c0: first column.
// (With types, addresses and strides worked out at every store a 32 x 32 piece took 1000
// cycles: 2000 x 4096 x 64 in 13.5 us, 12.3 now, and in rows on odd addresses, 2000 x 4095 x 2048, 26.5
// and 18.6.)
template <bool BF16, int NC>
__device__ __forceinline__ void store_rows_as(uint8_t *stg, uint32_t (&v)[NC][32], const MxArgs &p, int64_t row, int rows,
                                              int c0) {
    constexpr int ESZ = BF16 ? 2 : 4, PER = 64 / ESZ;   // columns per 64-byte piece
    const int lane = threadIdx.x & 31;
    const uint32_t sw = (lane >> 1) & 3;
    uint8_t *put = stg + lane * 64;
    const int r = lane >> 2, k = lane & 3;
    const int64_t ld = p.ldy * ESZ;
    char *d = reinterpret_cast<char *>(p.y) + row * ld + (int64_t)c0 * ESZ;
    char *dv = d + r * ld + k * 16;
#pragma unroll
    for (int h = 0; h < 32 * NC / PER; h++) {
        const int c = c0 + h * PER;
        if (c >= p.N) break;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint4 o;
            if constexpr (BF16) {
                const uint32_t *q = v[h] + 8 * i;
                o = make_uint4(f32x2_to_bf16x2(__uint_as_float(q[0]), __uint_as_float(q[1])),
                               f32x2_to_bf16x2(__uint_as_float(q[2]), __uint_as_float(q[3])),
                               f32x2_to_bf16x2(__uint_as_float(q[4]), __uint_as_float(q[5])),
                               f32x2_to_bf16x2(__uint_as_float(q[6]), __uint_as_float(q[7])));
            } else {
                const uint32_t *q = v[h / 2] + 16 * (h & 1) + 4 * i;
                o = make_uint4(q[0], q[1], q[2], q[3]);
            }
            *reinterpret_cast<uint4 *>(put + 16 * (i ^ sw)) = o;
        }
        __syncwarp();
        if (p.vec && c + PER <= p.N) {
            // rows r, r + 8, r + 16, r + 24: the rotation (r >> 1) & 3 is the same for all four
            const uint8_t *get = stg + r * 64 + 16 * (k ^ ((r >> 1) & 3));
#pragma unroll
            for (int i = 0; i < 4; i++) {   // one by one: in bursts they delay the next item's copies (3%)
                const uint4 o = *reinterpret_cast<const uint4 *>(get + 512 * i);
                if (r + 8 * i < rows) *reinterpret_cast<uint4 *>(dv + 8 * i * ld + 64 * h) = o;
            }
        } else {
            // element by element, a row's columns side by side: 32 lanes on one row of bf16 or two of fp32
            using E = typename std::conditional<BF16, uint16_t, uint32_t>::type;
            constexpr int RS = 32 / PER;
            const int e = lane % PER, r0 = lane / PER, at = e * ESZ;
            E *de = reinterpret_cast<E *>(d + r0 * ld + 64 * h) + e;
            const bool col = c + e < p.N;
#pragma unroll 8
            for (int i = 0; i < 32 / RS; i++) {
                const int ri = RS * i + r0;
                const E x = *reinterpret_cast<const E *>(stg + ri * 64 + 16 * ((at >> 4) ^ ((ri >> 1) & 3)) + (at & 15));
                if (ri < rows && col) *reinterpret_cast<E *>(reinterpret_cast<char *>(de) + (int64_t)(RS * i) * ld) = x;
            }
        }
    }
}
template <int NC>
__device__ __forceinline__ void store_rows(uint8_t *stg, uint32_t (&v)[NC][32], const MxArgs &p, int64_t row, int rows,
                                           int c0, bool ok) {
    if (!ok) {   // a wait gave up
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 32; i++) v[c][i] = 0x7FC00000u;
    }
    if (p.y_bf16) store_rows_as<true, NC>(stg, v, p, row, rows, c0);
    else store_rows_as<false, NC>(stg, v, p, row, rows, c0);
}

// ------------------------------------------------------------------ MXFP4 x MXFP4
// kind::mxf4: E2M1 A and B, K-major, UE8M0 scales per 32 (scale_vec::2X), M = 128, K = 64.
__host__ __device__ constexpr uint32_t idesc_mxf4(uint32_t n, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((128u >> 4) << 24) | (sf_id << 29);
}
__device__ __forceinline__ void tc_mma_mx4(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa,
                                           uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
}

constexpr int MM_M = 128;
constexpr int MM_ABOX = 32;                      // rows per A copy of a short tile; a full one takes one copy
constexpr int MM_A = MM_M * 128;                 // 128 rows x 256 codes
constexpr int MM_THREADS = 384;                  // warps: W copies, MMA, A scales, A copies, 8 of epilogue
constexpr int MM_EPI = 8;
constexpr int MM_KS = 4;                         // K blocks per fetch of A scales: one 32-byte sector a row
template <int NT>
struct MmCfg {
    static constexpr int B = NT * 128;
    static constexpr int NA = NT / 128 ? NT / 128 : 1;    // 128-row scale atoms of a column tile
    static constexpr int SF = 1024 + NA * 1024;           // A's and W's scales of 256 elements
    static constexpr int STAGE = MM_A + B + SF;
    static constexpr int STAGES = NT == 256 ? 4 : NT == 128 ? 6 : 7;
    static constexpr int NACC = NT == 256 ? 1 : 2;        // accumulators in TMEM
    static constexpr uint32_t SFW = 2 * (4 + 4 * NA);     // TMEM columns of a stage's scales
    static constexpr uint32_t SF_COL = NT * NACC;
    static constexpr int BAR = 256;
    static constexpr int BYTES = 1024 + STAGES * STAGE + BAR + MM_EPI * 2048;
    static_assert(STAGE % 1024 == 0, "stage bases stay 1024-byte aligned");
    static_assert(SF_COL + STAGES * SFW <= 512, "TMEM columns");
    static_assert(BYTES + sizeof(Plan) + 64 <= 227 * 1024, "one CTA per SM");
    static_assert((2 * STAGES + 2 * NACC) * 8 + 4 <= BAR, "barriers");
};

// A's codes of every K block of this CTA's items, by one thread, to sa0 in stage 0; item(it) gives
// the rows of this CTA. (With W's copies in the same thread a stage took 440 cycles to issue, as
// long as its MMAs: after a stall the copies never got ahead again.)
template <int STAGES, typename ItemFn>
__device__ __forceinline__ void copy_a(const MxArgs &p, int n_items, const ItemFn &item, const CUtensorMap &tmA,
                                       const CUtensorMap &tmA1, uint8_t *sa0, int stage_bytes, uint64_t *full,
                                       uint64_t *empty, int KB, int it0, int step) {
    uint32_t n = 0, st = 0, ph = 1;
    bool ok = true;
    for (int it = it0; ok && it < n_items; it += step) {
        const Item x = item(it);
        if (x.mat < 0) continue;
        const int boxes = (x.n + MM_ABOX - 1) / MM_ABOX;
        for (int kb = 0; kb < KB; kb++, n++) {
            if (!tc::mbar_wait(&empty[st], ph, p.err, 87)) { ok = false; break; }
            uint8_t *sa = sa0 + st * stage_bytes;
            tc::mbar_expect_tx(&full[st], boxes * MM_ABOX * 128);
            if (boxes == MM_M / MM_ABOX) tc::tma_load_3d(sa, &tmA, &full[st], kb * 128, x.row0, 0);
            else
                for (int b = 0; b < boxes; b++)
                    tc::tma_load_3d(sa + b * (MM_ABOX * 128), &tmA1, &full[st], kb * 128, x.row0 + b * MM_ABOX, 0);
            if (++st == STAGES) {
                st = 0;
                ph ^= 1u;
            }
        }
    }
    for (uint32_t i = n > STAGES ? n - STAGES : 0; i < n; i++)
        tc::mbar_wait(&full[i % STAGES], (i / STAGES) & 1u, p.err, 88);
}

// The scale bytes of four rows and MM_KS K blocks (32 bytes a row) as one lane holds them: the aligned
// 16-byte pieces they lie in, whatever the row's alignment, as loaded. They are shifted into words
// only when the K blocks before them are stored: right after the loads the shift would wait for
// them (8192 x 7168 x 7136: 315 us then, 196 now; 178 with a K of 7168).
// EVEN: every row starts on a piece.
template <bool EVEN>
struct ScaleRows {
    uint4 u[4][EVEN ? 2 : 3];
    uint32_t off[4];    // the rows' first byte within their first piece
};
// The 16 bytes at c of an array [lo, hi), zeros outside it: each of 16 lanes has loaded one byte.
__device__ __forceinline__ uint4 edge_piece(uint32_t byte, int at) {   // at: the byte's place, -1 for none
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; k++) w[k] = __reduce_or_sync(0xFFFFFFFFu, at >> 2 == k ? byte << (8 * (at & 3)) : 0u);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A's scales of every K block of this CTA's items, by one warp. Lane i fetches the bytes of rows i,
// 32+i, 64+i and 96+i and stores the four rows' words of each atom as one 16-byte piece (sf_byte's
// order). MM_KS K blocks are fetched at a time, while the MM_KS before them are stored, across
// items. The stores become visible to tcgen05.cp by a proxy fence of the thread that waits on
// `full`: one here would wait for the fetches in flight. sf0: the scales' place in stage 0; item(it)
// gives the rows of this CTA.
template <int STAGES, bool EVEN, typename ItemFn>
__device__ __forceinline__ void a_scales_of(const MxArgs &p, int n_items, const ItemFn &item, uint8_t *sf0, int stage_bytes,
                                            uint64_t *full, uint64_t *empty, int KB, int it0, int step) {
    const int lane = threadIdx.x & 31;
    const int SR = p.K / 32;
    const uint8_t *as_end = p.as + (size_t)p.M * SR;
    uint32_t st = 0, ph = 1;
    bool ok = true;
    // the array's first and last piece, which a 16-byte load would leave: a byte per lane
    const uint8_t *first = nullptr, *last = nullptr;
    uint32_t edge_byte = 0;
    if constexpr (!EVEN) {
        first = reinterpret_cast<const uint8_t *>((uintptr_t)p.as & ~(uintptr_t)15);
        last = reinterpret_cast<const uint8_t *>((uintptr_t)(as_end - 1) & ~(uintptr_t)15);
        const uint8_t *c = (lane < 16 ? first : last) + (lane & 15);
        if (c >= p.as && c < as_end) edge_byte = __ldg(c);
    }
    auto next_item = [&](int &it, Item &x) {   // the first item from `it` on that has a matrix
        for (; it < n_items; it += step) {
            x = item(it);
            if (x.mat >= 0) return;
        }
    };
    const uint4 ones = make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
    auto fetch = [&](ScaleRows<EVEN> &v, const Item &x, int k0) {
        if constexpr (EVEN) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
#pragma unroll
                for (int h = 0; h < 2; h++) v.u[q][h] = ones;   // rows past the tile: scale 1
                if (32 * q + lane < x.n) {
                    const uint8_t *s = p.as + (size_t)(x.row0 + 32 * q + lane) * SR + 8 * k0;
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (k0 + 2 * h < KB) v.u[q][h] = __ldg(reinterpret_cast<const uint4 *>(s + 16 * h));
                }
            }
        } else {
            bool edge = false;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const bool live = 32 * q + lane < x.n;
                const uint8_t *row = p.as + (size_t)(x.row0 + (live ? 32 * q + lane : 0)) * SR, *s = row + 8 * k0;
                v.off[q] = (uint32_t)((uintptr_t)s & 15);
#pragma unroll
                for (int h = 0; h < 3; h++) {
                    const uint8_t *c = s - v.off[q] + 16 * h;
                    v.u[q][h] = ones;
                    const bool want = live && c < row + SR && (h < 2 || v.off[q] != 0);
                    if (want && c >= p.as && c + 16 <= as_end) v.u[q][h] = __ldg(reinterpret_cast<const uint4 *>(c));
                    edge |= want && (c < p.as || c + 16 > as_end);
                }
            }
            if (__any_sync(0xFFFFFFFFu, edge)) {
                const uint4 head = edge_piece(edge_byte, lane < 16 ? lane : -1), tail = edge_piece(edge_byte, lane < 16 ? -1 : lane - 16);
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (32 * q + lane < x.n) {
                        const uint8_t *row = p.as + (size_t)(x.row0 + 32 * q + lane) * SR, *s = row + 8 * k0;
#pragma unroll
                        for (int h = 0; h < 3; h++) {
                            const uint8_t *c = s - v.off[q] + 16 * h;
                            if (c < row + SR && (c < p.as || c + 16 > as_end)) v.u[q][h] = c == last ? tail : head;
                        }
                    }
            }
        }
    };
    // The rows' 32 bytes as words, once the pieces are there; `left` bytes of a row remain, what lies
    // past them reads as scale 1.
    auto words = [&](uint32_t (&w)[4][8], const ScaleRows<EVEN> &v, int left) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if constexpr (EVEN) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    w[q][4 * h] = v.u[q][h].x;
                    w[q][4 * h + 1] = v.u[q][h].y;
                    w[q][4 * h + 2] = v.u[q][h].z;
                    w[q][4 * h + 3] = v.u[q][h].w;
                }
            } else {
                const uint32_t r[12] = {v.u[q][0].x, v.u[q][0].y, v.u[q][0].z, v.u[q][0].w, v.u[q][1].x, v.u[q][1].y,
                                        v.u[q][1].z, v.u[q][1].w, v.u[q][2].x, v.u[q][2].y, v.u[q][2].z, v.u[q][2].w};
                const bool one = v.off[q] & 4, two = v.off[q] & 8;
                const uint32_t sh = 8 * (v.off[q] & 3);
                uint32_t a[11], b[9];
#pragma unroll
                for (int i = 0; i < 11; i++) a[i] = one ? r[i + 1] : r[i];
#pragma unroll
                for (int i = 0; i < 9; i++) b[i] = two ? a[i + 2] : a[i];
#pragma unroll
                for (int i = 0; i < 8; i++) w[q][i] = __funnelshift_r(b[i], b[i + 1], sh);
                if (left < 32) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int n = left - 4 * i;
                        const uint32_t keep = n >= 4 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
                        w[q][i] = (w[q][i] & keep) | (0x7F7F7F7Fu & ~keep);
                    }
                }
            }
        }
    };
    ScaleRows<EVEN> nx;
    uint32_t w[4][8];
    int it = it0, k0 = 0;
    Item x = {};
    next_item(it, x);
    if (it < n_items) {
        fetch(nx, x, 0);
        words(w, nx, SR);
    }
    while (ok && it < n_items) {
        const int kn = min(MM_KS, KB - k0);
        k0 += MM_KS;
        if (k0 >= KB) {
            k0 = 0;
            it += step;
            next_item(it, x);
        }
        if (it < n_items) fetch(nx, x, k0);
#pragma unroll
        for (int e = 0; e < MM_KS; e++) {
            if (!ok || e >= kn) continue;
            ok = __all_sync(0xFFFFFFFFu, tc::mbar_wait(&empty[st], ph, p.err, 85));   // the warp gives up together
            if (!ok) continue;
            uint8_t *sf = sf0 + st * stage_bytes;
            *reinterpret_cast<uint4 *>(sf + 16 * lane) = make_uint4(w[0][2 * e], w[1][2 * e], w[2][2 * e], w[3][2 * e]);
            *reinterpret_cast<uint4 *>(sf + 512 + 16 * lane) =
                make_uint4(w[0][2 * e + 1], w[1][2 * e + 1], w[2][2 * e + 1], w[3][2 * e + 1]);
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&full[st]);
            if (++st == STAGES) {
                st = 0;
                ph ^= 1u;
            }
        }
        words(w, nx, SR - 8 * k0);
    }
}

template <int STAGES, typename ItemFn>
__device__ __forceinline__ void a_scales(const MxArgs &p, int n_items, const ItemFn &item, uint8_t *sf0, int stage_bytes,
                                         uint64_t *full, uint64_t *empty, int KB, int it0, int step) {
    if ((p.K / 32) % 16 == 0 && ((uintptr_t)p.as & 15) == 0)
        a_scales_of<STAGES, true>(p, n_items, item, sf0, stage_bytes, full, empty, KB, it0, step);
    else
        a_scales_of<STAGES, false>(p, n_items, item, sf0, stage_bytes, full, empty, KB, it0, step);
}

// 128 rows x NT columns per item, one CTA per SM. A K block is 256 codes of a row, 128 bytes: four
// MMAs of K = 64 and two TMEM copies of scale atoms per operand. Bound by HBM for few rows (16 x 8
// rows over 64 experts of 4096 x 7168: 122 us, the weights at 7.1 TB/s), by the chain of K
// blocks for one tile in a row (one token, 7168 x 7168: 9.8 to 10.4 us, 0.20 us a K block: about half of it
// waits, copies and commits, 25 ns an MMA however few its columns; fewer stages, a second accumulator
// or no proxy fence left it as it was. A K split would make a row's result depend on how many rows
// are beside it; more codes per wait and commit would not, and have not been tried), by L2 and power above.
template <int NT>
__global__ void __launch_bounds__(MM_THREADS, 1) k_mx4_mm(const __grid_constant__ CUtensorMap tmA,
                                                          const __grid_constant__ CUtensorMap tmA1,
                                                          const __grid_constant__ CUtensorMap tmW, MxArgs p) {
    using C = MmCfg<NT>;
    extern __shared__ uint8_t mm_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)mm_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::STAGES * C::STAGE);
    uint64_t *empty = full + C::STAGES, *tfull = empty + C::STAGES, *tempty = tfull + C::NACC;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tempty + C::NACC);
    uint8_t *stg_all = smem + C::STAGES * C::STAGE + C::BAR;
    __shared__ Plan plan;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; i++) {
            tc::mbar_init(&full[i], 3);     // W's thread, A's thread and the A scales' warp
            tc::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < C::NACC; i++) {
            tc::mbar_init(&tfull[i], 1);
            tc::mbar_init(&tempty[i], MM_EPI);
        }
        tc::fence_mbar_init();
        tc::prefetch_tmap(&tmA);
        tc::prefetch_tmap(&tmW);
    }
    if (warp == 1) tc::tmem_alloc(tmem_slot, 512);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dep_wait();   // everything read from here on may come from the kernel before
    const int tiles = plan_tiles<MM_THREADS>(plan, p.off, p.G, p.M, MM_M);
    const int n_items = tiles * p.NTL;
    const int KB = (p.K + 255) / 256;
    const int KA = (p.K + 127) / 128;              // scale atoms along K
    Walk walk{plan, p.off, p.mat_of, p.M, p.n_mats, p.G, p.NTL, MM_M};
    auto item = [&](int it) { return walk.at(it); };   // a thread takes one role

    if (warp == 0) {
        // ------------------------------------------------------------ W's codes and scales
        if (elect_one()) {
            bool ok = tc::tc_check((tc::smem_u32(smem) & 1023) == 0, p.err, 80);
            uint32_t n = 0, st = 0, ph = 1;
            for (int it = blockIdx.x; ok && it < n_items; it += gridDim.x) {
                const Item x = item(it);
                if (x.mat < 0) continue;
                const int arow = NT >= 128 ? x.nt * C::NA : x.nt / 2;         // W's 128-row atom
                const int atoms = min(C::NA, (p.N + 127) / 128 - arow);        // the last tile may end early
                const uint8_t *wsf = p.atoms + (size_t)x.mat * p.atom_stride + (size_t)arow * KA * 512;
                for (int kb = 0; kb < KB; kb++, n++) {
                    if (!tc::mbar_wait(&empty[st], ph, p.err, 81)) { ok = false; break; }
                    uint8_t *sb = smem + st * C::STAGE + MM_A, *sf = sb + C::B + 1024;
                    const uint32_t sfb = min(2, KA - 2 * kb) * 512;            // of this K block
                    tc::mbar_expect_tx(&full[st], C::B + atoms * sfb);
                    tc::tma_load_3d(sb, &tmW, &full[st], kb * 128, x.nt * NT, x.mat);
                    for (int a = 0; a < atoms; a++)
                        tc::bulk_load(sf + a * 1024, wsf + ((size_t)a * KA + 2 * kb) * 512, sfb, &full[st]);
                    if (++st == C::STAGES) {
                        st = 0;
                        ph ^= 1u;
                    }
                }
            }
            // no copy may still be landing when the CTA exits
            for (uint32_t i = n > C::STAGES ? n - C::STAGES : 0; i < n; i++)
                tc::mbar_wait(&full[i % C::STAGES], (i / C::STAGES) & 1u, p.err, 82);
        }
    } else if (warp == 3) {
        // ------------------------------------------------------------ A's codes
        if (elect_one()) copy_a<C::STAGES>(p, n_items, item, tmA, tmA1, smem, C::STAGE, full, empty, KB, blockIdx.x, gridDim.x);
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA
        if (elect_one()) {
            uint32_t st = 0, ph = 0, a = 0, aph = 1;   // aph: parity of an accumulator's last release
            bool ok = true;
            // descriptors of stage 0; a stage, a K step and an atom on are additions to the low words
            const uint64_t da0 = tc::desc_kmajor_sw128(tc::smem_u32(smem)), db0 = tc::desc_kmajor_sw128(tc::smem_u32(smem) + MM_A);
            const uint64_t dsf0 = tc::desc_sf_atom(tc::smem_u32(smem) + MM_A + C::B);
            for (int it = blockIdx.x; ok && it < n_items; it += gridDim.x) {
                const Item x = item(it);
                if (x.mat < 0) continue;
                if (!tc::mbar_wait(&tempty[a], aph, p.err, 83)) { ok = false; break; }
                tc::tc_fence_after();
                const uint32_t d = tmem + a * NT;
                const uint32_t shift = NT == 64 ? 2u * (x.nt & 1) : 0u;   // rows 64..127 of an atom: two columns on
                for (int kb = 0; kb < KB; kb++) {
                    if (!tc::mbar_wait(&full[st], ph, p.err, 84)) { ok = false; break; }
                    tc::fence_proxy_async_smem();   // A's scales, stored by warp 2
                    tc::tc_fence_after();
                    const uint64_t so = (uint64_t)(st * (C::STAGE >> 4));
                    const uint64_t da = da0 + so, db = db0 + so, dsf = dsf0 + so;
                    const uint32_t col = tmem + C::SF_COL + st * C::SFW;
                    // per 128 elements: A's four columns, then W's four per 128 rows
                    auto scales = [&](int j) {
                        tc::tc_cp_sf(col + j * (C::SFW / 2), dsf + j * 32);
#pragma unroll
                        for (int q = 0; q < C::NA; q++) tc::tc_cp_sf(col + j * (C::SFW / 2) + 4 + 4 * q, dsf + 64 + q * 64 + j * 32);
                    };
                    auto step = [&](int k, uint32_t acc) {
                        const uint32_t id = 2u * (k & 1), sfa = col + (k >> 1) * (C::SFW / 2);
                        tc_mma_mx4(d, da + 2 * k, db + 2 * k, idesc_mxf4(NT, id), sfa | (id << 30), (sfa + 4 + shift) | (id << 30), acc);
                    };
                    const int left = p.K - 256 * kb;
                    scales(0);
                    if (left >= 256) {
                        scales(1);
                        step(0, kb != 0);
#pragma unroll
                        for (int k = 1; k < 4; k++) step(k, 1);
                    } else {
                        if (left > 128) scales(1);
                        for (int k = 0; 64 * k < left; k++) step(k, (kb | k) != 0);
                    }
                    tc::tc_commit(&empty[st]);
                    if (++st == C::STAGES) {
                        st = 0;
                        ph ^= 1u;
                    }
                }
                if (ok) tc::tc_commit(&tfull[a]);
                if (++a == C::NACC) {
                    a = 0;
                    aph ^= 1u;
                }
            }
        }
    } else if (warp == 2) {
        a_scales<C::STAGES>(p, n_items, item, smem + MM_A + C::B, C::STAGE, full, empty, KB, blockIdx.x, gridDim.x);
    } else if (warp >= 4) {
        // ------------------------------------------------------------ epilogue
        const int q = warp & 3, half = (warp - 4) >> 2;   // TMEM lane quadrant, half of the columns
        constexpr int NC = NT / 64;                       // 32-column pieces per half
        const uint32_t lane_base = (uint32_t)(32 * q) << 16;
        uint8_t *stg = stg_all + (warp - 4) * 2048;
        uint32_t li = 0;
        bool alive = true;   // false after a wait gave up: the remaining results are NaN
        for (int it = blockIdx.x; it < n_items; it += gridDim.x) {
            const Item x = item(it);
            const int rows = min(32, x.n - 32 * q);
            uint32_t v[NC][32];
            bool ok = true;   // zeros of a group without a matrix stay zeros
            if (x.mat < 0) {
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int i = 0; i < 32; i++) v[c][i] = 0;
            } else {
                const uint32_t a = li % C::NACC, use = li / C::NACC;
                li++;
                ok = alive = alive && wait_for_sums(&tfull[a], use & 1u, p.err, 86, KB);
                __syncwarp();
                tc::tc_fence_after();
                // the whole share goes to registers first, so the accumulator is free again
#pragma unroll
                for (int c = 0; c < NC; c++) tc::tmem_ld32(tmem + lane_base + a * NT + 32u * (half * NC + c), v[c]);
                tc::tmem_ld_wait();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&tempty[a]);
            }
            if (rows > 0) store_rows<NC>(stg, v, p, x.row0 + 32 * q, rows, x.nt * NT + 32 * half * NC, ok);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == 1) tc::tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------ two CTAs on one tile
// k_mx4_mm on 256 rows x 256 columns per pair of CTAs (cta_group::2): each holds its 128 rows of A
// and its 128 rows of W, and the MMA reads both halves of W, so an SM fetches 32 KB of codes per
// K block instead of 48. 8192 x 7168 x 7168: 155 us, 5.4 PFLOP/s (one CTA 165); 16384 x 7168 x 2048:
// 113 (141). 470 cycles a K block, the MMAs' own time, at the 1.5 GHz that power leaves; the first
// blocks of an item and the last wave are the rest. W's scales of all 256 columns are in both CTAs.
// The pair's first CTA issues all MMAs. Its partner's warp 1 passes each filled stage on: it waits
// for the local copies, fences A's scales and arrives on `full` in the first CTA. MMA commits free
// the stage in both.
struct PrCfg {
    static constexpr int B = 128 * 128;
    static constexpr int SF = 1024 + 2048;
    static constexpr int STAGE = MM_A + B + SF;
    static constexpr int STAGES = 5;
    static constexpr uint32_t SFW = 24, SF_COL = 256;
    static constexpr int BYTES = 1024 + STAGES * STAGE + 256 + MM_EPI * 2048;
    static_assert(STAGE % 1024 == 0, "stage bases stay 1024-byte aligned");
    static_assert(SF_COL + STAGES * SFW <= 512, "TMEM columns");
    static_assert(BYTES + sizeof(Plan) + 64 <= 227 * 1024, "one CTA per SM");
};

__device__ __forceinline__ void mbar_arrive_cta(uint64_t *bar, uint32_t cta) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(tc::dsmem_addr(tc::smem_u32(bar), cta))
                 : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t *slot, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(slot)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t base, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(ncols) : "memory");
}
// Arrives on *bar of both CTAs once this thread's earlier tcgen05 operations have completed.
__device__ __forceinline__ void tc_commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            tc::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void tc_cp_sf_pair(uint32_t col, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(col), "l"(desc) : "memory");
}
__device__ __forceinline__ void tc_mma_mx4_pair(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa,
                                                uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
}
// idesc_mxf4 with M = 256 (the pair's rows).
__host__ __device__ constexpr uint32_t idesc_mxf4_pair(uint32_t n, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((256u >> 4) << 24) | (sf_id << 29);
}

__global__ void __launch_bounds__(MM_THREADS, 1) k_mx4_mm_pair(const __grid_constant__ CUtensorMap tmA,
                                                               const __grid_constant__ CUtensorMap tmA1,
                                                               const __grid_constant__ CUtensorMap tmW, MxArgs p) {
    using C = PrCfg;
    extern __shared__ uint8_t pr_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)pr_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::STAGES * C::STAGE);
    uint64_t *empty = full + C::STAGES, *tfull = empty + C::STAGES, *tempty = tfull + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tempty + 1);
    uint8_t *stg_all = smem + C::STAGES * C::STAGE + 256;
    __shared__ Plan plan;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_ctarank();

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; i++) {
            tc::mbar_init(&full[i], rank == 0 ? 4 : 3);   // the first CTA's: the partner's stage too
            tc::mbar_init(&empty[i], 1);
        }
        tc::mbar_init(tfull, 1);
        tc::mbar_init(tempty, 2 * MM_EPI);
        tc::fence_mbar_init();
        tc::prefetch_tmap(&tmA);
        tc::prefetch_tmap(&tmW);
    }
    if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();   // both CTAs' barriers and TMEM are there
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dep_wait();
    const int tiles = plan_tiles<MM_THREADS>(plan, p.off, p.G, p.M, 2 * MM_M);
    const int n_items = tiles * p.NTL;
    const int KB = (p.K + 255) / 256, KA = (p.K + 127) / 128;
    const int it0 = blockIdx.x >> 1, step = gridDim.x >> 1;
    Walk walk{plan, p.off, p.mat_of, p.M, p.n_mats, p.G, p.NTL, 2 * MM_M};
    auto pair_item = [&](int it) { return walk.at(it); };   // a thread takes one role
    auto item = [&](int it) {   // this CTA's rows of the pair's item
        Item x = pair_item(it);
        x.row0 += rank * MM_M;
        x.n = min(max(x.n - (int)rank * MM_M, 0), MM_M);
        return x;
    };

    if (warp == 0) {
        // ------------------------------------------------------------ W's codes and scales
        if (elect_one()) {
            bool ok = tc::tc_check((tc::smem_u32(smem) & 1023) == 0, p.err, 110);
            uint32_t n = 0, st = 0, ph = 1;
            for (int it = it0; ok && it < n_items; it += step) {
                const Item x = pair_item(it);
                if (x.mat < 0) continue;
                const int atoms = min(2, (p.N + 127) / 128 - 2 * x.nt);
                const uint8_t *wsf = p.atoms + (size_t)x.mat * p.atom_stride + (size_t)(2 * x.nt) * KA * 512;
                for (int kb = 0; kb < KB; kb++, n++) {
                    if (!tc::mbar_wait(&empty[st], ph, p.err, 111)) { ok = false; break; }
                    uint8_t *sb = smem + st * C::STAGE + MM_A, *sf = sb + C::B + 1024;
                    const uint32_t sfb = min(2, KA - 2 * kb) * 512;
                    tc::mbar_expect_tx(&full[st], C::B + atoms * sfb);
                    tc::tma_load_3d(sb, &tmW, &full[st], kb * 128, x.nt * 256 + rank * 128, x.mat);
                    for (int a = 0; a < atoms; a++)
                        tc::bulk_load(sf + a * 1024, wsf + ((size_t)a * KA + 2 * kb) * 512, sfb, &full[st]);
                    if (++st == C::STAGES) {
                        st = 0;
                        ph ^= 1u;
                    }
                }
            }
            for (uint32_t i = n > C::STAGES ? n - C::STAGES : 0; i < n; i++)
                tc::mbar_wait(&full[i % C::STAGES], (i / C::STAGES) & 1u, p.err, 112);
        }
    } else if (warp == 3) {
        // ------------------------------------------------------------ A's codes
        if (elect_one()) copy_a<C::STAGES>(p, n_items, item, tmA, tmA1, smem, C::STAGE, full, empty, KB, it0, step);
    } else if (warp == 1 && rank != 0) {
        // ------------------------------------------------------------ filled stages to the first CTA
        if (elect_one()) {
            uint32_t st = 0, ph = 0;
            bool ok = true;
            for (int it = it0; ok && it < n_items; it += step) {
                if (pair_item(it).mat < 0) continue;
                for (int kb = 0; kb < KB; kb++) {
                    if (!tc::mbar_wait(&full[st], ph, p.err, 113)) { ok = false; break; }
                    tc::fence_proxy_async_smem();
                    mbar_arrive_cta(&full[st], 0);
                    if (++st == C::STAGES) {
                        st = 0;
                        ph ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA
        if (elect_one()) {
            uint32_t st = 0, ph = 0, tph = 1;
            bool ok = true;
            const uint64_t da0 = tc::desc_kmajor_sw128(tc::smem_u32(smem)), db0 = tc::desc_kmajor_sw128(tc::smem_u32(smem) + MM_A);
            const uint64_t dsf0 = tc::desc_sf_atom(tc::smem_u32(smem) + MM_A + C::B);
            for (int it = it0; ok && it < n_items; it += step) {
                if (pair_item(it).mat < 0) continue;
                if (!tc::mbar_wait(tempty, tph, p.err, 114)) { ok = false; break; }
                tph ^= 1u;
                tc::tc_fence_after();
                for (int kb = 0; kb < KB; kb++) {
                    if (!tc::mbar_wait(&full[st], ph, p.err, 115)) { ok = false; break; }
                    tc::fence_proxy_async_smem();
                    tc::tc_fence_after();
                    const uint64_t so = (uint64_t)(st * (C::STAGE >> 4));
                    const uint64_t da = da0 + so, db = db0 + so, dsf = dsf0 + so;
                    const uint32_t col = tmem + C::SF_COL + st * C::SFW;
                    auto scales = [&](int j) {
                        tc_cp_sf_pair(col + j * 12, dsf + j * 32);
                        tc_cp_sf_pair(col + j * 12 + 4, dsf + 64 + j * 32);
                        tc_cp_sf_pair(col + j * 12 + 8, dsf + 128 + j * 32);
                    };
                    auto mma = [&](int k, uint32_t acc) {
                        const uint32_t id = 2u * (k & 1), sfa = col + (k >> 1) * 12;
                        tc_mma_mx4_pair(tmem, da + 2 * k, db + 2 * k, idesc_mxf4_pair(256, id), sfa | (id << 30), (sfa + 4) | (id << 30), acc);
                    };
                    const int left = p.K - 256 * kb;
                    scales(0);
                    if (left >= 256) {
                        scales(1);
                        mma(0, kb != 0);
#pragma unroll
                        for (int k = 1; k < 4; k++) mma(k, 1);
                    } else {
                        if (left > 128) scales(1);
                        for (int k = 0; 64 * k < left; k++) mma(k, (kb | k) != 0);
                    }
                    tc_commit_pair(&empty[st]);
                    if (++st == C::STAGES) {
                        st = 0;
                        ph ^= 1u;
                    }
                }
                if (ok) tc_commit_pair(tfull);
            }
        }
    } else if (warp == 2) {
        a_scales<C::STAGES>(p, n_items, item, smem + MM_A + C::B, C::STAGE, full, empty, KB, it0, step);
    } else if (warp >= 4) {
        // ------------------------------------------------------------ epilogue
        const int q = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lane_base = (uint32_t)(32 * q) << 16;
        uint8_t *stg = stg_all + (warp - 4) * 2048;
        uint32_t tph = 0;
        bool alive = true;
        for (int it = it0; it < n_items; it += step) {
            const Item x = item(it);
            const int rows = min(32, x.n - 32 * q);
            uint32_t v[4][32];
            bool ok = true;
            if (x.mat < 0) {
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int i = 0; i < 32; i++) v[c][i] = 0;
            } else {
                ok = alive = alive && wait_for_sums(tfull, tph, p.err, 117, KB);
                tph ^= 1u;
                __syncwarp();
                tc::tc_fence_after();
#pragma unroll
                for (int c = 0; c < 4; c++) tc::tmem_ld32(tmem + lane_base + 32u * (half * 4 + c), v[c]);
                tc::tmem_ld_wait();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cta(tempty, 0);
            }
            if (rows > 0) store_rows<4>(stg, v, p, x.row0 + 32 * q, rows, x.nt * 256 + 32 * half * 4, ok);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();   // the partner's MMAs, commits and arrivals reach this CTA's memory until here
    tc::tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ------------------------------------------------------------------ gradient of the activations
// Three rings: packed W tiles (copied), widened W tiles (written by the widening warps) and dY
// tiles (copied); the last two share their slots' numbers, and an MMA commit frees both. With
// one ring for all three a slot was held through copy, widening and MMA, 3900 cycles for 1024
// of MMAs: three slots' worth of them set the pace.
constexpr int MB_KB = 64;                        // W rows per K block
constexpr int MB_EPI = 8;
constexpr int MB_WIDE0 = 3;                      // warps: dY, MMA, W, widening, epilogue
// 128 rows x NT columns (W's in) per CTA and item; columns narrower than 256 make more items where
// there are too few for every SM. PAIR: two CTAs with 128 rows each on the same 2 * NT columns
// (cta_group::2); each widens NT of them and the MMA reads both CTAs' halves. Shared memory's
// bandwidth bounds these kernels: a K block of 128 x 256 takes one CTA 121 KB through it (copies
// in, packed tile out, widened tile in, both operands out), 950 cycles at 128 bytes a cycle, for
// 512 cycles of MMAs; a pair's CTA 73 KB, 580 cycles; 128 x 128 72 KB, 560 cycles, to which the
// widening's instructions add (without its arithmetic 64 x 7168 x 2048 takes 29 us of 34, with
// half its stores 30, without dY's copies 31). ACCS = 2: a pair takes 512 rows in two
// accumulators, so a widened tile serves both; what that saves is mostly power, which bounds the
// clock under large products. It leaves no TMEM for the next item's accumulators.
template <int NT, bool PAIR, int ACCS>
struct MbCfg {
    static constexpr int TN = PAIR ? 2 * NT : NT;            // columns of an item
    static constexpr int A = ACCS * 128 * 128;               // dY: 128 rows x 64 bf16 per accumulator
    static constexpr int B = NT * MB_KB * 2;                 // widened W: NT/64 blocks of 64 columns x 64 rows
    static constexpr int WB = NT / 2;                        // bytes of a packed W row
    static constexpr int W = MB_KB * WB;
    static constexpr int R = (W + NT / 128 * 512 + 1023) / 1024 * 1024;   // and its scale atoms
    static constexpr int RING = NT == 256 ? 3 : 4;           // slots of dY and widened W
    static constexpr int RAW = ACCS == 2 ? 4 : NT == 256 ? 6 : 12;        // slots of packed W
    static constexpr int NBUF = ACCS == 2 ? 1 : 2;           // items whose accumulators TMEM holds
    static constexpr int ROWS = (PAIR ? 256 : 128) * ACCS;   // rows of an item
    // Groups of widening warps. Both rings hold a multiple of TURNS, so a slot is always the same
    // group's, which then awaits each of the slot's phases in turn: a group that skipped a phase
    // could take the one before it, of the same parity, for the one it needs.
    static constexpr int TURNS = RING;
    // Warps that widen one K block. Where a single CTA widens 128 columns of it two do, with more in
    // flight each: four warps' issue slots are what few rows wait for (64 x 7168 x 2048 34.1 us,
    // 35.0 with four; 39.5 with one). Pairs and 256 columns need four (1200 x 7168 x 2048 39.1, 41.9
    // with two; 128 x 7168 x 37888 71 and 93).
    static constexpr int GROUP = !PAIR && NT == 128 ? 2 : 4;
    static constexpr int EPI0 = MB_WIDE0 + TURNS * GROUP, THREADS = 32 * (EPI0 + MB_EPI);
    static constexpr int BYTES = 1024 + RING * (A + B) + RAW * R + 512;
    static_assert(B % 1024 == 0, "slots stay 1024-byte aligned");
    static_assert(NBUF * ACCS * TN <= 512, "TMEM columns");
    static_assert(RING == TURNS && RAW % TURNS == 0, "a slot belongs to one group");
    static_assert((2 * RING + 2 * RAW + 4) * 8 + 4 <= 512, "barriers");
    static_assert(BYTES + sizeof(Plan) + 64 <= 227 * 1024, "one CTA per SM");
};

// kind::f16: bf16 A (K-major) and B (N-major: transpose bit 16), fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_bf16_tb(uint32_t m, uint32_t n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void tc_mma_bf16(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
}
// N-major operand, 128-byte swizzle: rows of 64 N-elements, 8 of the contracted index per 1024
// bytes (SBO), blocks of 64 N-elements MB_KB * 128 bytes apart (LBO).
__device__ __forceinline__ uint64_t desc_nmajor_sw128(uint32_t addr) { return tc::smem_desc(addr, MB_KB * 128, 1024, 2); }

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Eight E2M1 codes to bf16: a code's exponent and mantissa bits at bits 8..6 of a bf16 are its
// value times 2^-126, subnormals included, so f1 = 2^(byte-1) under both halves gives the scaled
// value in one exact product. Codes j and j + 4 share word j, as they lie 16 bits apart. A multiply
// puts a code's magnitude and sign in place at once (the bits between are masked), shifts and masks
// do the same on the other pipe: two words each (64 x 7168 x 2048: 34.1 us; all by shifts 35.4, all by
// multiplies 34.7).
__device__ __forceinline__ void e2m1x8_widen(uint32_t w, uint32_t f1, uint32_t (&o)[4]) {
    constexpr uint32_t mag = 0x01C001C0u, sign = 0x80008000u;
    o[0] = mul_bf16x2(((w & 0x000F000Fu) * 0x1040u) & (mag | sign), f1);
    o[1] = mul_bf16x2(((w & 0x00F000F0u) * 0x0104u) & (mag | sign), f1);
    o[2] = mul_bf16x2(((w >> 2) & mag) | ((w << 4) & sign), f1);
    o[3] = mul_bf16x2(((w >> 6) & mag) | (w & sign), f1);
}

// 16 rows x 32 fp32 columns of TMEM: lane l gets, of rows l/4 (v[4i], v[4i+1]) and l/4 + 8
// (v[4i+2], v[4i+3]), columns 8i + 2(l%4) and the next, for i = 0..3.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}

// Eight neighbouring columns of one row, q[2i] and q[2i + 1] holding columns i and i + 4 (i = 0..3).
__device__ __forceinline__ void put8(const MxArgs &p, int64_t row, int col, const uint32_t (&q)[8]) {
    if (p.y_bf16) {
        uint16_t *d = reinterpret_cast<uint16_t *>(p.y) + row * p.ldy + col;
        const uint32_t o[4] = {f32x2_to_bf16x2(__uint_as_float(q[0]), __uint_as_float(q[2])),
                               f32x2_to_bf16x2(__uint_as_float(q[4]), __uint_as_float(q[6])),
                               f32x2_to_bf16x2(__uint_as_float(q[1]), __uint_as_float(q[3])),
                               f32x2_to_bf16x2(__uint_as_float(q[5]), __uint_as_float(q[7]))};
        if (p.vec) *reinterpret_cast<uint4 *>(d) = make_uint4(o[0], o[1], o[2], o[3]);
        else
#pragma unroll
            for (int i = 0; i < 4; i++) {
                d[2 * i] = (uint16_t)o[i];
                d[2 * i + 1] = (uint16_t)(o[i] >> 16);
            }
    } else {
        uint32_t *d = reinterpret_cast<uint32_t *>(p.y) + row * p.ldy + col;
        if (p.vec) {
            reinterpret_cast<uint4 *>(d)[0] = make_uint4(q[0], q[2], q[4], q[6]);
            reinterpret_cast<uint4 *>(d)[1] = make_uint4(q[1], q[3], q[5], q[7]);
        } else
#pragma unroll
            for (int i = 0; i < 4; i++) {
                d[i] = q[2 * i];
                d[4 + i] = q[2 * i + 1];
            }
    }
}

// Dense 32768 x 7168 x 2048 (rows, contracted, columns): 627 us, 1.53 PFLOP/s, 692 after some
// seconds at the power limit. 32768 rows in 48 groups: 780-880 us at 1.37 GHz, 600 cycles a K block
// against 512 of MMAs, 15% of the tiles' rows empty. 2400 rows in 48 groups of 1432 x 992: 26 us, 28 with
// a cold L2.
template <int NT, bool PAIR, int ACCS>
__global__ void __launch_bounds__(MbCfg<NT, PAIR, ACCS>::THREADS, 1) k_mx4_bwd(const __grid_constant__ CUtensorMap tmD,
                                                           const __grid_constant__ CUtensorMap tmD1,
                                                           const __grid_constant__ CUtensorMap tmW, MxArgs p) {
    using C = MbCfg<NT, PAIR, ACCS>;
    extern __shared__ uint8_t mb_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)mb_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *s_a = smem, *s_b = s_a + C::RING * C::A, *s_r = s_b + C::RING * C::B;
    uint64_t *full = reinterpret_cast<uint64_t *>(s_r + C::RAW * C::R), *empty = full + C::RING;
    uint64_t *rfull = empty + C::RING, *rempty = rfull + C::RAW;
    uint64_t *tfull = rempty + C::RAW, *tempty = tfull + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tempty + 2);
    __shared__ Plan plan;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? tc::cluster_ctarank() : 0u;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::RING; i++) {
            // dY's copy, the widening warps and, in a pair's first CTA, the partner's slot
            tc::mbar_init(&full[i], 1 + C::GROUP + (PAIR && rank == 0 ? 1 : 0));
            tc::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < C::RAW; i++) {
            tc::mbar_init(&rfull[i], 1);
            tc::mbar_init(&rempty[i], C::GROUP);
        }
        for (int i = 0; i < C::NBUF; i++) {
            tc::mbar_init(&tfull[i], 1);
            tc::mbar_init(&tempty[i], (PAIR ? 2 : 1) * MB_EPI);
        }
        tc::fence_mbar_init();
        tc::prefetch_tmap(&tmD);
        tc::prefetch_tmap(&tmW);
    }
    if (warp == 1) {
        if constexpr (PAIR) tmem_alloc_pair(tmem_slot, 512);
        else tc::tmem_alloc(tmem_slot, 512);
    }
    tc::tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) tc::cluster_sync();   // both CTAs' barriers and TMEM are there
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dep_wait();
    const int tiles = plan_tiles<C::THREADS>(plan, p.off, p.G, p.M, C::ROWS);
    const int n_items = tiles * p.NTL;
    const int KB = (p.N + MB_KB - 1) / MB_KB;      // contracted: W's rows
    const int KA = (p.K + 127) / 128;
    const int it0 = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;
    Walk walk{plan, p.off, p.mat_of, p.M, p.n_mats, p.G, p.NTL, C::ROWS};
    auto item = [&](int it) { return walk.at(it); };   // a thread takes one role
    // This CTA's rows of an item in accumulator j: 128 j and, in pairs, 256 j + 128 rank on.
    auto first_row = [&](int j) { return (PAIR ? 256 : 128) * j + (int)rank * 128; };
    auto row_count = [&](const Item &x, int j) { return min(max(x.n - first_row(j), 0), 128); };

    if (warp == 0) {
        // ------------------------------------------------------------ dY copies
        if (elect_one()) {
            bool ok = tc::tc_check((tc::smem_u32(smem) & 1023) == 0, p.err, 90);
            uint32_t st = 0, ph = 1, n = 0;
            for (int it = it0; ok && it < n_items; it += step) {
                const Item x = item(it);
                if (x.mat < 0) continue;
                int boxes[ACCS], all = 0;
#pragma unroll
                for (int j = 0; j < ACCS; j++) {
                    boxes[j] = (row_count(x, j) + 31) / 32;
                    all += boxes[j];
                }
                for (int kb = 0; kb < KB; kb++, n++) {
                    if (!tc::mbar_wait(&empty[st], ph, p.err, 91)) { ok = false; break; }
                    uint8_t *sa = s_a + st * C::A;
                    tc::mbar_expect_tx(&full[st], all * 32 * 128);
#pragma unroll
                    for (int j = 0; j < ACCS; j++) {
                        const int row = x.row0 + first_row(j);
                        if (boxes[j] == 4) tc::tma_load_3d(sa + j * (128 * 128), &tmD, &full[st], kb * MB_KB, row, 0);
                        else
                            for (int b = 0; b < boxes[j]; b++)
                                tc::tma_load_3d(sa + j * (128 * 128) + b * (32 * 128), &tmD1, &full[st], kb * MB_KB, row + b * 32, 0);
                    }
                    if (++st == C::RING) {
                        st = 0;
                        ph ^= 1u;
                    }
                }
            }
            // no copy may still be landing when the CTA exits
            for (uint32_t i = n > C::RING ? n - C::RING : 0; i < n; i++)
                tc::mbar_wait(&full[i % C::RING], (i / C::RING) & 1u, p.err, 92);
        }
    } else if (warp == 2) {
        // ------------------------------------------------------------ W copies
        if (elect_one()) {
            bool ok = true;
            uint32_t st = 0, ph = 1, n = 0;
            for (int it = it0; ok && it < n_items; it += step) {
                const Item x = item(it);
                if (x.mat < 0) continue;
                const int col = x.nt * C::TN + (int)rank * NT;                   // the CTA's first column
                const uint32_t sfb = min(NT / 128, max(KA - col / 128, 0)) * 512;   // none past W's columns
                const uint8_t *wsf = p.atoms + (size_t)x.mat * p.atom_stride + (size_t)(col / 128) * 512;
                for (int kb = 0; kb < KB; kb++, n++) {
                    if (!tc::mbar_wait(&rempty[st], ph, p.err, 93)) { ok = false; break; }
                    uint8_t *sw = s_r + st * C::R;
                    tc::mbar_expect_tx(&rfull[st], C::W + sfb);
                    tc::tma_load_3d(sw, &tmW, &rfull[st], col / 2, kb * MB_KB, x.mat);
                    if (sfb) tc::bulk_load(sw + C::W, wsf + (size_t)(kb / 2) * KA * 512, sfb, &rfull[st]);
                    if (++st == C::RAW) {
                        st = 0;
                        ph ^= 1u;
                    }
                }
            }
            for (uint32_t i = n > C::RAW ? n - C::RAW : 0; i < n; i++)
                tc::mbar_wait(&rfull[i % C::RAW], (i / C::RAW) & 1u, p.err, 94);
        }
    } else if (PAIR && warp == 1 && rank != 0) {
        // ------------------------------------------------------------ filled slots to the first CTA
        if (elect_one()) {
            uint32_t st = 0, ph = 0;
            bool ok = true;
            for (int it = it0; ok && it < n_items; it += step) {
                if (item(it).mat < 0) continue;
                for (int kb = 0; kb < KB; kb++) {
                    if (!tc::mbar_wait(&full[st], ph, p.err, 101)) { ok = false; break; }
                    mbar_arrive_cta(&full[st], 0);
                    if (++st == C::RING) {
                        st = 0;
                        ph ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA
        if (elect_one()) {
            uint32_t st = 0, ph = 0, a = 0, aph = 1;
            bool ok = true;
            constexpr uint32_t idesc = idesc_bf16_tb(PAIR ? 256 : 128, C::TN);
            const uint64_t da0 = tc::desc_kmajor_sw128(tc::smem_u32(s_a)), db0 = desc_nmajor_sw128(tc::smem_u32(s_b));
            for (int it = it0; ok && it < n_items; it += step) {
                const Item x = item(it);
                if (x.mat < 0) continue;
                if (!tc::mbar_wait(&tempty[a], aph, p.err, 95)) { ok = false; break; }
                tc::tc_fence_after();
                const uint32_t d = tmem + a * ACCS * C::TN;
                const bool two = ACCS == 2 && x.n > C::ROWS / 2;
                for (int kb = 0; kb < KB; kb++) {
                    if (!tc::mbar_wait(&full[st], ph, p.err, 96)) { ok = false; break; }
                    tc::tc_fence_after();
                    const uint64_t da = da0 + st * (C::A >> 4), db = db0 + st * (C::B >> 4);
#pragma unroll
                    for (int k = 0; k < 4; k++) tc_mma_bf16<PAIR>(d, da + 2 * k, db + 128 * k, idesc, (kb | k) != 0);
                    if (two) {
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            tc_mma_bf16<PAIR>(d + C::TN, da + (128 * 128 >> 4) + 2 * k, db + 128 * k, idesc, (kb | k) != 0);
                    }
                    if constexpr (PAIR) tc_commit_pair(&empty[st]);
                    else tc::tc_commit(&empty[st]);
                    if (++st == C::RING) {
                        st = 0;
                        ph ^= 1u;
                    }
                }
                if (ok) {
                    if constexpr (PAIR) tc_commit_pair(&tfull[a]);
                    else tc::tc_commit(&tfull[a]);
                }
                if (++a == C::NBUF) {
                    a = 0;
                    aph ^= 1u;
                }
            }
        }
    } else if (warp >= MB_WIDE0 && warp < C::EPI0) {
        // ------------------------------------------------------------ widening
        const int w4 = (warp - MB_WIDE0) % C::GROUP;
        const uint32_t turn = (warp - MB_WIDE0) / C::GROUP;
        // A group steps straight from one of its K blocks to the next (counting through the others' cost
        // 250 cycles a block, a third of a group's time): its slot of the widened ring is number
        // `turn`, and its packed slots come round by TURNS.
        uint32_t n = 0, ph = 1, rt = turn, rph = 0;   // K blocks before the item; awaited parities, packed slot
        uint8_t *const sb = s_b + turn * C::B;
        bool ok = true;
        for (int it = it0; ok && it < n_items; it += step) {
            if (item(it).mat < 0) continue;
            for (int kb = (int)((turn + C::TURNS - n % C::TURNS) % C::TURNS); kb < KB; kb += C::TURNS) {
                ok = __all_sync(0xFFFFFFFFu, tc::mbar_wait(&rfull[rt], rph, p.err, 98));
                if (!ok) break;
                // a lane widens 32 codes of RJ W rows in each 128 columns: groups g and g + 4
                // (eight lanes touch eight rows: the swizzle spreads them over the banks)
                constexpr int GH = NT / 128, RJ = 8 / C::GROUP;
                const uint8_t *sw = s_r + rt * C::R;
                const int r0 = 8 * RJ * w4 + (lane & 7), g = lane >> 3;
                uint4 c[RJ][GH];
                uint32_t s[RJ][GH];
#pragma unroll
                for (int j = 0; j < RJ; j++)
#pragma unroll
                    for (int i = 0; i < GH; i++) {
                        const int r = r0 + 8 * j;
                        const int at = NT == 256 ? (g + 4 * i) ^ (r & 7) : g ^ ((r >> 1) & 3);   // 128- and 64-byte swizzle
                        c[j][i] = *reinterpret_cast<const uint4 *>(sw + r * C::WB + 16 * at);
                        s[j][i] = sw[C::W + i * 512 + sf_byte((kb & 1) * 64 + r, g)];
                    }
                ok = __all_sync(0xFFFFFFFFu, tc::mbar_wait(&empty[turn], ph, p.err, 99));
                if (!ok) break;
#pragma unroll
                for (int j = 0; j < RJ; j++)
#pragma unroll
                    for (int i = 0; i < GH; i++) {
                        const int r = r0 + 8 * j;
                        const uint32_t e = min(s[j][i], 128u) + 126u;    // 2^(min(byte, 128) - 1)
                        const uint32_t f1 = e << 7 | e << 23;
                        const uint32_t cw[4] = {c[j][i].x, c[j][i].y, c[j][i].z, c[j][i].w};
                        uint32_t o[4][4];
#pragma unroll
                        for (int k = 0; k < 4; k++) e2m1x8_widen(cw[k], f1, o[k]);
                        if (s[j][i] > 128) {                             // the rest of a scale above 2^1
                            const uint32_t h = s[j][i] - 1u, f2 = h << 7 | h << 23;   // 2^(byte - 128)
#pragma unroll
                            for (int k = 0; k < 4; k++)
#pragma unroll
                                for (int q = 0; q < 4; q++) o[k][q] = mul_bf16x2(o[k][q], f2);
                        }
                        // Column order within the 32: piece q holds codes q and q + 4 of each of
                        // the four words, so that a lane of the epilogue's 16x256b loads, which
                        // gets columns 2l and 2l + 1 of every piece, gets word l: eight neighbours.
                        uint8_t *row = sb + ((g + 4 * i) >> 1) * (MB_KB * 128) + r * 128;
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            *reinterpret_cast<uint4 *>(row + 16 * (((g & 1) * 4 + q) ^ (r & 7))) =
                                make_uint4(o[0][q], o[1][q], o[2][q], o[3][q]);
                    }
                // The packed slot is given back only here, where the stores above have used every load from
                // it and the proxy fence stands behind them. Given back right after the loads were issued, a
                // load that waited behind the epilogue's element stores came after the next copy into the slot.
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(&full[turn]);
                    tc::mbar_arrive(&rempty[rt]);
                }
                ph ^= 1u;
                rt += C::TURNS;
                if (rt >= C::RAW) {
                    rt -= C::RAW;
                    rph ^= 1u;
                }
            }
            n += KB;
        }
    } else if (warp >= C::EPI0) {
        // ------------------------------------------------------------ epilogue
        // A store covers 8 rows x 64 bytes (bf16); with a row per lane it was 32 rows x 16, and
        // the accumulators stayed taken for 12000 cycles an item instead of 8600.
        const int q = warp & 3, half = (warp - C::EPI0) >> 2;   // TMEM lane quadrant, half of the columns
        const uint32_t lanes = (uint32_t)(32 * q) << 16;
        uint32_t a = 0, aph = 0;
        bool alive = true;
        for (int it = it0; it < n_items; it += step) {
            const Item x = item(it);
            const int first = half * (C::TN / 2);                              // the warp's columns of the tile
            const int c0 = x.nt * C::TN, last = min(first + C::TN / 2, p.K - c0);   // a multiple of 32
            const uint32_t taddr = tmem + lanes + a * ACCS * C::TN;
            const bool real = x.mat >= 0;
            if (real) {
                alive = alive && wait_for_sums(&tfull[a], aph, p.err, 100, KB);
                __syncwarp();
                tc::tc_fence_after();
            }
#pragma unroll
            for (int j = 0; j < ACCS; j++) {
                const int n = row_count(x, j) - 32 * q;                        // rows of the warp's 32
                const int64_t row = x.row0 + first_row(j) + 32 * q;
                if (n <= 0) continue;
#pragma unroll 2
                for (int c = first; c < last; c += 32) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {                      // rows 16h ..
                        uint32_t v[16];
                        if (real) {
                            tmem_ld_16x32(taddr + ((uint32_t)(16 * h) << 16) + j * C::TN + c, v);
                            tc::tmem_ld_wait();
                        }
                        if (!real || !alive)
#pragma unroll
                            for (int i = 0; i < 16; i++) v[i] = real ? 0x7FC00000u : 0u;
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int r = 16 * h + 8 * e + (lane >> 2);
                            const uint32_t u[8] = {v[2 * e], v[2 * e + 1], v[4 + 2 * e], v[5 + 2 * e],
                                                   v[8 + 2 * e], v[9 + 2 * e], v[12 + 2 * e], v[13 + 2 * e]};
                            if (r < n) put8(p, row + r, c0 + c + 8 * (lane & 3), u);
                        }
                    }
                }
            }
            if (real) {
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) mbar_arrive_cta(&tempty[a], 0);
                    else tc::mbar_arrive(&tempty[a]);
                }
                if (++a == C::NBUF) {
                    a = 0;
                    aph ^= 1u;
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) tc::cluster_sync();   // the partner's MMAs, commits and arrivals end before this CTA's memory does
    tc::tc_fence_after();
    if (warp == 1) {
        if constexpr (PAIR) tmem_dealloc_pair(tmem, 512);
        else tc::tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------ host side
bool al16(const void *p) { return ((uintptr_t)p & 15) == 0; }
int known(int dt) { return dt == K3C_F32 || dt == K3C_BF16; }

int check_mat(const char *what, const k3c_mxfp4_mat *W, int M, const int *off, int n_groups) {
    if (!W || !W->codes || !W->atoms || W->rows < 1 || W->rows > MX_DIM || W->in < 32 || W->in > MX_DIM || W->in % 32 ||
        W->n_mats < 1)
        return set_error(K3C_EINVAL, "%s: matrix rows=%d in=%d (a multiple of 32) n_mats=%d", what, W ? W->rows : 0,
                         W ? W->in : 0, W ? W->n_mats : 0);
    if (!al16(W->codes) || !al16(W->atoms) || W->code_stride % 16 || W->atom_stride % 16)
        return set_error(K3C_EINVAL, "%s: codes, atoms and their strides must be 16-byte aligned", what);
    const size_t cb = (size_t)W->rows * (W->in / 2), ab = k3c_mxfp4_atom_bytes(W->rows, W->in);
    if (W->n_mats > 1 && (W->code_stride < cb || W->atom_stride < ab))
        return set_error(K3C_EINVAL, "%s: strides %zu, %zu below a matrix's %zu, %zu bytes", what, W->code_stride,
                         W->atom_stride, cb, ab);
    if (M < 0 || M > MX_DIM || n_groups < 1 || n_groups > MX_GMAX || (!off && n_groups != 1))
        return set_error(K3C_EINVAL, "%s: M=%d n_groups=%d (1..%d; 1 without offsets)", what, M, n_groups, MX_GMAX);
    if (off && !W->mat_of && n_groups > W->n_mats)
        return set_error(K3C_EINVAL, "%s: %d groups, %d matrices", what, n_groups, W->n_mats);
    return K3C_OK;
}

// Boxes of box_bytes (128 or 64: the swizzle) x box_rows of the packed matrices.
int map_weights(CUtensorMap *m, const k3c_mxfp4_mat *W, int box_bytes, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return set_error(K3C_ECUDA, "mxfp4: cuTensorMapEncodeTiled unavailable");
    const size_t stride = W->n_mats > 1 ? W->code_stride : (size_t)W->rows * (W->in / 2);
    cuuint64_t dims[3] = {(cuuint64_t)W->in / 2, (cuuint64_t)W->rows, (cuuint64_t)W->n_mats};
    cuuint64_t strides[2] = {(cuuint64_t)W->in / 2, (cuuint64_t)stride};
    cuuint32_t box[3] = {(cuuint32_t)box_bytes, (cuuint32_t)box_rows, 1}, es[3] = {1, 1, 1};
    CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(W->codes), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(K3C_ECUDA, "mxfp4: tensor map encode failed (%d)", (int)r);
    return K3C_OK;
}

int err_slot(int **err) {
    static int *err_of[64] = {};
    int *&e = err_of[cur_dev()];
    if (!e) K3C_TRY_CUDA(cudaGetSymbolAddress((void **)&e, g_mx_err));
    *err = e;
    return K3C_OK;
}

int check_waits(const char *what, int *err, cudaStream_t s) {
    static const int sync_check = getenv("K3C_SYNC_CHECK") ? 1 : 0;
    if (!sync_check) return K3C_OK;
    int code = 0;
    K3C_TRY_CUDA(cudaStreamSynchronize(s));
    K3C_TRY_CUDA(cudaMemcpy(&code, err, sizeof(int), cudaMemcpyDeviceToHost));
    if (code) {
        const int zero = 0;
        cudaMemcpy(err, &zero, sizeof(int), cudaMemcpyHostToDevice);
        return set_error(K3C_ETIMEOUT, "%s: device check code %d", what, code);
    }
    return K3C_OK;
}

// Items are numbered in 32 bits; 128 x 64 is the smallest tile.
int check_items(const char *what, int M, int n_groups, int cols) {
    const int64_t items = most_tiles(M, n_groups, 128) * ((cols + 63) / 64);
    return items <= MX_DIM ? K3C_OK : set_error(K3C_EINVAL, "%s: %lld tiles exceed 32 bits", what, (long long)items);
}

// A kernel's tile and what it costs: a launch takes about fixed + waves * max(K blocks * block + item,
// store) ns, a wave being one item on every SM (or pair of SMs) and `store` its epilogue. Fitted to
// measured launches of M = 1 to 16000 rows, dense and in 4 to 48 groups (e.g. 8 K blocks of
// k3c_mxfp4_mm, 4096 x 7168: pair 33.5 us, 256 columns 33.7, 128 38.8, 64 62; 1 x 7168: 9.5, 7.8, 6.4,
// 6.7; one K block, 8000 x 4096: 29.5, 26.1, 37.6, 65).
struct TileCost {
    int rows, cols, ctas, block, item, store, fixed;
};
// The cheapest of n kernels for M rows in n_groups groups (grouped: their sizes are on the device;
// each is taken to waste half a tile) and `cols` columns, kb K blocks. Ties go to the first. All M rows are
// taken to belong to groups: where an expert-parallel rank holds 3637 of 32768, in 48 groups, a
// product with 4096 x 7168 matrices takes 159 us on pairs and 135 on 128 x 256 tiles, which the rows alone
// would take; the gradient of 7168 x 2048 takes 247 us on pairs and 275 on those tiles.
int cheapest(const TileCost *t, int n, int M, int n_groups, bool grouped, int cols, int kb) {
    int best = 0;
    double least = 0;
    for (int i = 0; i < n; i++) {
        double tiles = (M + t[i].rows - 1) / t[i].rows;
        if (grouped) {
            const double half = (double)M / t[i].rows + 0.5 * n_groups, few = n_groups < M ? n_groups : M;
            tiles = half > few ? half : few;
        }
        const double items = tiles * ((cols + t[i].cols - 1) / t[i].cols), at_once = sm_count() / t[i].ctas;
        const double waves = items <= at_once ? 1 : (double)(int64_t)((items + at_once - 1) / at_once);
        const double loop = (double)kb * t[i].block + t[i].item;
        const double ns = t[i].fixed + waves * (loop > t[i].store ? loop : t[i].store);
        if (!i || ns < least) {
            best = i;
            least = ns;
        }
    }
    return best;
}

const TileCost MM_KINDS[] = {{256, 256, 2, 380, 700, 3400, 5400},
                             {128, 256, 1, 410, 1000, 3150, 3950},
                             {128, 128, 1, 270, 500, 2400, 3650},
                             {128, 64, 1, 240, 400, 2200, 3400}};
int mm_kind(int M, int n_groups, bool grouped, int rows, int in) {
    return cheapest(MM_KINDS, 4, M, n_groups, grouped, rows, (in + 255) / 256);
}
// (112 K blocks, 2048 columns: 64 rows take the pair 39 us, 256 columns 56, 128 columns 34; 2000 rows
// 44, 63, 72; two accumulators 75 there, but 261 to 282 and one 304 at 12000 rows. 4 K blocks, 2000 x 2048:
// the pair 8.8, 256 and 128 columns 8.3)
const TileCost BWD_KINDS[] = {{512, 256, 2, 555, 4050, 0, 5150},
                              {256, 256, 2, 325, 1100, 0, 6200},
                              {128, 256, 1, 505, 550, 0, 5100},
                              {128, 128, 1, 295, 300, 1700, 3850}};
int bwd_kind(int M, int n_groups, bool grouped, int rows, int in) {
    return cheapest(BWD_KINDS, 4, M, n_groups, grouped, in, (rows + MB_KB - 1) / MB_KB);
}

template <int NT>
int launch_mm(const CUtensorMap &ma, const CUtensorMap &ma1, const CUtensorMap &mw, MxArgs p, cudaStream_t s) {
    static bool attr_of[64] = {};
    bool &attr = attr_of[cur_dev()];
    if (!attr) {
        K3C_TRY_CUDA(cudaFuncSetAttribute(k_mx4_mm<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, MmCfg<NT>::BYTES));
        attr = true;
    }
    p.NTL = (p.N + NT - 1) / NT;
    const int64_t items = most_tiles(p.M, p.G, MM_M) * p.NTL;
    const int grid = (int)(items < sm_count() ? items : sm_count());
    K3C_TRY_CUDA(launch_pdl(k_mx4_mm<NT>, dim3(grid), dim3(MM_THREADS), MmCfg<NT>::BYTES, s, ma, ma1, mw, p));
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

// A kernel of CTA pairs, as a programmatic dependent.
template <typename... KArgs, typename... Args>
cudaError_t launch_pairs(void (*kernel)(KArgs...), int grid, int block, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 2;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

int launch_mm_pair(const CUtensorMap &ma, const CUtensorMap &ma1, const CUtensorMap &mw, MxArgs p, cudaStream_t s) {
    static bool attr_of[64] = {};
    bool &attr = attr_of[cur_dev()];
    if (!attr) {
        K3C_TRY_CUDA(cudaFuncSetAttribute(k_mx4_mm_pair, cudaFuncAttributeMaxDynamicSharedMemorySize, PrCfg::BYTES));
        attr = true;
    }
    p.NTL = (p.N + 255) / 256;
    const int64_t items = most_tiles(p.M, p.G, 2 * MM_M) * p.NTL;
    const int grid = 2 * (int)(items < sm_count() / 2 ? items : sm_count() / 2);
    K3C_TRY_CUDA(launch_pairs(k_mx4_mm_pair, grid, MM_THREADS, PrCfg::BYTES, s, ma, ma1, mw, p));
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

template <int NT, bool PAIR, int ACCS>
int launch_bwd(MxArgs p, const k3c_mxfp4_mat *W, const void *dy, int64_t lddy, cudaStream_t s) {
    using C = MbCfg<NT, PAIR, ACCS>;
    CUtensorMap md, md1, mw;
    K3C_TRY(make_map3(&md, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dy, p.N, p.M, 1, lddy * 2, (uint64_t)lddy * 2 * p.M, 64, 128));
    K3C_TRY(make_map3(&md1, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dy, p.N, p.M, 1, lddy * 2, (uint64_t)lddy * 2 * p.M, 64, 32));
    K3C_TRY(map_weights(&mw, W, C::WB, MB_KB));
    static bool attr_of[64] = {};
    bool &attr = attr_of[cur_dev()];
    if (!attr) {
        K3C_TRY_CUDA(cudaFuncSetAttribute(k_mx4_bwd<NT, PAIR, ACCS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES));
        attr = true;
    }
    p.NTL = (p.K + C::TN - 1) / C::TN;
    const int64_t items = most_tiles(p.M, p.G, C::ROWS) * p.NTL;
    if constexpr (PAIR) {
        const int grid = 2 * (int)(items < sm_count() / 2 ? items : sm_count() / 2);
        K3C_TRY_CUDA(launch_pairs(k_mx4_bwd<NT, PAIR, ACCS>, grid, C::THREADS, C::BYTES, s, md, md1, mw, p));
    } else {
        const int grid = (int)(items < sm_count() ? items : sm_count());
        K3C_TRY_CUDA(launch_pdl(k_mx4_bwd<NT, PAIR, ACCS>, dim3(grid), dim3(C::THREADS), C::BYTES, s, md, md1, mw, p));
    }
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

}  // namespace
}  // namespace k3c

using namespace k3c;

extern "C" int k3c_mxfp4_quant(uint8_t *packed, uint8_t *scales, const void *x, int x_dtype, int64_t ldx, int rows, int in,
                               k3c_stream_t stream) {
    clear_error();
    if (rows < 0 || in < 2 || in > MX_DIM || in % 2 || ldx < in || !known(x_dtype))
        return set_error(K3C_EINVAL, "mxfp4_quant: rows=%d in=%d (even) ldx=%lld dtype=%d", rows, in, (long long)ldx, x_dtype);
    if (!rows) return K3C_OK;
    if (!packed || !scales || !x) return set_error(K3C_EINVAL, "mxfp4_quant: NULL array");
    cudaStream_t s = (cudaStream_t)stream;
    const int esz = x_dtype == K3C_F32 ? 4 : 2;
    const bool wide = al16(x) && ((uintptr_t)packed & 3) == 0 && in % 32 == 0 && (ldx * esz) % 16 == 0;
    const size_t work = wide ? (size_t)rows * (in / 8) / QUANT_U : (size_t)rows * ((in + 31) / 32);
    const unsigned grid = (unsigned)(work / 256 + 1 < 148 * 64 ? work / 256 + 1 : 148 * 64);
    const bool dense = ldx == in || rows == 1;
    if (x_dtype == K3C_F32) {
        const float *xf = (const float *)x;
        if (wide && dense) k_mx4_quant<float, true><<<grid, 256, 0, s>>>(packed, scales, xf, ldx, rows, in);
        else if (wide) k_mx4_quant<float, false><<<grid, 256, 0, s>>>(packed, scales, xf, ldx, rows, in);
        else k_mx4_quant_any<<<grid, 256, 0, s>>>(packed, scales, xf, ldx, rows, in);
    } else {
        const uint16_t *xb = (const uint16_t *)x;
        if (wide && dense) k_mx4_quant<uint16_t, true><<<grid, 256, 0, s>>>(packed, scales, xb, ldx, rows, in);
        else if (wide) k_mx4_quant<uint16_t, false><<<grid, 256, 0, s>>>(packed, scales, xb, ldx, rows, in);
        else k_mx4_quant_any<<<grid, 256, 0, s>>>(packed, scales, xb, ldx, rows, in);
    }
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

extern "C" size_t k3c_mxfp4_atom_bytes(int rows, int in) {
    if (rows < 1 || in < 1) return 0;
    return (size_t)((rows + 127) / 128) * ((in + 127) / 128) * 512;
}

extern "C" int k3c_mxfp4_pack(uint8_t *codes, uint8_t *atoms, const uint8_t *packed, const uint8_t *scales, int n_mats,
                              int rows, int in, k3c_stream_t stream) {
    clear_error();
    if (n_mats < 1 || rows < 1 || rows > MX_DIM || in < 32 || in > MX_DIM || in % 32)
        return set_error(K3C_EINVAL, "mxfp4_pack: n_mats=%d rows=%d in=%d (a multiple of 32)", n_mats, rows, in);
    if (!codes || !atoms || !packed || !scales) return set_error(K3C_EINVAL, "mxfp4_pack: NULL array");
    if (!al16(codes) || !al16(packed)) return set_error(K3C_EINVAL, "mxfp4_pack: codes and packed must be 16-byte aligned");
    const size_t n = (size_t)n_mats * k3c_mxfp4_atom_bytes(rows, in);   // one byte per group
    const unsigned grid = (unsigned)((n + 255) / 256 < 148 * 64 ? (n + 255) / 256 : 148 * 64);
    k_mx4_pack<<<grid, 256, 0, (cudaStream_t)stream>>>(codes, atoms, packed, scales, n_mats, rows, in);
    K3C_CHECK_LAUNCH();
    return K3C_OK;
}

extern "C" int k3c_mxfp4_mm_tile(int M, int n_groups, int grouped, int rows, int in, int gradient) {
    clear_error();
    if (M < 1 || M > MX_DIM || n_groups < 1 || n_groups > MX_GMAX || rows < 1 || rows > MX_DIM || in < 32 || in > MX_DIM)
        return set_error(K3C_EINVAL, "mxfp4_mm_tile: M=%d n_groups=%d rows=%d in=%d", M, n_groups, rows, in);
    const TileCost &t = gradient ? BWD_KINDS[bwd_kind(M, n_groups, grouped != 0, rows, in)]
                                 : MM_KINDS[mm_kind(M, n_groups, grouped != 0, rows, in)];
    return t.rows << 16 | t.cols;
}

extern "C" int k3c_mxfp4_mm(void *y, int y_dtype, int64_t ldy, const uint8_t *a, const uint8_t *a_scales, int M,
                            const k3c_mxfp4_mat *W, const int *off, int n_groups, k3c_stream_t stream) {
    clear_error();
    K3C_TRY(check_mat("mxfp4_mm", W, M, off, n_groups));
    if (!known(y_dtype) || ldy < W->rows)
        return set_error(K3C_EINVAL, "mxfp4_mm: y_dtype=%d ldy=%lld rows=%d", y_dtype, (long long)ldy, W->rows);
    if (!M) return K3C_OK;
    if (!y || !a || !a_scales) return set_error(K3C_EINVAL, "mxfp4_mm: NULL array");
    if (!al16(a)) return set_error(K3C_EINVAL, "mxfp4_mm: a must be 16-byte aligned");
    K3C_TRY(check_items("mxfp4_mm", M, n_groups, W->rows));
    cudaStream_t s = (cudaStream_t)stream;
    MxArgs p = {};
    K3C_TRY(err_slot(&p.err));
    p.y = y;
    p.ldy = ldy;
    p.y_bf16 = y_dtype == K3C_BF16;
    p.vec = al16(y) && (ldy * (p.y_bf16 ? 2 : 4)) % 16 == 0;
    p.M = M;
    p.N = W->rows;
    p.K = W->in;
    p.G = n_groups;
    p.off = off;
    p.mat_of = W->mat_of;
    p.n_mats = W->n_mats;
    p.as = a_scales;
    p.atoms = W->atoms;
    p.atom_stride = W->atom_stride;
    const int kind = mm_kind(M, n_groups, off != nullptr, p.N, p.K);
    CUtensorMap ma, ma1, mw;
    K3C_TRY(make_map3(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, a, p.K / 2, M, 1, p.K / 2, (uint64_t)(p.K / 2) * M, 128, MM_M));
    K3C_TRY(make_map3(&ma1, CU_TENSOR_MAP_DATA_TYPE_UINT8, a, p.K / 2, M, 1, p.K / 2, (uint64_t)(p.K / 2) * M, 128, MM_ABOX));
    K3C_TRY(map_weights(&mw, W, 128, kind == 0 ? 128 : MM_KINDS[kind].cols));   // a pair's CTAs copy half the columns each
    if (kind == 0) K3C_TRY(launch_mm_pair(ma, ma1, mw, p, s));
    else if (kind == 1) K3C_TRY(launch_mm<256>(ma, ma1, mw, p, s));
    else if (kind == 2) K3C_TRY(launch_mm<128>(ma, ma1, mw, p, s));
    else K3C_TRY(launch_mm<64>(ma, ma1, mw, p, s));
    return check_waits("mxfp4_mm", p.err, s);
}

extern "C" int k3c_mxfp4_mm_bwd(void *da, int da_dtype, int64_t ldda, const void *dy, int64_t lddy, int M,
                                const k3c_mxfp4_mat *W, const int *off, int n_groups, k3c_stream_t stream) {
    clear_error();
    K3C_TRY(check_mat("mxfp4_mm_bwd", W, M, off, n_groups));
    if (!known(da_dtype) || ldda < W->in || lddy < W->rows || lddy % 8)
        return set_error(K3C_EINVAL, "mxfp4_mm_bwd: da_dtype=%d ldda=%lld in=%d lddy=%lld (a multiple of 8) rows=%d", da_dtype,
                         (long long)ldda, W->in, (long long)lddy, W->rows);
    if (!M) return K3C_OK;
    if (!da || !dy) return set_error(K3C_EINVAL, "mxfp4_mm_bwd: NULL array");
    if (!al16(dy)) return set_error(K3C_EINVAL, "mxfp4_mm_bwd: dy must be 16-byte aligned");
    K3C_TRY(check_items("mxfp4_mm_bwd", M, n_groups, W->in));
    cudaStream_t s = (cudaStream_t)stream;
    MxArgs p = {};
    K3C_TRY(err_slot(&p.err));
    p.y = da;
    p.ldy = ldda;
    p.y_bf16 = da_dtype == K3C_BF16;
    p.vec = al16(da) && (ldda * (p.y_bf16 ? 2 : 4)) % 16 == 0;
    p.M = M;
    p.N = W->rows;
    p.K = W->in;
    p.G = n_groups;
    p.off = off;
    p.mat_of = W->mat_of;
    p.n_mats = W->n_mats;
    p.atoms = W->atoms;
    p.atom_stride = W->atom_stride;
    const int kind = bwd_kind(M, n_groups, off != nullptr, p.N, p.K);
    if (kind == 0) K3C_TRY((launch_bwd<128, true, 2>(p, W, dy, lddy, s)));
    else if (kind == 1) K3C_TRY((launch_bwd<128, true, 1>(p, W, dy, lddy, s)));
    else if (kind == 2) K3C_TRY((launch_bwd<256, false, 1>(p, W, dy, lddy, s)));
    else K3C_TRY((launch_bwd<128, false, 1>(p, W, dy, lddy, s)));
    return check_waits("mxfp4_mm_bwd", p.err, s);
}
