// The product of rows and a weight in 8 bits, and what brings tensors to that form.
//
//   y[m][n] = sum over blocks b of 128 columns:  xs[m][b] ws[n / 128][b] sum over k in b of xc[m][k] wc[n][k]   [+ bias[n]]
//
// Codes are e4m3; their products and the sums of a block are exact or nearly so in fp32, and each block's sum is multiplied by its two scales
// and added up in fp32.  y is rounded once.
//
// What bounds it.  Few tokens: the weight's bytes (8x4096x32000 24.7 us, 81 % of a copy's rate; 1x4096x4096 7.7 us, of which the weight takes 2.6: a
// launch, the first copies and the join of a cluster).  Many tokens: products and sums in turn (8192x4096x16384 among pauses 505 us, 2.17 PFLOP/s, 66 % of
// twice the measured bf16 rate, and 421 without the sums; in passes one behind another, whose clocks fall, 595, 1.85 PFLOP/s, 56 %): a block of 256 x 256 takes a pair 512 clocks of products, and its sums 650 of eight warps, of
// which 400 are their additions.  Between them a wave or two of tiles: 512x4096x4096 15.7 us, 1024x4096x4096 21.6, 4096x4096x4096 69.5.
#include <algorithm>
#include "kernels.h"
#include "e4m3.cuh"
#include "launch.cuh"
#include "ring.h"
#include "tma.cuh"

namespace adder {
namespace {

// ------------------------------------------------------------------------------------------ to 8 bits

struct QuantArgs {
    const void* x;
    uint8_t* values;
    float* scales;
    long long rows, x_stride, values_stride;
    int d;
};

constexpr int QR_BLOCKS = 4;      // blocks of 128 columns that a warp has in flight where rows are no vectors

// Four elements of a row from column c on: consecutive ones, or (unaligned rows) every 32nd.
template <class T, bool VECTORS> __device__ __forceinline__ void quant_load(const T* row, int c, int d, float (&f)[4]) {
    if constexpr (VECTORS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = 0.f;
        if (c < d) {
            if constexpr (sizeof(T) == 4) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(row + c));
                f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
            } else {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(row + c));
                const float2 a = unpack_pair<T>(v.x), b = unpack_pair<T>(v.y);
                f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = c + 32 * j < d ? to_float(row[c + 32 * j]) : 0.f;
    }
}
template <bool VECTORS> __device__ __forceinline__ void quant_store(uint8_t* row, int c, int d, const float (&f)[4], float inverse) {
    if constexpr (VECTORS) {
        if (c < d) *reinterpret_cast<uint32_t*>(row + c) = e4m3_word(f[0], f[1], f[2], f[3], inverse);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + 32 * j < d) row[c + 32 * j] = e4m3_code(f[j], inverse);
    }
}
__device__ __forceinline__ float largest_of(const float (&f)[4]) {
    return max_nan(max_nan(fabsf(f[0]), fabsf(f[1])), max_nan(fabsf(f[2]), fabsf(f[3])));
}

// Largest magnitude of a vector, NaN if one is.
template <class T> __device__ __forceinline__ float largest_of(const uint4& q) {
    constexpr uint32_t MAGNITUDE = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
    return word_max<T>(max_word<T>(max_word<T>(q.x & MAGNITUDE, q.y & MAGNITUDE), max_word<T>(q.z & MAGNITUDE, q.w & MAGNITUDE)));
}

// Rows of 16-byte vectors: a warp takes 32 x QR_VECTORS of a row, a block of 128 columns lies with 128 / VE neighbouring lanes (8192x4096 bf16 19.4 us, 79 % of
// a copy's rate; four elements a lane, as the rows below, 28.8).  Rows that are no vectors: 8192x4001 42 us.
constexpr int QR_VECTORS = 4;
template <class T> __global__ void __launch_bounds__(256) quantize_vectors_kernel(const QuantArgs a) {
    constexpr int VE = Vec16<T>::N, LANES = E4M3_BLOCK / VE;
    const int lane = threadIdx.x & 31, nvec = a.d / VE, blocks = (a.d + E4M3_BLOCK - 1) / E4M3_BLOCK, turns = (nvec + 32 * QR_VECTORS - 1) / (32 * QR_VECTORS);
    const long long task = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    if (task >= a.rows * turns) return;
    const long long row = task / turns;
    const int v0 = (int)(task % turns) * 32 * QR_VECTORS + lane;
    const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.x_stride);
    uint8_t* out = a.values + row * a.values_stride;
    uint4 q[QR_VECTORS];
#pragma unroll
    for (int i = 0; i < QR_VECTORS; ++i) q[i] = v0 + 32 * i < nvec ? __ldg(x + v0 + 32 * i) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < QR_VECTORS; ++i) {
        const int v = v0 + 32 * i;
        float largest = largest_of<T>(q[i]), f[VE];
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, off));
        const E4m3Scale s = e4m3_scale(largest);
        Vec16<T>::unpack(q[i], f);
        if (v < nvec) {
            if constexpr (VE == 8) *reinterpret_cast<uint2*>(out + v * 8) = make_uint2(e4m3_word(f[0], f[1], f[2], f[3], s.inverse), e4m3_word(f[4], f[5], f[6], f[7], s.inverse));
            else *reinterpret_cast<uint32_t*>(out + v * 4) = e4m3_word(f[0], f[1], f[2], f[3], s.inverse);
            if (v % LANES == 0) a.scales[row * blocks + v / LANES] = s.scale;
        }
    }
}

// Other rows: a warp takes QR_BLOCKS blocks of one, 32 neighbouring elements at a time.
template <class T> __global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs a) {
    const int lane = threadIdx.x & 31, blocks = (a.d + E4M3_BLOCK - 1) / E4M3_BLOCK, turns = (blocks + QR_BLOCKS - 1) / QR_BLOCKS;
    const long long task = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    if (task >= a.rows * turns) return;
    const long long row = task / turns;
    const int b0 = (int)(task % turns) * QR_BLOCKS;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    uint8_t* out = a.values + row * a.values_stride;
    float f[QR_BLOCKS][4];
#pragma unroll
    for (int i = 0; i < QR_BLOCKS; ++i) quant_load<T, false>(x, (b0 + i) * E4M3_BLOCK + lane, a.d, f[i]);
#pragma unroll
    for (int i = 0; i < QR_BLOCKS; ++i) {
        float largest = largest_of(f[i]);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, off));
        const E4m3Scale s = e4m3_scale(largest);
        quant_store<false>(out, (b0 + i) * E4M3_BLOCK + lane, a.d, f[i], s.inverse);
        if (lane == 0 && b0 + i < blocks) a.scales[row * blocks + b0 + i] = s.scale;
    }
}

// A CTA takes a block of 128 x 128: 16 rows a warp.
template <class T, bool VECTORS> __global__ void __launch_bounds__(256) quantize_weight_kernel(const QuantArgs a) {
    __shared__ float part[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, blocks = (a.d + E4M3_BLOCK - 1) / E4M3_BLOCK;
    const long long row0 = (long long)(blockIdx.x / blocks) * E4M3_BLOCK;
    const int b = blockIdx.x % blocks, from = b * E4M3_BLOCK + (VECTORS ? 4 * lane : lane);
    float f[16][4], largest = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const long long row = row0 + warp + 8 * i;
        const bool in = row < a.rows;
        quant_load<T, VECTORS>(static_cast<const T*>(a.x) + (in ? row : row0) * a.x_stride, in ? from : a.d, a.d, f[i]);
        largest = max_nan(largest, largest_of(f[i]));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, off));
    if (lane == 0) part[warp] = largest;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max_nan(largest, part[i]);
    const E4m3Scale s = e4m3_scale(largest);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const long long row = row0 + warp + 8 * i;
        if (row < a.rows) quant_store<VECTORS>(a.values + row * a.values_stride, from, a.d, f[i], s.inverse);
    }
    if (threadIdx.x == 0) a.scales[blockIdx.x] = s.scale;
}

// ------------------------------------------------------------------------------------------ the product

struct L8Args {
    const float* xs;
    const float* ws;
    const void* bias;      // may be null
    void* y;
    int tokens, outer, blocks;      // blocks of 128 columns
    int m_tiles, n_tiles;
    bool whole_fours;               // scales may be read four at a time
    bool whole_rows;                // rows of y are whole 16-byte vectors
};
// Scales of blocks b to b + 3, as far as there are that many.
__device__ __forceinline__ void l8_four(const float* p, int b, int blocks, bool whole, float (&f)[4]) {
    if (whole) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p + b));
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = p[min(b + i, blocks - 1)];
    }
}

constexpr uint32_t L8_SLAB = 128 * 128;      // bytes of 128 rows of a block

// Shared-memory operand descriptor of rows of 128 bytes in the 128-byte swizzle: eight rows are 1024 bytes.  A step of 32 bytes along the
// row adds 2 to the low word.
__device__ __forceinline__ uint32_t l8_desc(uint32_t addr) { return ((addr >> 4) & 0x3fff) | (1u << 16); }
constexpr uint32_t L8_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
// fp32 sums of e4m3 x e4m3, both operands along k
__host__ __device__ constexpr uint32_t l8_instruction(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }

__device__ __forceinline__ bool l8_elect() {
    uint32_t e;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(e));
    return e != 0;
}
// A block of both operands: four steps of 32 along k, the first of which overwrites the accumulator.
template <int CTAS> __device__ __forceinline__ void l8_multiply(uint32_t d, uint32_t a, uint32_t b, uint32_t instruction) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (CTAS == 2)
            asm volatile("{ .reg .pred p; .reg .b64 da, db; setp.ne.b32 p, %5, 0; mov.b64 da, {%1, %3}; mov.b64 db, {%2, %3};"
                         " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %4, p; }"
                         ::"r"(d), "r"(a + 2 * k), "r"(b + 2 * k), "r"(L8_DESC_HI), "r"(instruction), "r"(k) : "memory");
        else
            asm volatile("{ .reg .pred p; .reg .b64 da, db; setp.ne.b32 p, %5, 0; mov.b64 da, {%1, %3}; mov.b64 db, {%2, %3};"
                         " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %4, p; }"
                         ::"r"(d), "r"(a + 2 * k), "r"(b + 2 * k), "r"(L8_DESC_HI), "r"(instruction), "r"(k) : "memory");
    }
}
// Arrives at `bar` (of both CTAs of a pair) when all products issued so far are done.
template <int CTAS> __device__ __forceinline__ void l8_commit(uint64_t* bar) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t l8_map_shared(const void* p, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
// Loads `box` rows of a block from row y on; bar is an address in the cluster's shared memory.
template <int CTAS> __device__ __forceinline__ void l8_load(uint32_t to, const CUtensorMap* map, uint32_t bar, int x, int y) {
    if constexpr (CTAS == 2)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(to), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(to), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
// mbar_wait by a whole warp, which goes on or gives up as one.
__device__ __forceinline__ bool l8_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }
// Until the products have let go of every stage that a copy thread has used: their word goes to the shared memory of both CTAs of a pair, whenever
// it is ready, so a CTA that left without it would leave a barrier on which an arrival is under way.
template <int STAGES> __device__ __forceinline__ bool l8_released(uint64_t (&empty)[STAGES], int stage, int turn) {
    return ring_drain<STAGES>(stage, turn, [&](int i, uint32_t parity) { return mbar_wait(&empty[i], parity); });
}
__device__ __forceinline__ void l8_prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void l8_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void l8_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void l8_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void l8_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 16 columns of a warp's 32 rows, a row a lane.  The values are there after l8_wait_loads.
__device__ __forceinline__ void l8_read(uint32_t (&r)[16], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr));
}
__device__ __forceinline__ void l8_read(uint32_t (&r)[32], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
                 "%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(addr));
}
// Keeps the uses of r behind the wait.
template <int N> __device__ __forceinline__ void l8_hold(uint32_t (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ uint64_t l8_pair(uint32_t lo, uint32_t hi) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "r"(lo), "r"(hi));
    return p;
}

// ---- many tokens: a pair of CTAs computes 256 tokens x 256 outputs

// Each CTA of a pair loads 128 tokens and 128 weight rows of a block; the leader issues products of 256 x 256 x 32 over both CTAs' shared memory,
// and each has the sums of its 128 tokens in 256 columns of its tensor memory, twice: while one block's sums are being made, eight warps read
// those of the block before, multiply them by its scales and add them up in registers (a row and 128 columns a thread, so that both scales are
// one number a thread).
constexpr int L8P_STAGES = 5, L8P_THREADS = 384, L8P_STAGING = 4096;      // staging: bytes of a part of a warp's rows, two of them
constexpr uint32_t L8P_SMEM = L8P_STAGES * 2 * L8_SLAB + 16 * L8P_STAGING + 1024;

template <class T> __global__ void __launch_bounds__(L8P_THREADS, 1)
linear8_pair_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap y_map, const L8Args a,
                    int* error_flag) {
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[L8P_STAGES], empty[L8P_STAGES], made[2], taken[2];
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;      // clusters are pairs of neighbours
    const uint32_t smem0 = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t* const staging = raw + (smem0 - smem_u32(raw)) + L8P_STAGES * 2 * L8_SLAB;

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < L8P_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&made[b], 1); mbar_init(&taken[b], 16); }
        mbar_fence_init();
    }
    if (wid == 9) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    l8_before_sync();
    __syncthreads();
    l8_cluster_sync();
    l8_after_sync();
    const uint32_t tmem = tmem_base;
    const int pairs = gridDim.x >> 1, tiles = a.m_tiles * a.n_tiles;
    // tiles go in groups of 8 rows of tiles, so that those computed at a time share both operands in L2
    const auto place = [&](int tile, int& m0, int& n0) {
        const int group = tile / (8 * a.n_tiles), first = group * 8, rows = min(8, a.m_tiles - first), in = tile - group * 8 * a.n_tiles;
        m0 = (first + in % rows) * 256;
        n0 = in / rows * 256;
    };
    bool ok = true;
    // registers: 384 threads begin with 168 each, 64512 in all; the eight warps of the sums take 240, the other four keep 24
    if (wid >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
        if (wid == 8) {      // ---- copies
            if (l8_elect()) {
                l8_prefetch_map(&x_map);
                l8_prefetch_map(&w_map);
                int stage = 0, turn = 0;
                for (int tile = blockIdx.x >> 1; tile < tiles && ok; tile += pairs) {
                    int m0, n0;
                    place(tile, m0, n0);
                    for (int b = 0; b < a.blocks; ++b) {
                        if (!mbar_wait(&empty[stage], (turn & 1) ^ 1)) { ok = false; break; }
                        const uint32_t bar = l8_map_shared(&full[stage], 0), to = smem0 + stage * 2 * L8_SLAB;
                        if (rank == 0) mbar_arrive_expect_tx(&full[stage], 4 * L8_SLAB);
                        l8_load<2>(to, &x_map, bar, b * E4M3_BLOCK, m0 + (int)rank * 128);
                        l8_load<2>(to + L8_SLAB, &w_map, bar, b * E4M3_BLOCK, n0 + (int)rank * 128);
                        if (++stage == L8P_STAGES) { stage = 0; ++turn; }
                    }
                }
                if (!ok) {      // no copy is left in flight
                    gave_up = 1;
                    for (int i = 0; i < L8P_STAGES && rank == 0; ++i) {
                        const int t = i < stage ? turn : turn - 1;
                        if (t >= 0) mbar_wait(&full[i], t & 1);
                    }
                }
                if (!l8_released(empty, stage, turn)) gave_up = 1;
            }
            __syncwarp();
        } else if (wid == 9) {      // ---- products
            // one thread: its products of a block follow the word that a buffer is free by a wait alone (by the whole warp, which asked for
            // the copies last, it took 500 clocks, and the product 8192x4096x16384 525 us)
            if (rank == 0 && l8_elect()) {
                int stage = 0, turn = 0, it = 0;
                for (int tile = blockIdx.x >> 1; tile < tiles && ok; tile += pairs)
                    for (int b = 0; b < a.blocks; ++b, ++it) {
                        if (!mbar_wait(&full[stage], turn & 1) || !mbar_wait(&taken[it & 1], ((it >> 1) & 1) ^ 1)) { ok = false; break; }
                        l8_after_sync();
                        const uint32_t at = smem0 + stage * 2 * L8_SLAB;
                        l8_multiply<2>(tmem + (it & 1) * 256, l8_desc(at), l8_desc(at + L8_SLAB), l8_instruction(256, 256));
                        l8_commit<2>(&made[it & 1]);
                        l8_commit<2>(&empty[stage]);
                        if (++stage == L8P_STAGES) { stage = 0; ++turn; }
                    }
                if (!ok) {      // no product is left in flight
                    gave_up = 1;
                    if (it > 0) mbar_wait(&made[(it - 1) & 1], ((it - 1) >> 1) & 1);
                }
            }
            __syncwarp();
        }
    } else {      // ---- sums
        asm volatile("setmaxnreg.inc.sync.aligned.u32 240;");
        const int quarter = wid & 3, half = wid >> 2;
        const uint32_t from = tmem + ((uint32_t)quarter << 21) + half * 128;
        const uint32_t taken_at = l8_map_shared(taken, 0);
        int it = 0, turn = 0;
        for (int tile = blockIdx.x >> 1; tile < tiles && ok; tile += pairs) {
            int m0, n0;
            place(tile, m0, n0);
            m0 += (int)rank * 128 + quarter * 32;
            n0 += half * 128;
            const bool in = m0 + lane < a.tokens && n0 < a.outer;
            const float* xs = a.xs + (long long)(in ? m0 + lane : 0) * a.blocks;
            const float* ws = a.ws + (long long)(in ? n0 / E4M3_BLOCK : 0) * a.blocks;
            uint64_t acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0;
            // Scales of four blocks at a time, the next four on their way: a warp's rows lie in 32 lines, of which hardly any L1 is left to keep one
            float s[4], x4[4], w4[4];
            const auto fetch = [&](int b) {
                l8_four(xs, b, a.blocks, a.whole_fours, x4);
                l8_four(ws, b, a.blocks, a.whole_fours, w4);
            };
            fetch(0);
            // 32 columns at a time, the next ones on their way while some are added: without that all warps wait for their loads, and then
            // for one another's additions
            uint32_t r[2][32];
            const auto arrived = [&](int part) {
                l8_wait_loads();
                l8_hold(r[part & 1]);
            };
            if (!l8_wait(&made[it & 1], (it >> 1) & 1)) ok = false;
            else {
                l8_after_sync();
                l8_read(r[0], from + (it & 1) * 256);
            }
            for (int b = 0; b < a.blocks && ok; ++b, ++it) {
                if ((b & 3) == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[i] = x4[i] * w4[i];
                    if (b + 4 < a.blocks) fetch(b + 4);
                }
                const uint64_t s2 = pack2(s[0], s[0]);
                s[0] = s[1]; s[1] = s[2]; s[2] = s[3];
                const uint32_t at = from + (it & 1) * 256;
                const auto add = [&](int part) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[16 * part + i] = fma2(l8_pair(r[part & 1][2 * i], r[part & 1][2 * i + 1]), s2, acc[16 * part + i]);
                };
#pragma unroll
                for (int part = 0; part < 3; ++part) {
                    arrived(part);
                    l8_read(r[(part + 1) & 1], at + 32 * (part + 1));
                    add(part);
                }
                arrived(3);
                l8_before_sync();
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(taken_at + 8 * (it & 1)) : "memory");
                if (b + 1 < a.blocks) {
                    if (!l8_wait(&made[(it + 1) & 1], ((it + 1) >> 1) & 1)) ok = false;
                    l8_after_sync();
                    l8_read(r[0], from + ((it + 1) & 1) * 256);
                }
                add(3);
            }
            if (!ok) {
                if (lane == 0) gave_up = 1;
                break;
            }
            // Through shared memory, 128 bytes of each row at a time, in the swizzle of the copy that stores them while the next tile's sums begin (by the
            // warps' own stores a tile took 3500 clocks, a tenth of its time).  Rows of y that are no whole vectors are stored by the warps,
            // neighbouring lanes a row's elements.
            constexpr int C = 128 / sizeof(T), V = 16 / sizeof(T);      // columns of a part, of a vector
            const int rows = min(32, a.tokens - m0);
#pragma unroll
            for (int p = 0; p < 128 / C; ++p) {
                const int c0 = n0 + p * C;
                if (c0 >= a.outer || rows <= 0) break;
                // parts take turns from tile to tile, whatever each had of them: what was committed before the last one has been read
                uint8_t* const mine = staging + (2 * wid + turn) * L8P_STAGING;
                turn ^= 1;
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                __syncwarp();
#pragma unroll
                for (int v = 0; v < C / V; ++v) {
                    float f[V];
#pragma unroll
                    for (int j = 0; j < V; j += 2) unpack2(acc[(p * C + v * V + j) / 2], f[j], f[j + 1]);
                    if (a.bias != nullptr) {
#pragma unroll
                        for (int j = 0; j < V; ++j) f[j] += c0 + v * V + j < a.outer ? to_float(static_cast<const T*>(a.bias)[c0 + v * V + j]) : 0.f;
                    }
                    *reinterpret_cast<uint4*>(mine + lane * 128 + ((v ^ (lane & 7)) * 16)) = Vec16<T>::pack(f);
                }
                if (a.whole_rows) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&y_map), "r"(smem_u32(mine)), "r"(c0), "r"(m0) : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {
                    __syncwarp();
                    T* out = static_cast<T*>(a.y) + (long long)m0 * a.outer + c0;
                    for (int r0 = 0; r0 < rows; r0 += 8) {
                        T held[8][C / 32];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int k = 0; k < C / 32; ++k) {
                                const int row = r0 + i, c = lane + 32 * k;
                                held[i][k] = *reinterpret_cast<const T*>(mine + row * 128 + (((c / V) ^ (row & 7)) * 16) + c % V * sizeof(T));
                            }
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int k = 0; k < C / 32; ++k)
                                if (r0 + i < rows && c0 + lane + 32 * k < a.outer) out[(long long)(r0 + i) * a.outer + lane + 32 * k] = held[i][k];
                    }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    l8_before_sync();
    __syncthreads();
    l8_cluster_sync();      // no CTA leaves while the other's products read its shared memory, or before their word has come to its own
    if (threadIdx.x == 0 && gave_up) *error_flag = 1;
    if (wid == 9) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// ---- fewer tokens: a tile of 128 outputs x N tokens a CTA, the columns' blocks shared out over a cluster

// Up to 32 tokens the weight's rows are the rows of the products, so that few tokens fill the tensor core; its bytes are what counts.  Four warps
// add up the blocks' sums in registers, an output and all tokens a thread, whose scales lie in shared memory.  That costs as much of its bandwidth
// as reading N numbers a thread: with 128 tokens a block took 1330 clocks.  So N = 128 has the tokens as the rows, as a pair has: eight warps, a token
// and 64 outputs a thread, one number as scale (512x4096x4096 28.8 us before).  In the end the CTAs of a cluster share out a thread's sums, and
// each adds up its own in the order of the CTAs.
template <int N> struct L8Small {
    static constexpr bool ROWS = N == 128;                                          // tokens are rows
    static constexpr int COLUMNS = ROWS ? 64 : N;                                   // a thread's sums
    static constexpr int SUMS = ROWS ? 256 : 128, THREADS = SUMS + 64;              // threads that add up; two warps more
    static constexpr int CTAS = ROWS ? 1 : 2;                                       // an SM
    static constexpr int STAGES = N <= 16 ? 6 : N <= 32 ? 5 : 6;
    static constexpr int BUFFERS = 4;                                               // of sums
    static constexpr uint32_t STAGE = L8_SLAB + N * 128, SMEM = STAGES * STAGE + 1024;
    // in the end the stages hold what the CTAs of a cluster hand over, and rows of y on their way out
    static_assert(SUMS * COLUMNS * 4 + (ROWS ? SUMS * (COLUMNS + 4) * 4 : 0) <= STAGES * STAGE);
};

// The CTAs of a cluster share out a thread's sums: each gets the others' of its own part, [CTA][sums / V][thread][V], so that the lanes of a warp
// store side by side (a lane's sums side by side took three times as long), and adds them up in the order of the CTAs.  store(first, values)
// takes V of them.
template <int COLUMNS, int PARTS, int THREADS, class Store> __device__ __forceinline__ void l8_join(const float (&acc)[COLUMNS], float* sums, uint32_t rank, Store&& store) {
    constexpr int SHARE = COLUMNS / PARTS, V = SHARE < 4 ? SHARE : 4;
    float* const mine = sums + threadIdx.x * V;
    if (threadIdx.x < THREADS) {
#pragma unroll
        for (int r = 0; r < PARTS; ++r) {
            const uint32_t to = l8_map_shared(mine + rank * THREADS * SHARE, r);
#pragma unroll
            for (int c = 0; c < SHARE; c += V) {
                const float* f = acc + r * SHARE + c;
                if constexpr (V == 4)
                    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + 4 * c * THREADS), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]) : "memory");
                else
                    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to + 4 * c * THREADS), "f"(f[0]), "f"(f[1]) : "memory");
            }
        }
    }
    l8_cluster_sync();
    if (threadIdx.x >= THREADS) return;
#pragma unroll
    for (int c = 0; c < SHARE; c += V) {
        float f[V] = {};
#pragma unroll
        for (int r = 0; r < PARTS; ++r) {
            const float* from = mine + (r * SHARE + c) * THREADS;
            if constexpr (V == 4) {
                const float4 v = *reinterpret_cast<const float4*>(from);
                f[0] += v.x; f[1] += v.y; f[2] += v.z; f[3] += v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(from);
                f[0] += v.x; f[1] += v.y;
            }
        }
        store((int)rank * SHARE + c, f);
    }
}

template <class T, int N> __global__ void __launch_bounds__(L8Small<N>::THREADS, L8Small<N>::CTAS)
linear8_small_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, const L8Args a, int* error_flag) {
    using S = L8Small<N>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[S::STAGES], empty[S::STAGES], made[S::BUFFERS], taken[S::BUFFERS];
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    __shared__ __align__(16) float scales[S::ROWS ? 1 : 4][2][S::ROWS ? 4 : N];      // of each warp: a block's scales of all tokens, times the weight's
    const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem0 = (smem_u32(raw) + 1023u) & ~1023u;
    float* const parts_of = reinterpret_cast<float*>(raw + (smem0 - smem_u32(raw)));
    uint32_t rank, parts;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
    const int tile = blockIdx.x / parts, m0 = tile % a.m_tiles * N, n0 = tile / a.m_tiles * 128;
    const int b0 = (int)((long long)a.blocks * rank / parts), b1 = (int)((long long)a.blocks * (rank + 1) / parts);

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < S::BUFFERS; ++b) { mbar_init(&made[b], 1); mbar_init(&taken[b], S::SUMS / 32); }
        mbar_fence_init();
    }
    if (wid == S::SUMS / 32 + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(N * S::BUFFERS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    l8_before_sync();
    __syncthreads();
    l8_after_sync();
    const uint32_t tmem = tmem_base;
    bool ok = true;
    uint64_t pairs[S::COLUMNS / 2];
#pragma unroll
    for (int i = 0; i < S::COLUMNS / 2; ++i) pairs[i] = 0;
    // what a thread adds up: row m or n of the tile, and COLUMNS columns from `first` on
    const int line = threadIdx.x & 127, first = S::ROWS ? (wid >> 2) * S::COLUMNS : 0;

    if (wid == S::SUMS / 32) {      // ---- copies
        if (l8_elect()) {
            l8_prefetch_map(&w_map);
            l8_prefetch_map(&x_map);
            int stage = 0, turn = 0;
            for (int b = b0; b < b1; ++b) {
                if (!mbar_wait(&empty[stage], (turn & 1) ^ 1)) { ok = false; break; }
                const uint32_t to = smem0 + stage * S::STAGE;
                mbar_arrive_expect_tx(&full[stage], S::STAGE);
                l8_load<1>(to, &w_map, smem_u32(&full[stage]), b * E4M3_BLOCK, n0);
                l8_load<1>(to + L8_SLAB, &x_map, smem_u32(&full[stage]), b * E4M3_BLOCK, m0);
                if (++stage == S::STAGES) { stage = 0; ++turn; }
            }
            if (!ok) {      // no copy is left in flight
                gave_up = 1;
                for (int i = 0; i < S::STAGES; ++i) {
                    const int t = i < stage ? turn : turn - 1;
                    if (t >= 0) mbar_wait(&full[i], t & 1);
                }
            }
            if (!l8_released(empty, stage, turn)) gave_up = 1;
        }
        __syncwarp();
    } else if (wid == S::SUMS / 32 + 1) {      // ---- products
        if (l8_elect()) {
            int stage = 0, turn = 0, it = 0;
            for (; it < b1 - b0; ++it) {
                const int buffer = it % S::BUFFERS;
                if (!mbar_wait(&full[stage], turn & 1) || !mbar_wait(&taken[buffer], ((it / S::BUFFERS) & 1) ^ 1)) { ok = false; break; }
                l8_after_sync();
                const uint32_t w = l8_desc(smem0 + stage * S::STAGE), x = l8_desc(smem0 + stage * S::STAGE + L8_SLAB);
                l8_multiply<1>(tmem + buffer * N, S::ROWS ? x : w, S::ROWS ? w : x, l8_instruction(128, N));
                l8_commit<1>(&made[buffer]);
                l8_commit<1>(&empty[stage]);
                if (++stage == S::STAGES) { stage = 0; ++turn; }
            }
            if (!ok) {      // no product is left in flight
                gave_up = 1;
                if (it > 0) mbar_wait(&made[(it - 1) % S::BUFFERS], ((it - 1) / S::BUFFERS) & 1);
            }
        }
        __syncwarp();
    } else {      // ---- sums
        const uint32_t from = tmem + ((uint32_t)(wid & 3) << 21) + first;
        const float* ws = a.ws + (long long)(n0 / E4M3_BLOCK) * a.blocks;
        const bool fours = a.whole_fours && b0 % 4 == 0;
        constexpr int PART = S::COLUMNS < 32 ? 16 : 32, READS = S::COLUMNS / PART;
        const int token = m0 + (S::ROWS ? line : lane);      // whose scales this thread reads: four blocks', and the next four on their way
        const bool reads = token < a.tokens && (S::ROWS || lane < N);
        float scale[4], x4[4] = {0.f, 0.f, 0.f, 0.f}, w4[4];
        const auto fetch = [&](int b) {
            l8_four(ws, b, a.blocks, fours, w4);
            if (reads) l8_four(a.xs + (long long)token * a.blocks, b, a.blocks, fours, x4);
        };
        fetch(b0);
        for (int it = 0; it < b1 - b0; ++it) {
            const int buffer = it % S::BUFFERS;
            if ((it & 3) == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) scale[j] = x4[j] * w4[j];
                if (b0 + it + 4 < b1) fetch(b0 + it + 4);
            }
            const float* sc = scales[S::ROWS ? 0 : wid][it & 1];
            if constexpr (!S::ROWS) {
                if (lane < N) scales[wid][it & 1][lane] = scale[0];
            }
            const uint64_t same = pack2(scale[0], scale[0]);
            scale[0] = scale[1]; scale[1] = scale[2]; scale[2] = scale[3];
            __syncwarp();
            if (!l8_wait(&made[buffer], (it / S::BUFFERS) & 1)) { ok = false; break; }
            l8_after_sync();
            uint32_t r[READS][PART];
#pragma unroll
            for (int i = 0; i < READS; ++i) l8_read(r[i], from + buffer * N + i * PART);
            l8_wait_loads();
#pragma unroll
            for (int i = 0; i < READS; ++i) l8_hold(r[i]);
            l8_before_sync();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&taken[buffer])) : "memory");
#pragma unroll
            for (int c = 0; c < S::COLUMNS; c += 4) {
                const uint32_t* v = &r[c / PART][c % PART];
                ulonglong2 s2 = make_ulonglong2(same, same);
                if constexpr (!S::ROWS) s2 = *reinterpret_cast<const ulonglong2*>(sc + c);
                pairs[c / 2] = fma2(l8_pair(v[0], v[1]), s2.x, pairs[c / 2]);
                pairs[c / 2 + 1] = fma2(l8_pair(v[2], v[3]), s2.y, pairs[c / 2 + 1]);
            }
        }
        if (!ok && lane == 0) gave_up = 1;
    }
    // Everything loaded has been multiplied and everything multiplied has been added: the stages are free.
    float acc[S::COLUMNS];
#pragma unroll
    for (int i = 0; i < S::COLUMNS / 2; ++i) unpack2(pairs[i], acc[2 * i], acc[2 * i + 1]);
    const T* bias = static_cast<const T*>(a.bias);
    const bool vectors = a.whole_rows;
    // Where the rows of y are no whole vectors, those of a warp go through shared memory, so that neighbouring lanes store a row's elements
    // (a row a lane, element by element, 333x2000x5003 took 29.4 us).
    constexpr int PITCH = S::COLUMNS + 4 / sizeof(T);
    T* const mine = reinterpret_cast<T*>(parts_of + S::SUMS * S::COLUMNS) + wid * 32 * PITCH;
    const auto store = [&](int c, auto& f) {
        constexpr int V = sizeof(f) / sizeof(float);
        if constexpr (S::ROWS) {
            const int m = m0 + line, n = n0 + first + c;
            if (m >= a.tokens) return;
            T* out = static_cast<T*>(a.y) + (long long)m * a.outer + n;
            if (bias != nullptr) {
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] += n + j < a.outer ? to_float(bias[n + j]) : 0.f;
            }
            if (!vectors) {      // through shared memory: see below
#pragma unroll
                for (int j = 0; j < V; ++j) mine[lane * PITCH + c + j] = from_float<T>(f[j]);
            } else if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    if (n + j < a.outer) *reinterpret_cast<float4*>(out + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
            } else if constexpr (V == 8) {
                if (n < a.outer) *reinterpret_cast<uint4*>(out) = Vec16<T>::pack(f);
            } else {
                if (n < a.outer) *reinterpret_cast<uint2*>(out) = make_uint2(pack_pair<T>(f[0], f[1]), pack_pair<T>(f[2], f[3]));
            }
        } else {
            const int n = n0 + line;
            if (n >= a.outer) return;
            const float shift = bias != nullptr ? to_float(bias[n]) : 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (m0 + c + j < a.tokens) static_cast<T*>(a.y)[(long long)(m0 + c + j) * a.outer + n] = from_float<T>(f[j] + shift);
        }
    };
    if (parts == 1) {
        if (threadIdx.x < S::SUMS) {
#pragma unroll
            for (int c = 0; c < S::COLUMNS; c += 8) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = acc[c + j];
                store(c, f);
            }
        }
    } else {
        __syncthreads();
        l8_cluster_sync();      // ... of all CTAs
        switch (parts) {
            case 2: l8_join<S::COLUMNS, 2, S::SUMS>(acc, parts_of, rank, store); break;
            case 4: l8_join<S::COLUMNS, 4, S::SUMS>(acc, parts_of, rank, store); break;
            default: l8_join<S::COLUMNS, 8, S::SUMS>(acc, parts_of, rank, store); break;
        }
    }
    if (S::ROWS && !vectors && threadIdx.x < S::SUMS) {
        __syncwarp();
        const int share = S::COLUMNS / (int)parts, c0 = (int)rank * share, m1 = m0 + (wid & 3) * 32, rows = min(32, a.tokens - m1);
        T* out = static_cast<T*>(a.y) + (long long)m1 * a.outer + n0 + first + c0;
        for (int i = lane; i < rows * share; i += 32) {      // share: a power of two
            const int row = i >> (31 - __clz(share)), c = i & (share - 1);
            if (n0 + first + c0 + c < a.outer) out[(long long)row * a.outer + c] = mine[row * PITCH + c0 + c];
        }
    }
    l8_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && gave_up) *error_flag = 1;
    if (wid == S::SUMS / 32 + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(N * S::BUFFERS));
}

struct L8Call {
    const uint8_t *x, *w;
    long long x_stride, w_stride, inner;
    int type;
    L8Args a;
};

template <class T> int launch_linear8_pair(L8Call c, int* flag, cudaStream_t s) {
    CUtensorMap x_map, w_map, y_map;
    if (!make_byte_rows_map(&x_map, c.x, c.a.tokens, c.inner, c.x_stride, 128) || !make_byte_rows_map(&w_map, c.w, c.a.outer, c.inner, c.w_stride, 128)) return ADDER_ERR_CUDA;
    y_map = x_map;
    if (c.a.whole_rows && !make_rows_map(&y_map, c.a.y, c.type, c.a.tokens, c.a.outer, 32)) return ADDER_ERR_CUDA;
    c.a.m_tiles = (c.a.tokens + 255) / 256;
    c.a.n_tiles = (c.a.outer + 255) / 256;
    const auto kernel = linear8_pair_kernel<T>;
    const int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), L8P_SMEM);
    if (st != ADDER_OK) return st;
    const long long tiles = (long long)c.a.m_tiles * c.a.n_tiles;
    if (tiles > 2147483647LL / 8) return ADDER_ERR_UNSUPPORTED;
    return launch_clusters(kernel, 2 * (unsigned)std::min((long long)sm_count() / 2, tiles), L8P_THREADS, L8P_SMEM, 2, s, x_map, w_map, y_map, c.a, flag);
}

template <class T, int N> int launch_linear8_small(L8Call c, int* flag, cudaStream_t s) {
    using S = L8Small<N>;
    CUtensorMap x_map, w_map;
    if (!make_byte_rows_map(&x_map, c.x, c.a.tokens, c.inner, c.x_stride, N) || !make_byte_rows_map(&w_map, c.w, c.a.outer, c.inner, c.w_stride, 128)) return ADDER_ERR_CUDA;
    c.a.m_tiles = (c.a.tokens + N - 1) / N;
    c.a.n_tiles = (c.a.outer + 127) / 128;
    const auto kernel = linear8_small_kernel<T, N>;
    const int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), S::SMEM);
    if (st != ADDER_OK) return st;
    const long long tiles = (long long)c.a.m_tiles * c.a.n_tiles;
    if (tiles > 2147483647LL / 8) return ADDER_ERR_UNSUPPORTED;
    int parts = 1;      // as long as all CTAs are resident at once and have two blocks each
    while (parts < 8 && tiles * parts * 2 <= (long long)S::CTAS * sm_count() && c.a.blocks >= 4 * parts) parts *= 2;
    return launch_clusters(kernel, (unsigned)(tiles * parts), S::THREADS, S::SMEM, parts, s, x_map, w_map, c.a, flag);
}

template <class T> int launch_linear8(const L8Call& c, cudaStream_t s) {
    int* flag = nullptr;
    const int st = device_error_flag(&flag);
    if (st != ADDER_OK) return st;
    const int tokens = c.a.tokens;
    if (tokens <= 16) return launch_linear8_small<T, 16>(c, flag, s);
    if (tokens <= 32) return launch_linear8_small<T, 32>(c, flag, s);
    // Turns of all SMs: a pair's takes some 1.6 times as long as that of CTAs of 128 x 128.  us by those and by pairs: 512x4096x4096 15.7 and 20.3,
    // 200x4096x4096 13.0 and 19.9, 300x4096x11008 31.5 and 37.1; on the other side 700x4096x4096 28.8 and 20.7, 160x4096x32000 58 and 38,
    // 2048x512x2048 11.3 and 8.3.
    const long long pair_tiles = (long long)((tokens + 255) / 256) * ((c.a.outer + 255) / 256), small_tiles = (long long)((tokens + 127) / 128) * ((c.a.outer + 127) / 128);
    const long long pair_turns = (pair_tiles + sm_count() / 2 - 1) / (sm_count() / 2), small_turns = (small_tiles + sm_count() - 1) / sm_count();
    if (tokens <= 128 || 5 * small_turns <= 8 * pair_turns) return launch_linear8_small<T, 128>(c, flag, s);
    return launch_linear8_pair<T>(c, flag, s);
}

int quant_check(long long rows, long long d, long long x_stride, long long values_stride, int dtype) {
    if (rows < 0 || d <= 0 || x_stride < 0 || values_stride < d) return ADDER_ERR_BAD_SHAPE;
    if (dtype < ADDER_TYPE_F32 || dtype > ADDER_TYPE_F16 || d > 2147483647LL - 1024 || rows > 2147483647LL) return ADDER_ERR_UNSUPPORTED;
    return ADDER_OK;
}
template <class T> bool quant_vectors(const QuantArgs& a) {
    return a.d % 4 == 0 && a.x_stride % 4 == 0 && a.values_stride % 4 == 0 && aligned_to(a.x, 4 * sizeof(T)) && aligned_to(a.values, 4);
}

}  // namespace
}  // namespace adder

using namespace adder;

extern "C" {

int adder_b200_quantize_rows(const void* x, unsigned char* values, float* scales, long long rows, long long d, long long x_stride,
                             long long values_stride, int dtype, void* stream) {
    const int st = quant_check(rows, d, x_stride, values_stride, dtype);
    if (st != ADDER_OK) return st;
    if (rows == 0) return ADDER_OK;
    if (!x || !values || !scales) return ADDER_ERR_NULL_POINTER;
    if (!aligned_to(x, dtype == ADDER_TYPE_F32 ? 4 : 2) || !aligned_to(scales, 4)) return ADDER_ERR_ALIGNMENT;
    const QuantArgs a{x, values, scales, rows, x_stride, values_stride, (int)d};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int VE = Vec16<T>::N;
        const bool vectors = d % VE == 0 && x_stride % VE == 0 && values_stride % VE == 0 && aligned_to(x, 16) && aligned_to(values, VE);
        const long long each = vectors ? 32LL * QR_VECTORS * VE : QR_BLOCKS * E4M3_BLOCK, grid = (rows * ((d + each - 1) / each) + 7) / 8;
        if (grid > 2147483647LL) return (int)ADDER_ERR_UNSUPPORTED;
        if (vectors) quantize_vectors_kernel<T><<<(unsigned)grid, 256, 0, s>>>(a);
        else quantize_rows_kernel<T><<<(unsigned)grid, 256, 0, s>>>(a);
        return launched();
    });
}

int adder_b200_quantize_weight(const void* w, unsigned char* values, float* scales, long long rows, long long d, long long w_stride,
                               long long values_stride, int dtype, void* stream) {
    const int st = quant_check(rows, d, w_stride, values_stride, dtype);
    if (st != ADDER_OK) return st;
    if (rows == 0) return ADDER_OK;
    if (!w || !values || !scales) return ADDER_ERR_NULL_POINTER;
    if (!aligned_to(w, dtype == ADDER_TYPE_F32 ? 4 : 2) || !aligned_to(scales, 4)) return ADDER_ERR_ALIGNMENT;
    const long long grid = (rows + E4M3_BLOCK - 1) / E4M3_BLOCK * ((d + E4M3_BLOCK - 1) / E4M3_BLOCK);
    if (grid > 2147483647LL) return ADDER_ERR_UNSUPPORTED;
    const QuantArgs a{w, values, scales, rows, w_stride, values_stride, (int)d};
    return with_type(dtype, [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        if (quant_vectors<T>(a)) quantize_weight_kernel<T, true><<<(unsigned)grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
        else quantize_weight_kernel<T, false><<<(unsigned)grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
        return launched();
    });
}

int adder_b200_linear_8bit(const unsigned char* x, const float* x_scales, const unsigned char* w, const float* w_scales, const void* bias, void* y,
                           long long tokens, long long inner, long long outer, long long x_stride, long long w_stride, int dtype, void* stream) {
    if (tokens < 0 || inner <= 0 || outer < 0 || x_stride < inner || w_stride < inner) return ADDER_ERR_BAD_SHAPE;
    if (dtype < ADDER_TYPE_F32 || dtype > ADDER_TYPE_F16 || tokens > 2147483647LL / 2 || inner > 2147483647LL / 2 || outer > 2147483647LL / 2) return ADDER_ERR_UNSUPPORTED;
    if (tokens == 0 || outer == 0) return ADDER_OK;
    if (!x || !x_scales || !w || !w_scales || !y) return ADDER_ERR_NULL_POINTER;
    const unsigned size = dtype == ADDER_TYPE_F32 ? 4 : 2;
    if (!aligned_to(x, 16) || !aligned_to(w, 16) || x_stride % 16 != 0 || w_stride % 16 != 0 || !aligned_to(x_scales, 4) || !aligned_to(w_scales, 4) ||
        !aligned_to(bias, size) || !aligned_to(y, size))
        return ADDER_ERR_ALIGNMENT;
    const L8Call c{x, w, x_stride, w_stride, inner, dtype, {x_scales, w_scales, bias, y, (int)tokens, (int)outer, (int)((inner + E4M3_BLOCK - 1) / E4M3_BLOCK), 0, 0,
                    (inner + E4M3_BLOCK - 1) / E4M3_BLOCK % 4 == 0 && aligned_to(x_scales, 16) && aligned_to(w_scales, 16),
                    outer * size % 16 == 0 && aligned_to(y, 16)}};
    return with_type(dtype, [&](auto* type) { return launch_linear8<std::remove_pointer_t<decltype(type)>>(c, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
