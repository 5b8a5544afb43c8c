// nt_mx4_product.cu -- d = activation(alpha a b^T + bias) of two 4-bit microscaled matrices on the
// tensor cores' block-scaled product (nt_mx4_product).
//
// One operand's rows are the accumulator's 128 lanes (the lane operand), the other's its bn columns
// (the column operand).  A thread block computes 128 x bn tiles, 256 values of K a stage:
//   warp 0      copies: TMA tiles of codes (rows of 128 bytes, or 32 or 64 where K is no longer, swizzled;
//               zeros past the matrix) and the scale tiles, which lie in memory as tensor memory wants them.  A
//               column operand of one tile and one stage, the weights of a narrow layer, comes once: copies
//               of short rows are bound by their number, which the SMs of a GPC share
//   warp 1      per stage: scale tiles shared -> tensor memory, four products of K = 64, commit
//   warps 4-11  epilogue: accumulator -> scale, bias, activation, rounding -> shared -> rows of d by TMA.  Two
//               warps for each quarter of the lanes: they halve a tile's columns, or, of tiles of 64 columns
//               and less, take every other tile
// There are two accumulators in tensor memory, four of 64 columns and less, so that the epilogue of a tile runs
// under the products of the next; blocks take tiles gridDim apart.  Two of 256 columns and the scales do
// not fit: they share 96 columns, which the epilogue reads first.
//
// Few rows (m <= 64): the weights' rows go to the lanes, and bn is m rounded up, so that a token costs no
// empty columns.  Few tiles: a cluster of up to 8 blocks splits K, leaves its partial sums in shared
// memory, and each block joins its share of the columns in rank order.
//
// One B200: 8192^3 bf16 in blocks of 16 4.1 PFLOP/s alone, 3.4 in a loop at the power limit; a stage of 128 x 256 x 256 takes about
// 1,100 cycles where the tensor core needs 512 and shared memory 850.  262144 x 64 x 64 13 us (3.3 TB/s), 1 x 4096 x 4096
// 6.4 us.
//
// Every wait is bounded; a timeout sets bit 0 of the status word that nt_read_device_status returns.
#include <cuda.h>

#include <algorithm>

#include "nt_mx4.cuh"
#include "nt_umma.cuh"

namespace nt {
namespace mx4 {

__device__ unsigned int g_product_status;  // bit 0: a bounded wait gave up

struct ProductLaunch {
    const uint8_t *l_scales, *c_scales;  // of the lane and the column operand
    int32_t l_rows, c_rows, k;
    int32_t bn, l_tiles, c_tiles;
    int32_t scale_tiles;       // scale tiles of 128 rows of either operand
    int32_t stages, stage_bytes;
    int32_t resident;          // the column operand is one tile of one stage: loaded once, behind the stages
    int32_t row_bytes;         // codes of a row in a stage: 32, 64 or 128 bytes
    uint64_t layout;           // their swizzle and group stride, as descriptor bits
    int32_t split;             // thread blocks of a cluster, each with a share of K
    int32_t swapped;           // 1: lanes are b's rows (d's columns)
    int32_t dtype, tma_store;  // tma_store: d's address and rows suit a tensor map
    int32_t turns;             // epilogue warps of a quarter take turns, tile by tile
    const float *bias;
    int32_t activation;
    float alpha;
    void *d;
    int64_t row_stride;
};

constexpr int kThreads = 384, kEpilogueWarps = 8;
constexpr int kMaxStages = 8;
constexpr int kMaxAcc = 4;
constexpr int kAccStep = 160, kNarrowAccStep = 64;  // columns between two accumulators
constexpr int kStaging = 32 * 128;  // epilogue staging of a warp: 32 rows of 128 bytes, swizzled as TMA expects
constexpr uint32_t kTmemCols = 512, kScaleCol = 416, kScaleCols = 48;

struct Control {
    alignas(8) uint64_t full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t acc_full[kMaxAcc], acc_empty[kMaxAcc];
    uint64_t acc_part[2];  // the columns that the other accumulator shares are free
    uint32_t tmem;
};

struct Shared {
    alignas(1024) uint8_t staging[kEpilogueWarps][kStaging];
    alignas(16) float bias[kEpilogueWarps][64];
    Control ctl;
};

// A launch parameter in a register: the loops branch on these, and a chain of branches each behind a load from
// the constant bank cost the epilogue of a tile 500 cycles, the issuing warps 200 a stage.
__device__ __forceinline__ int held(int v)
{
    asm volatile("" : "+r"(v));
    return v;
}
__device__ __forceinline__ float held(float v)
{
    asm volatile("" : "+f"(v));
    return v;
}
template <class T>
__device__ __forceinline__ T *held(T *v)
{
    asm volatile("" : "+l"(v));
    return v;
}

// What the epilogue reads of the launch.
struct Output {
    int bn, l_rows, c_rows, dtype, tma_store;
    float alpha;
    const float *bias;
    void *d;
    int64_t row_stride;
    __device__ __forceinline__ explicit Output(const ProductLaunch &p)
        : bn(held(p.bn)), l_rows(held(p.l_rows)), c_rows(held(p.c_rows)), dtype(held(p.dtype)), tma_store(held(p.tma_store)),
          alpha(held(p.alpha)), bias(held(p.bias)), d(held(p.d)), row_stride(p.row_stride)
    {
    }
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, int x, int y, uint32_t src)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n\t"
                 "cp.async.bulk.commit_group;" ::"l"(map), "r"(x), "r"(y), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Codes: `layout` with the address of the first row.
__device__ __forceinline__ uint64_t codes_desc(uint32_t addr, uint64_t layout) { return umma::desc(addr, 16, 0) | layout; }

// A scale tile: 32 rows of 16 bytes -> 4 columns of all four lane quarters.
__device__ __forceinline__ void copy_scale_tile(uint32_t tmem, uint32_t addr)
{
    const uint64_t d = umma::desc(addr, 0, 128);
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}

// Instruction descriptor: E2M1 operands, 128 x n, scale format (0: E4M3, 1: E8M0), the byte of each
// scale word at which the step's scales start.
template <int BLOCK>
__device__ __forceinline__ uint32_t idesc(int n, uint32_t scale_byte)
{
    return (scale_byte << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((BLOCK == 32 ? 1u : 0u) << 23) |
           (8u << 24) | (scale_byte << 29);
}

template <int BLOCK>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t sa, uint32_t sb, uint32_t acc)
{
    if (BLOCK == 16)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(desc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(desc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
}

__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// One lane of a converged warp, the same one every time.  The issuing warps run their loops whole and only
// their asynchronous instructions under this predicate: operands then stay in uniform registers, without
// which every such instruction took 80 to 100 cycles to issue.
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity)
{
    if (umma::mbar_wait(bar, parity)) return true;
    atomicOr(&g_product_status, 1u);
    return false;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t peer_address(uint32_t addr, uint32_t rank)
{
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    return remote;
}
__device__ __forceinline__ void peer_store(uint32_t remote, uint32_t v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}

__device__ __forceinline__ void store_one(const Output &p, int64_t at, float v)
{
    if (p.dtype == NT_DTYPE_F32) static_cast<float *>(p.d)[at] = v;
    else if (p.dtype == NT_DTYPE_F16) static_cast<__half *>(p.d)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p.d)[at] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint32_t pack2(int dtype, float lo, float hi)
{
    if (dtype == NT_DTYPE_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Lanes are b's rows: lane = column of d, accumulator columns = rows of d; a warp's store is contiguous.  The two
// warps of a quarter take every other 32 columns (`half`).
template <int ACT>
__device__ __forceinline__ void epilogue_swapped(const Output &p, uint32_t tmem, int lane0, int col0, int half)
{
    const int64_t n = lane0 + (threadIdx.x & 127);
    const float bias = p.bias && n < p.l_rows ? __ldg(p.bias + n) : 0.f;
    for (int c0 = 32 * half; c0 < p.bn; c0 += 64) {
        uint32_t v[32];
        ld32(tmem + c0, v);
        umma::wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float2 y = activate2<ACT>(__ffma2_rn(f2(p.alpha), make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), f2(bias)));
            const int64_t m = col0 + c0 + i;
            if (n < p.l_rows) {
                if (c0 + i < p.bn && m < p.c_rows) store_one(p, m * p.row_stride + n, y.x);
                if (c0 + i + 1 < p.bn && m + 1 < p.c_rows) store_one(p, (m + 1) * p.row_stride + n, y.y);
            }
        }
    }
}

// Lanes are a's rows: a warp stages 32 rows x 128 bytes (64 columns, or 32 of fp32) and writes them row by row.
// `i0` is its first column range and `di` the distance to its next; of 256 columns, those from `first` on come
// first, and `part` is told when they have been read.  `bias_at`: the columns that `bias` holds.
template <int ACT>
__device__ __forceinline__ void epilogue_rows(const Output &p, const CUtensorMap *d_map, uint32_t tmem, int lane0, int col0, int i0,
                                              int di, int first, uint32_t part, uint8_t *mine, float *bias, int &bias_at)
{
    const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3;
    const int size = p.dtype == NT_DTYPE_F32 ? 4 : 2, width = 128 / size;
    for (; i0 < p.bn; i0 += di) {
        const int c0 = p.bn > kAccStep ? i0 ^ first : i0, n0 = col0 + c0;
        if (p.bn > kAccStep && i0 >= 128 && i0 < 128 + di) {  // 128 columns have been read, the shared ones among them
            umma::fence_before();
            __syncwarp();
            if (lane == 0) umma::mbar_arrive(part);
        }
        if (n0 >= p.c_rows) continue;
        if (p.bias && bias_at != n0) {
            for (int i = lane; i < width; i += 32) bias[i] = n0 + i < p.c_rows ? __ldg(p.bias + n0 + i) : 0.f;
            bias_at = n0;
            __syncwarp();
        }
        uint8_t *const row = mine + lane * 128;
        // both halves of 64 columns are on their way before the first is waited for
        const bool two = size == 2 && c0 + 32 < p.bn;
        uint32_t v[2][32];
        ld32(tmem + c0, v[0]);
        if (two) ld32(tmem + c0 + 32, v[1]);
        umma::wait_ld();
        if (p.tma_store && elect_one()) store_wait_read();  // the last store has read the staging
        __syncwarp();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (s && !two) break;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 b = *reinterpret_cast<const float4 *>(bias + 32 * s + i);
                uint32_t(&w)[32] = v[s];
                const float2 y0 = activate2<ACT>(
                    __ffma2_rn(f2(p.alpha), make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1])), make_float2(b.x, b.y)));
                const float2 y1 = activate2<ACT>(
                    __ffma2_rn(f2(p.alpha), make_float2(__uint_as_float(w[i + 2]), __uint_as_float(w[i + 3])), make_float2(b.z, b.w)));
                w[i] = __float_as_uint(y0.x);
                w[i + 1] = __float_as_uint(y0.y);
                w[i + 2] = __float_as_uint(y1.x);
                w[i + 3] = __float_as_uint(y1.y);
            }
            if (size == 4) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    *reinterpret_cast<uint4 *>(row + ((i ^ (lane & 7)) << 4)) =
                        make_uint4(v[s][4 * i], v[s][4 * i + 1], v[s][4 * i + 2], v[s][4 * i + 3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t h[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        h[e] = pack2(p.dtype, __uint_as_float(v[s][8 * i + 2 * e]), __uint_as_float(v[s][8 * i + 2 * e + 1]));
                    *reinterpret_cast<uint4 *>(row + ((4 * s + i ^ (lane & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
                }
            }
        }
        const int64_t m0 = lane0 + quarter * 32;
        if (p.tma_store) {
            umma::fence_async_smem();
            __syncwarp();
            if (m0 < p.l_rows && elect_one()) tma_store_2d(d_map, n0, (int)m0, smem_u32(mine));
            __syncwarp();
            continue;
        }
        __syncwarp();
        // rows of d that no tensor map takes: a row at a time, 4 bytes a lane where its address allows it, eight in flight
        const int rows = (int)min((int64_t)32, p.l_rows - m0), bytes = min(min(width, p.bn - c0), p.c_rows - n0) * size;
        uint8_t *const dst = static_cast<uint8_t *>(p.d) + (m0 * p.row_stride + n0) * size;
        const int64_t pitch = p.row_stride * size;
        const bool words = ((reinterpret_cast<uintptr_t>(p.d) | (uintptr_t)pitch) & 3) == 0;
        for (int r0 = 0; r0 < rows; r0 += 8) {
            uint32_t v[8];
#pragma unroll
            for (int r = 0; r < 8; ++r)
                v[r] = *reinterpret_cast<const uint32_t *>(mine + (r0 + r) * 128 + (((lane >> 2) ^ r) << 4) + (lane & 3) * 4);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                uint8_t *const at = dst + (r0 + r) * pitch + 4 * lane;
                if (r0 + r >= rows || 4 * lane >= bytes) continue;
                if (words && 4 * lane + 4 <= bytes) {
                    *reinterpret_cast<uint32_t *>(at) = v[r];
                } else {  // 16-bit values
                    *reinterpret_cast<uint16_t *>(at) = (uint16_t)v[r];
                    if (4 * lane + 4 <= bytes) *reinterpret_cast<uint16_t *>(at + 2) = (uint16_t)(v[r] >> 16);
                }
            }
        }
        __syncwarp();
    }
}

// The tiles of a block, `step` apart in the order lane tiles first; kept as (lane tile, column tile) without
// divisions.
struct Tiles {
    int l, c, dl, dc, l_tiles, c_tiles;
    __device__ __forceinline__ Tiles(const ProductLaunch &p)
    {
        const unsigned first = blockIdx.x / p.split, step = gridDim.x / p.split;
        l_tiles = held(p.l_tiles);
        c_tiles = held(p.c_tiles);
        l = (int)(first % (unsigned)l_tiles), c = (int)(first / (unsigned)l_tiles);
        dl = (int)(step % (unsigned)l_tiles), dc = (int)(step / (unsigned)l_tiles);
    }
    __device__ __forceinline__ bool valid() const { return c < c_tiles; }
    __device__ __forceinline__ void next()
    {
        l += dl;
        c += dc;
        if (l >= l_tiles) l -= l_tiles, ++c;
    }
};

struct EpilogueArgs {
    const CUtensorMap *d_map;
    uint32_t acc_full, acc_empty, acc_part, accs;  // accs: the accumulators' lanes of this warp
    uint8_t *staging;
    float *bias;
    int turns, swapped;
};

// All tiles of the block, for one epilogue warp.
template <int ACT>
__device__ __forceinline__ void epilogue(const Output &out, const ProductLaunch &p, const EpilogueArgs &e)
{
    const int lane = threadIdx.x & 31, half = (threadIdx.x - 128) >> 7, width = out.dtype == NT_DTYPE_F32 ? 32 : 64;
    const int i0 = e.turns ? 0 : half * width, di = e.turns ? width : 2 * width;
    const int num_acc = e.turns ? 4 : 2, acc_step = e.turns ? kNarrowAccStep : kAccStep;
    int buf = 0, bias_at = -1;
    uint32_t phase = 0;
    e.bias[lane] = e.bias[lane + 32] = 0.f;
    __syncwarp();
    for (Tiles t(p); t.valid(); t.next()) {
        if (!e.turns || (buf & 1) == half) {
            const uint32_t acc = e.accs + buf * acc_step;
            if (!__all_sync(0xffffffffu, wait(e.acc_full + 8 * buf, phase))) break;
            umma::fence_after();
            if (e.swapped)
                epilogue_swapped<ACT>(out, acc, t.l * 128, t.c * out.bn, half);
            else
                epilogue_rows<ACT>(out, e.d_map, acc, t.l * 128, t.c * out.bn, i0, di, buf ? 0 : 128, e.acc_part + 8 * buf, e.staging,
                                   e.bias, bias_at);
            umma::fence_before();
            __syncwarp();
            if (lane == 0) umma::mbar_arrive(e.acc_empty + 8 * buf);
        }
        if (++buf == num_acc) buf = 0, phase ^= 1;
    }
    if (out.tma_store && elect_one()) store_wait();
    __syncwarp();
}

// A block's partial sums to the blocks of the cluster that own their columns: there, `sums` holds
// [block][own column][lane].
constexpr int kPartialPitch = 129;  // lanes of a column and a bank more: columns are read across too

__device__ __forceinline__ void send_partials(const Output &out, int split, int rank, uint32_t acc_full, uint32_t acc, uint32_t sums, int half)
{
    const bool ok = __all_sync(0xffffffffu, wait(acc_full, 0));
    umma::fence_after();
    cluster_wait();  // the peers run
    if (!ok) return;
    const int lane = threadIdx.x & 127, cols = out.bn / split, log = __ffs(cols) - 1;  // powers of two
    for (int c0 = 32 * half; c0 < out.bn; c0 += 64) {
        uint32_t v[32];
        ld32(acc + c0, v);
        umma::wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int c = c0 + i;
            if (c >= out.bn) break;
            peer_store(peer_address(sums + ((rank * cols + (c & (cols - 1))) * kPartialPitch + lane) * 4, c >> log), v[i]);
        }
    }
}

template <int BLOCK>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap l_map, const __grid_constant__ CUtensorMap c_map,
                   const __grid_constant__ CUtensorMap d_map, const ProductLaunch p)
{
    constexpr int kTiles = BLOCK == 16 ? 4 : 2;  // scale tiles of a stage
    extern __shared__ uint8_t raw[];
    __shared__ Shared sh;
    Control &ctl = sh.ctl;
    uint8_t *stages = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5;
    const uint32_t base = smem_u32(stages), full = smem_u32(ctl.full), empty = smem_u32(ctl.empty),
                   acc_full = smem_u32(ctl.acc_full), acc_empty = smem_u32(ctl.acc_empty), acc_part = smem_u32(ctl.acc_part);
    const int bn = held(p.bn), row_bytes = held(p.row_bytes), num_stages = held(p.stages), stage_bytes = held(p.stage_bytes),
              split = held(p.split);
    // of a stage: the lane operand, its scales, the column operand, its scales; the latter two behind all stages
    // where they are resident
    const bool resident = held(p.resident);
    const int ls_off = 128 * row_bytes, lane_bytes = ls_off + kTiles * kTileBytes,
              c_off = resident ? num_stages * stage_bytes : (lane_bytes + 1023) & ~1023, cs_off = c_off + bn * row_bytes;
    const int c_scales = bn > 128 ? 2 : 1;  // row tiles of the column operand's scales
    const int k_steps = held((p.k + 63) / 64), stage_steps = row_bytes / 32, k_stages = (k_steps + stage_steps - 1) / stage_steps;
    const int rank = split > 1 ? blockIdx.x % split : 0;
    const int k_lo = split > 1 ? (int)((int64_t)k_stages * rank / split) : 0,
              k_hi = split > 1 ? (int)((int64_t)k_stages * (rank + 1) / split) : k_stages;

    if (threadIdx.x == 0) {
        for (int i = 0; i < num_stages; ++i) {
            umma::mbar_init(full + 8 * i, 1);
            umma::mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < kMaxAcc; ++i) {
            umma::mbar_init(acc_full + 8 * i, 1);
            umma::mbar_init(acc_empty + 8 * i, p.turns ? kEpilogueWarps / 2 : kEpilogueWarps);
        }
        for (int i = 0; i < 2; ++i) umma::mbar_init(acc_part + 8 * i, kEpilogueWarps);
        umma::mbar_fence_init();
    }
    if (warp == 2) umma::alloc(smem_u32(&ctl.tmem), kTmemCols);
    umma::fence_before();
    __syncthreads();
    umma::fence_after();
    const uint32_t tmem = ctl.tmem;
    if (split > 1) cluster_arrive();  // peers write into this block's shared memory: only once it runs
    after_previous();

    if (warp == 0) {
        int s = 0;
        uint32_t phase = 0;
        bool ok = true;
        const int scale_tiles = held(p.scale_tiles), c_rows = held(p.c_rows);
        const uint8_t *const l_scales = held(p.l_scales), *const c_scale_data = held(p.c_scales);
        bool columns = true;  // to be loaded
        for (Tiles t(p); ok && t.valid(); t.next()) {
            const int lt = t.l, c0 = t.c * bn, cs = min(c_scales, (c_rows - c0 + 127) >> 7);
            const uint8_t *const ls = l_scales + (int64_t)lt * scale_tiles * kTileBytes;
            const uint8_t *const sc = c_scale_data + (int64_t)(c0 >> 7) * scale_tiles * kTileBytes;
            for (int ks = k_lo; ks < k_hi; ++ks) {
                if (!(ok = __all_sync(0xffffffffu, wait(empty + 8 * s, phase ^ 1)))) break;
                const uint32_t at = base + s * stage_bytes, bar = full + 8 * s;
                const int st = min(kTiles, scale_tiles - ks * kTiles);
                const int64_t from = tile_offset(ks * kTiles);
                const uint32_t ct = resident ? base : at;
                if (elect_one()) {
                    expect_tx(bar, ls_off + st * kTileBytes + (columns ? bn * row_bytes + cs * st * kTileBytes : 0));
                    tma_2d(at, &l_map, ks * row_bytes, lt * 128, bar);
                    bulk_copy(at + ls_off, ls + from, st * kTileBytes, bar);
                    if (columns) {
                        tma_2d(ct + c_off, &c_map, ks * row_bytes, c0, bar);
                        bulk_copy(ct + cs_off, sc + from, st * kTileBytes, bar);
                        if (cs == 2)
                            bulk_copy(ct + cs_off + kTiles * kTileBytes, sc + (int64_t)scale_tiles * kTileBytes + from, st * kTileBytes, bar);
                    }
                }
                columns = !resident;
                __syncwarp();
                if (++s == num_stages) s = 0, phase ^= 1;
            }
        }
        // no copy is in flight when the block ends, whether or not the products took them all
        for (int i = 0; i < num_stages; ++i) umma::mbar_wait(full + 8 * i, i < s ? phase : phase ^ 1, 1u << 16);
    } else if (warp == 1) {
        int s = 0, buf = 0, sbuf = 0;
        uint32_t phase = 0, acc_phase = 0, part_phase = 0;
        bool ok = true, first = true, columns = true;  // columns: their scales are to be copied
        const int num_acc = p.turns ? 4 : 2, acc_step = p.turns ? kNarrowAccStep : kAccStep;
        const uint64_t da0 = codes_desc(base, p.layout), db0 = codes_desc(base + c_off, p.layout);
        const uint32_t id0 = idesc<BLOCK>(bn, 0), id1 = BLOCK == 16 ? id0 : idesc<BLOCK>(bn, 2);
        for (Tiles t(p); ok && t.valid(); t.next()) {
            if (!(ok = __all_sync(0xffffffffu, wait(acc_empty + 8 * buf, acc_phase ^ 1)))) break;
            if (bn > kAccStep && !first && !(ok = __all_sync(0xffffffffu, wait(acc_part + 8 * (buf ^ 1), part_phase)))) break;
            if (buf == 0) part_phase ^= !first;
            first = false;
            umma::fence_after();
            const uint32_t acc = tmem + buf * acc_step;
            for (int ks = k_lo; ks < k_hi; ++ks) {
                const uint32_t at = base + s * stage_bytes, sl = tmem + kScaleCol + sbuf * kScaleCols,
                               sc = resident ? tmem + kScaleCol + 16 : sl + 16;
                const int steps = min(stage_steps, k_steps - ks * stage_steps);
                const uint64_t step = (uint64_t)((uint32_t)(s * stage_bytes) >> 4), da = da0 + step, db = resident ? db0 : db0 + step;
                if (!(ok = __all_sync(0xffffffffu, wait(full + 8 * s, phase)))) break;
                umma::fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < kTiles; ++i)
                        if (i * (4 / kTiles) < steps) {
                            copy_scale_tile(sl + 4 * i, at + ls_off + i * kTileBytes);
                            if (columns) {
                                const uint32_t from = (resident ? base : at) + cs_off;
                                copy_scale_tile(sc + 4 * i * c_scales, from + i * kTileBytes);
                                if (c_scales == 2) copy_scale_tile(sc + 8 * i + 4, from + (kTiles + i) * kTileBytes);
                            }
                        }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < steps) {
                            const int tile = BLOCK == 16 ? i : i >> 1;
                            mma<BLOCK>(acc, da + 2 * i, db + 2 * i, i & 1 ? id1 : id0, sl + 4 * tile, sc + 4 * tile * c_scales,
                                       ks > k_lo || i > 0);
                        }
                    umma::commit(empty + 8 * s);
                    if (ks + 1 == k_hi) umma::commit(acc_full + 8 * buf);
                }
                __syncwarp();
                columns = !resident;
                if (++s == num_stages) s = 0, phase ^= 1;
                sbuf ^= 1;
            }
            if (++buf == num_acc) buf = 0, acc_phase ^= 1;
        }
    } else if (warp >= 4) {
        const Output out(p);
        const uint32_t accs = tmem + ((uint32_t)(warp & 3) << 21);
        if (split > 1) {
            send_partials(out, split, rank, acc_full, accs, base + num_stages * stage_bytes, (warp - 4) >> 2);
        } else {
            const EpilogueArgs e = {&d_map, acc_full, acc_empty, acc_part, accs, sh.staging[warp - 4], sh.bias[warp - 4], held(p.turns),
                                    held(p.swapped)};
            switch (p.activation) {
            case NT_ACT_RELU: epilogue<NT_ACT_RELU>(out, p, e); break;
            case NT_ACT_SILU: epilogue<NT_ACT_SILU>(out, p, e); break;
            case NT_ACT_GELU: epilogue<NT_ACT_GELU>(out, p, e); break;
            default: epilogue<NT_ACT_NONE>(out, p, e); break;
            }
        }
    }
    __syncwarp();
    if (split > 1) {
        if (warp < 4) cluster_wait();  // of the arrival at the start; the others waited before they sent
        __syncthreads();
        cluster_arrive();
        cluster_wait();  // every block's partial sums have arrived
        const Output out(p);
        const Tiles t(p);
        const int lane0 = t.l * 128, col0 = t.c * bn;
        const int cols = bn / split, lo = cols * rank;
        const float *sums = reinterpret_cast<const float *>(stages + num_stages * stage_bytes);
        for (int i = threadIdx.x; i < cols * 128; i += kThreads) {
            // consecutive threads along d's rows
            const int l = p.swapped ? i & 127 : i / cols, c = p.swapped ? i >> 7 : i % cols;
            float sum = 0.f;
            for (int r = 0; r < split; ++r) sum += sums[(r * cols + c) * kPartialPitch + l];
            const int64_t row = p.swapped ? col0 + lo + c : lane0 + l, col = p.swapped ? lane0 + l : col0 + lo + c;
            if (lane0 + l < out.l_rows && col0 + lo + c < out.c_rows)
                store_one(out, row * out.row_stride + col, activate1(fmaf(out.alpha, sum, out.bias ? __ldg(out.bias + col) : 0.f), p.activation));
        }
    }
    umma::fence_before();
    __syncthreads();
    umma::fence_after();
    if (warp == 2) umma::dealloc(tmem, kTmemCols);
}

// ---- host ------------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled()
{
    static const EncodeTiled fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// d, written in boxes of 32 rows x 128 bytes.
bool encode_output(CUtensorMap *map, const ProductLaunch &p)
{
    const EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    const int size = p.dtype == NT_DTYPE_F32 ? 4 : 2;
    const cuuint64_t shape[2] = {(cuuint64_t)p.c_rows, (cuuint64_t)p.l_rows}, stride[1] = {(cuuint64_t)p.row_stride * size};
    const cuuint32_t box[2] = {128u / size, 32}, step[2] = {1, 1};
    return encode(map, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.d, shape, stride, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Codes as a byte matrix, read in boxes of `box_rows` rows x `row_bytes`.
bool encode_codes(CUtensorMap *map, const NtMx4Matrix *m, int box_rows, int row_bytes)
{
    const EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    const cuuint64_t size[2] = {(cuuint64_t)row_pitch(m->cols), (cuuint64_t)m->rows}, stride[1] = {(cuuint64_t)m->pitch};
    const cuuint32_t box[2] = {(cuuint32_t)row_bytes, (cuuint32_t)box_rows}, step[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, m->data, size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  row_bytes == 32   ? CU_TENSOR_MAP_SWIZZLE_32B
                  : row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                    : CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Columns of a tile when the lanes are a's rows.  Tiles of several start at a multiple of 128 columns, where
// their scale tile starts; a narrower one is the only one.  256 columns read the lane operand half as
// often; they are taken where that does not cost a wave of blocks.
int choose_bn(int64_t m, int64_t n, int sms)
{
    if (n <= 128) return n <= 32 ? 32 : n <= 64 ? 64 : 128;
    const int64_t rows = ceil_div(m, 128), wide = ceil_div(rows * ceil_div(n, 256), sms), narrow = ceil_div(rows * ceil_div(n, 128), sms);
    return wide * 3 <= narrow * 2 ? 256 : 128;
}

template <int BLOCK>
nt_status launch_product(const NtMx4Matrix *a, const NtMx4Matrix *b, ProductLaunch p, cudaStream_t st)
{
    constexpr int kTiles = BLOCK == 16 ? 4 : 2;
    const int sms = sm_count();
    p.swapped = a->rows <= 64;
    const NtMx4Matrix *l = p.swapped ? b : a, *c = p.swapped ? a : b;
    p.bn = !p.swapped ? choose_bn(a->rows, b->rows, sms)
           : a->rows <= 8 ? 8 : a->rows <= 16 ? 16 : a->rows <= 32 ? 32 : 64;
    p.l_rows = l->rows;
    p.c_rows = c->rows;
    p.k = a->cols;
    // a box that reaches past the end of its rows is copied several times slower than a whole one
    p.row_bytes = p.k <= 64 ? 32 : p.k <= 128 ? 64 : 128;
    p.layout = (uint64_t)(p.row_bytes / 2) << 32 | (uint64_t)(p.row_bytes == 32 ? 6 : p.row_bytes == 64 ? 4 : 2) << 61;
    p.l_tiles = (int32_t)ceil_div(l->rows, 128);
    p.c_tiles = (int32_t)ceil_div(c->rows, p.bn);
    p.scale_tiles = tiles_per_row(p.k, BLOCK);
    p.l_scales = static_cast<const uint8_t *>(l->scales);
    p.c_scales = static_cast<const uint8_t *>(c->scales);
    const int64_t tiles = (int64_t)p.l_tiles * p.c_tiles, k_stages = ceil_div(p.k, 2 * p.row_bytes);
    // split K while blocks stand idle and every share keeps two stages
    p.split = 1;
    while (p.split < 8 && p.bn <= 128 && tiles * p.split * 2 <= sms && k_stages >= p.split * 4) p.split *= 2;
    p.turns = !p.swapped && p.split == 1 && p.bn <= 64;
    p.resident = p.split == 1 && p.c_tiles == 1 && k_stages == 1 && tiles > sms;
    const int64_t lane_bytes = 128 * p.row_bytes + kTiles * kTileBytes,
                  column_bytes = ceil_div(p.bn * p.row_bytes + (p.bn > 128 ? 2 : 1) * kTiles * kTileBytes, 1024) * 1024;
    p.stage_bytes = (int32_t)(ceil_div(lane_bytes, 1024) * 1024 + (p.resident ? 0 : column_bytes));
    const size_t partials = p.split > 1 ? (size_t)p.bn * kPartialPitch * 4 : 0;
    const size_t behind = p.resident ? (size_t)column_bytes : partials;
    const int room = 227 * 1024 - 1024 - (int)sizeof(Shared) - (int)behind;
    p.stages = std::min(kMaxStages, room / p.stage_bytes);
    const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + behind;
    const int64_t grid = p.split > 1 ? tiles * p.split : std::min<int64_t>(tiles, sms);
    CUtensorMap l_map, c_map, d_map = {};
    if (!encode_codes(&l_map, l, 128, p.row_bytes) || !encode_codes(&c_map, c, p.bn, p.row_bytes))
        return set_error(NT_ERR_CUDA, "4-bit product: the tensor maps could not be encoded");
    // d by TMA where 16-byte rows allow it, and 64 columns of a tile fill a row of the staging
    p.tma_store = p.tma_store && !p.swapped && p.split == 1 && (p.bn >= 64 || p.dtype == NT_DTYPE_F32) && encode_output(&d_map, p);
    const void *kernel = reinterpret_cast<const void *>(&product_kernel<BLOCK>);
    cudaError_t e = set_smem_limit(kernel, 227 * 1024 - sizeof(Shared));
    if (e == cudaSuccess)
        e = launch_next(product_kernel<BLOCK>, dim3((unsigned)grid), kThreads, smem, st, (unsigned)p.split, l_map, c_map, d_map, p);
    if (e != cudaSuccess) return set_error(NT_ERR_CUDA, "4-bit product: %s", cudaGetErrorString(e));
    return NT_OK;
}

nt_status check_matrix(const NtMx4Matrix *m, const char *name);

}  // namespace mx4

cudaError_t read_product_status(uint32_t *status, bool clear)
{
    cudaError_t e = cudaMemcpyFromSymbol(status, mx4::g_product_status, sizeof(uint32_t));
    if (e != cudaSuccess || !clear) return e;
    const uint32_t zero = 0;
    return cudaMemcpyToSymbol(mx4::g_product_status, &zero, sizeof(uint32_t));
}

}  // namespace nt

using namespace nt;

extern "C" nt_status nt_mx4_product(const NtMx4Matrix *a, const NtMx4Matrix *b, const float *bias, int32_t activation,
                                    float alpha, void *d, int32_t dtype, int64_t row_stride, nt_stream_t stream)
{
    nt_status st = mx4::check_matrix(a, "a");
    if (st != NT_OK) return st;
    if ((st = mx4::check_matrix(b, "b")) != NT_OK) return st;
    NT_LAYER_REQUIRE(a->cols == b->cols && a->block == b->block,
                     "a and b must have the same cols and block (got %d / %d and %d / %d)", a->cols, a->block, b->cols,
                     b->block);
    const int size = layer_dtype_size(dtype);
    NT_LAYER_REQUIRE(size, "dtype must be NT_DTYPE_F16, NT_DTYPE_BF16 or NT_DTYPE_F32 (got %d)", dtype);
    NT_LAYER_REQUIRE(activation >= NT_ACT_NONE && activation <= NT_ACT_GELU, "unknown activation %d", activation);
    NT_LAYER_REQUIRE(a->rows <= 1 || row_stride >= b->rows, "row_stride (%lld) must be at least b's rows (%d)",
                     (long long)row_stride, b->rows);
    if (a->rows == 0 || b->rows == 0) return NT_OK;
    NT_LAYER_REQUIRE(d && is_aligned(d, size), "d must be a non-null device pointer aligned to its element");
    NT_LAYER_REQUIRE(is_aligned(bias, 4), "bias must be a 4-byte aligned device pointer");
    mx4::ProductLaunch p = {};
    p.bias = bias;
    p.activation = activation;
    p.alpha = alpha;
    p.d = d;
    p.dtype = dtype;
    p.row_stride = row_stride;
    p.tma_store = is_aligned(d, 16) && row_stride * size % 16 == 0 && row_stride * size < (int64_t)1 << 40;
    return a->block == 16 ? mx4::launch_product<16>(a, b, p, (cudaStream_t)stream)
                          : mx4::launch_product<32>(a, b, p, (cudaStream_t)stream);
}
