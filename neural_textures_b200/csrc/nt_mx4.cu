// nt_mx4.cu -- 4-bit microscaled matrices: quantisation from fp16 / bf16 / fp32 and back
// (nt_mx4_quantize, nt_mx4_dequantize).
//
// Bound by HBM where a matrix is large and its rows lie along the memory: 16384 x 8192 bf16 in blocks of 16 takes 60 us
// (5.7 TB/s) and 54 us back (6.4 TB/s), 8192 x 8192 fp32 52 and 48 us.  Transposed (8192 x 8192 fp32 85 us) and unaligned rows (16384 x 8191
// bf16 118 us) are bound by their narrower loads.
#include "nt_mx4.cuh"

namespace nt {
namespace mx4 {

constexpr int kThreads = 256;
constexpr int kGroupCols = 128;  // columns of one thread block of the quantise kernels

struct QuantizeLaunch {
    const void *src;
    int64_t row_stride, col_stride;
    uint8_t *data, *scales;
    int64_t pitch;
    int32_t rows, cols, tiles, groups;  // scale tiles a row of tiles; column groups
};

// How a row's values are read: 16 bytes at a time, through shared memory (rows that are not aligned: a warp reads
// 32 consecutive values of a row at a time), or one by one at any stride.
enum Access { kVector, kStaged, kStrided };
constexpr int kStagePitch = kGroupCols + 4;

// 16 values of a row from column c (0 past the matrix).
template <class T, Access ACCESS>
__device__ __forceinline__ void load16(const QuantizeLaunch &p, int64_t row, int64_t c, T (&v)[16])
{
    const T *src = static_cast<const T *>(p.src) + row * p.row_stride;
    if (ACCESS == kVector && row < p.rows && c + 16 <= p.cols) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i)
            reinterpret_cast<uint4 *>(v)[i] = __ldg(reinterpret_cast<const uint4 *>(src + c) + i);
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const bool in = row < p.rows && c + i < p.cols;
        v[i] = in ? src[(c + i) * p.col_stride] : from_f32<T>(0.f);
    }
}

// Larger magnitudes of two packed 16-bit values, as fp16 / bf16 bits without signs.  As integers NaN and
// infinity compare above every number.
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t v) { return __vmaxu2(m, v & 0x7fff7fffu); }
template <class T>
__device__ __forceinline__ uint32_t f32_bits(uint32_t v)  // of one 16-bit value
{
    return __float_as_uint(to_f32(*reinterpret_cast<const T *>(&v)));
}

// The bits of max |v| as fp32.
template <class T, int N>
__device__ __forceinline__ uint32_t amax_bits(const T (&v)[N])
{
    uint32_t m = 0;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) m = max_abs2(m, reinterpret_cast<const uint32_t *>(v)[i]);
        return f32_bits<T>(max(m & 0xffffu, m >> 16));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        return m;
    }
}

template <class T, int BLOCK, int N>
__device__ __forceinline__ void quantize_codes(const T (&v)[N], uint32_t byte, uint32_t (&codes)[N / 8])
{
    const float inv = inverse_scale<BLOCK>(byte), s = BLOCK == 16 ? scale_value<16>(byte) : 0.f;
#pragma unroll
    for (int q = 0; q < N / 8; ++q) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 y = scaled2<BLOCK, sizeof(T) == 4>(make_float2(to_f32(v[8 * q + i]), to_f32(v[8 * q + i + 1])), inv, s);
            f[i] = y.x;
            f[i + 1] = y.y;
        }
        codes[q] = codes8(f);
    }
}

// Rows along the memory.  A thread block takes 128 rows x 128 columns.  BLOCK / 4 lanes share a row
// (16 values each), so that they hold the four scales of one word; a lane takes rows r, r + 32,
// r + 64 and r + 96, whose words are the 16 bytes of row r in the scale tile: one store.  NARROW: no more than 64
// columns, and two tiles of rows instead.
template <class T, int BLOCK, Access ACCESS, bool NARROW>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantizeLaunch p)
{
    __shared__ T stage[ACCESS == kStaged ? 32 * kStagePitch : 1];
    after_previous();
    constexpr int LPR = NARROW ? 4 : BLOCK / 4, RPW = 32 / LPR;
    constexpr bool kHalves = NARROW || BLOCK == 16;  // four warps cover the rows of a tile
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t tile = NARROW ? 2 * (int64_t)blockIdx.x + (warp >> 2) : blockIdx.x / p.groups;
    const int group = NARROW ? 0 : blockIdx.x % p.groups;
    const int half = kHalves && !NARROW ? warp >> 2 : 0;
    const int residue = (kHalves ? warp & 3 : warp) * RPW + lane / LPR;
    const int64_t c = (int64_t)group * kGroupCols + half * 64 + (lane % LPR) * 16;
    uint32_t words[4];
    constexpr int U = ACCESS == kStaged ? 1 : sizeof(T) == 2 ? 4 : 2;  // rows in flight
#pragma unroll
    for (int j0 = 0; j0 < 4; j0 += U) {
        alignas(16) T v[U][16];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (ACCESS != kStaged) load16<T, ACCESS>(p, tile * kTileRows + (j0 + u) * 32 + residue, c, v[u]);
        if (ACCESS == kStaged) {
            const int64_t row0 = tile * kTileRows + j0 * 32 + warp * 4, col0 = (int64_t)group * kGroupCols + lane;
            T w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool in = row0 + i / 4 < p.rows && col0 + i % 4 * 32 < p.cols;
                w[i] = in ? static_cast<const T *>(p.src)[(row0 + i / 4) * p.row_stride + col0 + i % 4 * 32] : from_f32<T>(0.f);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 16; ++i) stage[(warp * 4 + i / 4) * kStagePitch + i % 4 * 32 + lane] = w[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[0][i] = stage[residue * kStagePitch + (int)(c - (int64_t)group * kGroupCols) + i];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t row = tile * kTileRows + (j0 + u) * 32 + residue;
            uint32_t m = amax_bits(v[u]);
            if (BLOCK == 32) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            const uint32_t byte = scale_byte<BLOCK>(m);
            uint32_t codes[2];
            quantize_codes<T, BLOCK>(v[u], byte, codes);
            if (row < p.rows && c < row_pitch(p.cols) * 2)
                *reinterpret_cast<uint2 *>(p.data + row * p.pitch + (c >> 1)) = make_uint2(codes[0], codes[1]);
            uint32_t w = byte << (8 * ((lane % LPR) * 16 / BLOCK));
            w |= __shfl_xor_sync(0xffffffffu, w, LPR / 2);
            w |= __shfl_xor_sync(0xffffffffu, w, LPR / 4);
            words[j0 + u] = w;
        }
    }
    const int tcol = BLOCK == 16 ? group * 2 + half : group;
    if (lane % LPR == 0 && tcol < p.tiles && (!NARROW || tile * kTileRows < p.rows))
        *reinterpret_cast<uint4 *>(p.scales + (tile * p.tiles + tcol) * kTileBytes + residue * 16) =
            make_uint4(words[0], words[1], words[2], words[3]);
}

// Columns along the memory (a transposed matrix): lanes along the rows, so that a warp's load of one column is
// contiguous; a thread quantises 32 columns of its row, 16 bytes of codes, without any exchange.  PAIRS: of two
// neighbouring rows of a 16-bit matrix, for loads of 4 bytes.  The warps of a block lie along the rows: 1 KB of every
// column rather than 256 bytes of four times the columns (8190 x 8192 fp16: 61.3 -> 59.5 us).
constexpr int kColumnsGroup = 32;  // columns of a thread block
constexpr int kColumnsTiles = 2;   // row tiles of a thread block, twice that for pairs

template <class T, int BLOCK>
__device__ __forceinline__ void quantize_column_run(const QuantizeLaunch &p, const T (&v)[32], int64_t row, int64_t c0)
{
    uint32_t codes[4], bytes;
    if (BLOCK == 32) {
        bytes = scale_byte<32>(amax_bits(v));
        quantize_codes<T, 32>(v, bytes, codes);
    } else {
        const T(&lo)[16] = *reinterpret_cast<const T(*)[16]>(&v[0]);
        const T(&hi)[16] = *reinterpret_cast<const T(*)[16]>(&v[16]);
        const uint32_t b0 = scale_byte<16>(amax_bits(lo)), b1 = scale_byte<16>(amax_bits(hi));
        quantize_codes<T, 16>(lo, b0, *reinterpret_cast<uint32_t(*)[2]>(&codes[0]));
        quantize_codes<T, 16>(hi, b1, *reinterpret_cast<uint32_t(*)[2]>(&codes[2]));
        bytes = b0 | b1 << 8;
    }
    if (row < p.rows && c0 < row_pitch(p.cols) * 2)
        *reinterpret_cast<uint4 *>(p.data + row * p.pitch + (c0 >> 1)) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
    const int k = (int)(c0 / BLOCK);  // first block
    if ((k >> 2) < p.tiles && (row & ~127) < p.rows) {  // rows past the matrix too: their scales are 0
        uint8_t *at = p.scales + ((row >> 7) * p.tiles + (k >> 2)) * kTileBytes + (row & 31) * 16 + (row >> 5 & 3) * 4 + (k & 3);
        if (BLOCK == 16) *reinterpret_cast<uint16_t *>(at) = (uint16_t)bytes;
        else *at = (uint8_t)bytes;
    }
}

template <class T, int BLOCK, bool PAIRS>
__global__ void __launch_bounds__(kThreads) quantize_columns_kernel(const QuantizeLaunch p)
{
    after_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t band = blockIdx.x / p.groups, c0 = (int64_t)(blockIdx.x % p.groups) * kColumnsGroup;
    if constexpr (PAIRS) {
        const int64_t row = band * 2 * kColumnsTiles * kTileRows + warp * 64 + 2 * lane;
        const T *src = static_cast<const T *>(p.src) + row;
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            w[i] = 0;
            if (c0 + i >= p.cols) continue;
            if (row + 1 < p.rows) w[i] = *reinterpret_cast<const uint32_t *>(src + (c0 + i) * p.col_stride);
            else if (row < p.rows) w[i] = *reinterpret_cast<const uint16_t *>(src + (c0 + i) * p.col_stride);
        }
        alignas(4) T v[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                reinterpret_cast<uint32_t *>(v)[i] = __byte_perm(w[2 * i], w[2 * i + 1], h ? 0x7632 : 0x5410);
            quantize_column_run<T, BLOCK>(p, v, row + h, c0);
        }
    } else {
        const int64_t row = band * kColumnsTiles * kTileRows + warp * 32 + lane;
        const T *src = static_cast<const T *>(p.src) + row;
        alignas(4) T v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = row < p.rows && c0 + i < p.cols ? src[(c0 + i) * p.col_stride] : from_f32<T>(0.f);
        quantize_column_run<T, BLOCK>(p, v, row, c0);
    }
}

template <class T, int BLOCK>
cudaError_t launch_quantize(QuantizeLaunch p, cudaStream_t st)
{
    p.tiles = tiles_per_row(p.cols, BLOCK);
    const bool unit = p.col_stride == 1 || p.cols == 1, columns = !unit && p.row_stride == 1;
    // a scale tile's padding is written too: whole tiles of 4 blocks
    const bool pairs = sizeof(T) == 2 && is_aligned(p.src, 4) && p.col_stride % 2 == 0;
    const int64_t width = columns ? kColumnsGroup : kGroupCols, height = columns ? (pairs ? 2 : 1) * kColumnsTiles * kTileRows : kTileRows;
    p.groups = (int32_t)(((int64_t)p.tiles * 4 * BLOCK + width - 1) / width);
    int64_t blocks = (p.rows + height - 1) / height * p.groups;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const bool vec = unit && is_aligned(p.src, 16) && (p.rows == 1 || p.row_stride * sizeof(T) % 16 == 0);
    void (*kernel)(QuantizeLaunch) = quantize_rows_kernel<T, BLOCK, kStrided, false>;
    if (columns) {
        kernel = quantize_columns_kernel<T, BLOCK, false>;
        if constexpr (sizeof(T) == 2)
            if (pairs) kernel = quantize_columns_kernel<T, BLOCK, true>;
    } else if (vec && p.cols <= 64) {
        blocks = ((int64_t)p.rows + 2 * kTileRows - 1) / (2 * kTileRows);
        kernel = quantize_rows_kernel<T, BLOCK, kVector, true>;
    } else if (vec) {
        kernel = quantize_rows_kernel<T, BLOCK, kVector, false>;
    } else if (unit) {
        kernel = quantize_rows_kernel<T, BLOCK, kStaged, false>;
    }
    return launch_next(kernel, dim3((unsigned)blocks), kThreads, 0, st, 1, p);
}

// ---- back --------------------------------------------------------------------------------

struct DequantizeLaunch {
    const uint8_t *data, *scales;
    void *dst;
    int64_t pitch, row_stride;
    int32_t rows, cols, tiles;
    int32_t lanes_log2;  // lanes that share a row
    int32_t col_blocks;  // thread blocks that share a row
    int32_t vec;         // 16-byte stores
};

constexpr int kDequantRows = 4;  // rows of one lane

template <class T>
__device__ __forceinline__ uint32_t pack_pair(float2 f)
{
    if constexpr (sizeof(T) == 4) {
        return 0;
    } else {
        const auto h = f32_pair<T>(f);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// A lane takes 8 codes (one word) of a row and writes 16 or 32 bytes.  WIDE: a warp to a row and 32 rows to a block, whose
// codes, scales and results then lie at constant distances.
template <class T, int BLOCK, bool WIDE>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const DequantizeLaunch p)
{
    after_previous();
    const int lanes_log2 = WIDE ? 5 : p.lanes_log2, lanes = 1 << lanes_log2;
    const int sub = threadIdx.x & (lanes - 1);
    const int rows_per_pass = kThreads >> lanes_log2;
    const int64_t row0 = (int64_t)(blockIdx.x / p.col_blocks) * rows_per_pass * kDequantRows + (threadIdx.x >> lanes_log2);
    const int64_t c = ((int64_t)(blockIdx.x % p.col_blocks) * lanes + sub) * 8;
    __shared__ alignas(16) T turn[WIDE ? kThreads / 32 : 1][256];
    const bool in = c < p.cols;  // every lane of a warp stays for its exchange
    const uint8_t *const data = p.data + row0 * p.pitch + (c >> 1);
    const uint8_t *const scales = p.scales + (WIDE ? scale_at(row0, (int)(c / BLOCK), p.tiles) : 0);
    uint32_t codes[kDequantRows], bytes[kDequantRows];
#pragma unroll
    for (int j = 0; j < kDequantRows; ++j) {
        const int64_t row = row0 + (int64_t)j * rows_per_pass;
        codes[j] = bytes[j] = 0;
        if (row >= p.rows || !in) continue;
        codes[j] = __ldg(reinterpret_cast<const uint32_t *>(data + (int64_t)j * rows_per_pass * p.pitch));
        // WIDE: 8 rows on, 16 bytes each, in the same quarter of the tile
        bytes[j] = __ldg(WIDE ? scales + 128 * j : p.scales + scale_at(row, (int)(c / BLOCK), p.tiles));
    }
    T *dst = static_cast<T *>(p.dst) + row0 * p.row_stride + c;
#pragma unroll
    for (int j = 0; j < kDequantRows; ++j, dst += rows_per_pass * p.row_stride) {
        if (row0 + (int64_t)j * rows_per_pass >= p.rows) break;
        const float s = scale_value<BLOCK>(bytes[j]);
        uint32_t h2[4];
        values8(codes[j], h2);
        alignas(16) T out[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2 *>(&h2[i])), f2(s));
            if constexpr (sizeof(T) == 2) {
                reinterpret_cast<uint32_t *>(out)[i] = pack_pair<T>(f);
            } else {
                out[2 * i] = f.x;
                out[2 * i + 1] = f.y;
            }
        }
        if (WIDE && !p.vec) {  // unaligned rows: a warp's 256 values through shared memory, 32 consecutive ones at a time
            T *const mine = turn[threadIdx.x >> 5];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                reinterpret_cast<uint4 *>(mine + 8 * sub)[i] = reinterpret_cast<const uint4 *>(out)[i];
            __syncwarp();
            T *const first = dst - 8 * sub;
            const int64_t left = p.cols - (c - 8 * sub);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (32 * i + sub < left) first[32 * i + sub] = mine[32 * i + sub];
        } else if (WIDE && sizeof(T) == 4 && c - 8 * sub + 256 <= p.cols) {  // the same for whole aligned rows, 512 bytes at a time
            T *const mine = turn[threadIdx.x >> 5];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 2; ++i) reinterpret_cast<uint4 *>(mine + 8 * sub)[i] = reinterpret_cast<const uint4 *>(out)[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 2; ++i)
                reinterpret_cast<uint4 *>(dst - 8 * sub)[32 * i + sub] = reinterpret_cast<const uint4 *>(mine)[32 * i + sub];
        } else if (p.vec && c + 8 <= p.cols) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<const uint4 *>(out)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < p.cols) dst[i] = out[i];
        }
    }
}

template <class T, int BLOCK>
cudaError_t launch_dequantize(DequantizeLaunch p, cudaStream_t st)
{
    p.tiles = tiles_per_row(p.cols, BLOCK);
    const int64_t words = ((int64_t)p.cols + 7) / 8;
    p.lanes_log2 = 0;
    while (p.lanes_log2 < 5 && (1 << p.lanes_log2) < words) ++p.lanes_log2;
    p.vec = is_aligned(p.dst, 16) && p.row_stride * sizeof(T) % 16 == 0;
    p.col_blocks = (int32_t)((words + (1 << p.lanes_log2) - 1) >> p.lanes_log2);
    const int64_t rows_per_block = (int64_t)(kThreads >> p.lanes_log2) * kDequantRows;
    const int64_t grid = ((int64_t)p.rows + rows_per_block - 1) / rows_per_block * p.col_blocks;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return launch_next(p.lanes_log2 == 5 ? dequantize_kernel<T, BLOCK, true> : dequantize_kernel<T, BLOCK, false>, dim3((unsigned)grid),
                       kThreads, 0, st, 1, p);
}

// Shared checks of a matrix argument.
nt_status check_matrix(const NtMx4Matrix *m, const char *name)
{
    NT_LAYER_REQUIRE(m, "%s is null", name);
    NT_LAYER_REQUIRE(m->block == 16 || m->block == 32, "%s: block must be 16 or 32 (got %d)", name, m->block);
    NT_LAYER_REQUIRE(m->rows >= 0 && m->cols >= 1 && m->rows <= 0x7fffff00 && m->cols <= 0x7fffff00, "%s: %d x %d is not a matrix size", name, m->rows, m->cols);
    NT_LAYER_REQUIRE(m->pitch >= row_pitch(m->cols) && m->pitch % 16 == 0,
                     "%s: pitch must be a multiple of 16 and at least %lld (got %lld)", name,
                     (long long)row_pitch(m->cols), (long long)m->pitch);
    NT_LAYER_REQUIRE(m->rows == 0 || (m->data && m->scales && is_aligned(m->data, 16) && is_aligned(m->scales, 16)),
                     "%s: data and scales must be non-null 16-byte aligned device pointers", name);
    return NT_OK;
}

}  // namespace mx4
}  // namespace nt

using namespace nt;

extern "C" {

size_t nt_mx4_pitch(int32_t cols) { return cols < 1 ? 0 : (size_t)mx4::row_pitch(cols); }

size_t nt_mx4_scales_bytes(int32_t rows, int32_t cols, int32_t block)
{
    if (rows < 1 || cols < 1 || (block != 16 && block != 32)) return 0;
    return (size_t)(((int64_t)rows + mx4::kTileRows - 1) / mx4::kTileRows) * mx4::tiles_per_row(cols, block) * mx4::kTileBytes;
}

nt_status nt_mx4_quantize(const void *src, int32_t dtype, int64_t row_stride, int64_t col_stride,
                          const NtMx4Matrix *dst, nt_stream_t stream)
{
    nt_status st = mx4::check_matrix(dst, "dst");
    if (st != NT_OK) return st;
    const int size = layer_dtype_size(dtype);
    NT_LAYER_REQUIRE(size, "dtype must be NT_DTYPE_F16, NT_DTYPE_BF16 or NT_DTYPE_F32 (got %d)", dtype);
    NT_LAYER_REQUIRE(row_stride >= 0 && col_stride >= 0, "strides must be non-negative");
    if (dst->rows == 0) return NT_OK;
    NT_LAYER_REQUIRE(src && is_aligned(src, size), "src must be a non-null device pointer aligned to its element");
    mx4::QuantizeLaunch p = {};
    p.src = src;
    p.row_stride = row_stride;
    p.col_stride = col_stride;
    p.data = static_cast<uint8_t *>(dst->data);
    p.scales = static_cast<uint8_t *>(dst->scales);
    p.pitch = dst->pitch;
    p.rows = dst->rows;
    p.cols = dst->cols;
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
    if (dst->block == 16)
        e = dtype == NT_DTYPE_F16    ? mx4::launch_quantize<__half, 16>(p, s)
            : dtype == NT_DTYPE_BF16 ? mx4::launch_quantize<__nv_bfloat16, 16>(p, s)
                                     : mx4::launch_quantize<float, 16>(p, s);
    else
        e = dtype == NT_DTYPE_F16    ? mx4::launch_quantize<__half, 32>(p, s)
            : dtype == NT_DTYPE_BF16 ? mx4::launch_quantize<__nv_bfloat16, 32>(p, s)
                                     : mx4::launch_quantize<float, 32>(p, s);
    return e == cudaSuccess ? NT_OK : set_error(NT_ERR_CUDA, "4-bit quantise: %s", cudaGetErrorString(e));
}

nt_status nt_mx4_dequantize(const NtMx4Matrix *src, void *dst, int32_t dtype, int64_t row_stride, nt_stream_t stream)
{
    nt_status st = mx4::check_matrix(src, "src");
    if (st != NT_OK) return st;
    const int size = layer_dtype_size(dtype);
    NT_LAYER_REQUIRE(size, "dtype must be NT_DTYPE_F16, NT_DTYPE_BF16 or NT_DTYPE_F32 (got %d)", dtype);
    NT_LAYER_REQUIRE(src->rows <= 1 || row_stride >= src->cols, "row_stride (%lld) must be at least cols (%d)",
                     (long long)row_stride, src->cols);
    if (src->rows == 0) return NT_OK;
    NT_LAYER_REQUIRE(dst && is_aligned(dst, size), "dst must be a non-null device pointer aligned to its element");
    mx4::DequantizeLaunch p = {};
    p.data = static_cast<const uint8_t *>(src->data);
    p.scales = static_cast<const uint8_t *>(src->scales);
    p.dst = dst;
    p.pitch = src->pitch;
    p.row_stride = row_stride;
    p.rows = src->rows;
    p.cols = src->cols;
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
    if (src->block == 16)
        e = dtype == NT_DTYPE_F16    ? mx4::launch_dequantize<__half, 16>(p, s)
            : dtype == NT_DTYPE_BF16 ? mx4::launch_dequantize<__nv_bfloat16, 16>(p, s)
                                     : mx4::launch_dequantize<float, 16>(p, s);
    else
        e = dtype == NT_DTYPE_F16    ? mx4::launch_dequantize<__half, 32>(p, s)
            : dtype == NT_DTYPE_BF16 ? mx4::launch_dequantize<__nv_bfloat16, 32>(p, s)
                                     : mx4::launch_dequantize<float, 32>(p, s);
    return e == cudaSuccess ? NT_OK : set_error(NT_ERR_CUDA, "4-bit read-back: %s", cudaGetErrorString(e));
}

}  // extern "C"
