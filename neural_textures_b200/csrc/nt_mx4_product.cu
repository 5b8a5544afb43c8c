// nt_mx4_product.cu -- d = activation(alpha a b^T + bias) of two 4-bit microscaled matrices
// (nt_mx4_product).
#include "nt_mx4.cuh"

namespace nt {
namespace mx4 {

struct ProductLaunch {
    const uint8_t *a, *b, *a_scales, *b_scales;
    int64_t a_pitch, b_pitch;
    int32_t m, n, k, tiles;
    const float *bias;
    int32_t activation;
    float alpha;
    void *d;
    int64_t row_stride;
};

constexpr int kSide = 64, kStep = 32;

// Codes of kSide rows x kStep columns -> fp32 values [column][row].
template <int BLOCK>
__device__ __forceinline__ void stage(const uint8_t *data, const uint8_t *scales, int64_t pitch, int rows, int cols,
                                      int tiles, int64_t row0, int k0, float (*out)[kSide + 1])
{
    const int r = threadIdx.x >> 2, q = threadIdx.x & 3;  // 4 threads a row, 8 columns each
    const int64_t row = row0 + r;
    const int k = k0 + 8 * q;
    uint32_t h2[4] = {0, 0, 0, 0};
    float s = 0.f;
    if (row < rows && k < cols) {
        values8(*reinterpret_cast<const uint32_t *>(data + row * pitch + (k >> 1)), h2);
        s = scale_value<BLOCK>(scales[scale_at(row, k / BLOCK, tiles)]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h2[i]));
        out[8 * q + 2 * i][r] = f.x * s;
        out[8 * q + 2 * i + 1][r] = f.y * s;
    }
}

template <class T, int BLOCK>
__global__ void __launch_bounds__(256) product_kernel(const ProductLaunch p)
{
    __shared__ float sa[kStep][kSide + 1], sb[kStep][kSide + 1];
    const int64_t tiles_n = (p.n + kSide - 1) / kSide;
    const int64_t m0 = blockIdx.x / tiles_n * kSide, n0 = blockIdx.x % tiles_n * kSide;
    const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < p.k; k0 += kStep) {
        stage<BLOCK>(p.a, p.a_scales, p.a_pitch, p.m, p.k, p.tiles, m0, k0, sa);
        stage<BLOCK>(p.b, p.b_scales, p.b_pitch, p.n, p.k, p.tiles, n0, k0, sb);
        __syncthreads();
#pragma unroll 8
        for (int k = 0; k < kStep; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][tm + 16 * i], sb[k][tn + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
            if (m >= p.m || n >= p.n) continue;
            const float z = p.alpha * acc[i][j] + (p.bias ? p.bias[n] : 0.f);
            static_cast<T *>(p.d)[m * p.row_stride + n] = from_f32<T>(activate(z, p.activation));
        }
}

template <class T, int BLOCK>
cudaError_t launch_product(const ProductLaunch &p, cudaStream_t st)
{
    const int64_t blocks = ((int64_t)p.m + kSide - 1) / kSide * (((int64_t)p.n + kSide - 1) / kSide);
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    product_kernel<T, BLOCK><<<(unsigned)blocks, 256, 0, st>>>(p);
    count_launch();
    return cudaGetLastError();
}

nt_status check_matrix(const NtMx4Matrix *m, const char *name);

}  // namespace mx4
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
    p.a = static_cast<const uint8_t *>(a->data);
    p.b = static_cast<const uint8_t *>(b->data);
    p.a_scales = static_cast<const uint8_t *>(a->scales);
    p.b_scales = static_cast<const uint8_t *>(b->scales);
    p.a_pitch = a->pitch;
    p.b_pitch = b->pitch;
    p.m = a->rows;
    p.n = b->rows;
    p.k = a->cols;
    p.tiles = mx4::tiles_per_row(a->cols, a->block);
    p.bias = bias;
    p.activation = activation;
    p.alpha = alpha;
    p.d = d;
    p.row_stride = row_stride;
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
    if (a->block == 16)
        e = dtype == NT_DTYPE_F16    ? mx4::launch_product<__half, 16>(p, s)
            : dtype == NT_DTYPE_BF16 ? mx4::launch_product<__nv_bfloat16, 16>(p, s)
                                     : mx4::launch_product<float, 16>(p, s);
    else
        e = dtype == NT_DTYPE_F16    ? mx4::launch_product<__half, 32>(p, s)
            : dtype == NT_DTYPE_BF16 ? mx4::launch_product<__nv_bfloat16, 32>(p, s)
                                     : mx4::launch_product<float, 32>(p, s);
    return e == cudaSuccess ? NT_OK : set_error(NT_ERR_CUDA, "4-bit product: %s", cudaGetErrorString(e));
}
