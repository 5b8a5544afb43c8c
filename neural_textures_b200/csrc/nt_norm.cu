// nt_norm.cu -- channels-last group normalisation with an activation, forward and backward
// (nt_group_norm_forward, nt_group_norm_backward).
//
// Sums over an image are split over kSplit thread blocks and joined in a fixed order:
//   forward   per (split, channel) count, mean and centred sum of squares, joined per group
//   backward  per (split, channel) sums of e and e h (e = dy act'(z)), joined per group for dx
//             and over images for dgamma and dbeta
#include <algorithm>

#include "nt_layer_common.cuh"

namespace nt {
namespace norm {

constexpr int kThreads = 256;
constexpr int kSplit = 64;

struct NormLaunch {
    NtGroupNorm p;
    int32_t per;  // channels of a group
    float *partials;  // [image][split][channel][2]
    float *sums;      // [image][group][2]
};

__device__ __forceinline__ int64_t offset(const NtFeatureMap &f, int64_t n, int64_t texel, int width)
{
    return n * f.image_stride + texel / width * f.row_stride + texel % width * f.texel_stride;
}

struct Stats {
    float count, mean, m2;
};

__device__ __forceinline__ Stats join(const Stats &a, const Stats &b)
{
    if (b.count == 0.f) return a;
    if (a.count == 0.f) return b;
    const float n = a.count + b.count, d = b.mean - a.mean, w = b.count / n;
    return {n, a.mean + d * w, a.m2 + b.m2 + d * d * a.count * w};
}

// grid (split, image): a thread takes a channel and every (256 / channels)-th texel of the split
template <class T>
__global__ void __launch_bounds__(kThreads) forward_stats_kernel(const NormLaunch L)
{
    const NtGroupNorm &p = L.p;
    __shared__ Stats part[kThreads];
    const int64_t texels = (int64_t)p.height * p.width, n = blockIdx.y;
    const int64_t lo = texels * blockIdx.x / kSplit, hi = texels * (blockIdx.x + 1) / kSplit;
    const int rows = p.channels < kThreads ? kThreads / p.channels : 1;
    for (int c0 = 0; c0 < p.channels; c0 += kThreads) {
        const int width = min(kThreads, p.channels - c0), c = c0 + threadIdx.x % width, row = threadIdx.x / width;
        Stats s = {0.f, 0.f, 0.f};
        if (row < rows)
            for (int64_t t = lo + row; t < hi; t += rows) {
                const float v = to_f32(static_cast<const T *>(p.x.data)[offset(p.x, n, t, p.width) + c]);
                s.count += 1.f;
                const float d = v - s.mean;
                s.mean += d / s.count;
                s.m2 += d * (v - s.mean);
            }
        part[threadIdx.x] = s;
        __syncthreads();
        if (row == 0) {
            for (int r = 1; r < rows; ++r) s = join(s, part[r * width + threadIdx.x]);
            float *out = L.partials + ((n * kSplit + blockIdx.x) * p.channels + c) * 2;
            out[0] = s.mean;
            out[1] = s.m2;
        }
        __syncthreads();
    }
}

// grid (group, image)
__global__ void forward_join_kernel(const NormLaunch L)
{
    const NtGroupNorm &p = L.p;
    __shared__ Stats part[kThreads];
    const int64_t texels = (int64_t)p.height * p.width, n = blockIdx.y;
    Stats s = {0.f, 0.f, 0.f};
    for (int i = threadIdx.x; i < kSplit * L.per; i += kThreads) {
        const int split = i / L.per, c = blockIdx.x * L.per + i % L.per;
        const float *in = L.partials + ((n * kSplit + split) * p.channels + c) * 2;
        const float count = (float)(texels * (split + 1) / kSplit - texels * split / kSplit);
        s = join(s, {count, in[0], in[1]});
    }
    part[threadIdx.x] = s;
    for (int w = kThreads / 2; w > 0; w >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < w) part[threadIdx.x] = join(part[threadIdx.x], part[threadIdx.x + w]);
    }
    if (threadIdx.x == 0) {
        const float rstd = 1.f / sqrtf(part[0].m2 / part[0].count + p.epsilon);
        const int64_t at = n * p.groups + blockIdx.x;
        L.sums[2 * at] = part[0].mean;
        L.sums[2 * at + 1] = rstd;
        if (p.mean) p.mean[at] = part[0].mean;
        if (p.rstd) p.rstd[at] = rstd;
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) forward_apply_kernel(const NormLaunch L)
{
    const NtGroupNorm &p = L.p;
    const int64_t texels = (int64_t)p.height * p.width, count = texels * p.channels, n = blockIdx.y;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads) {
        const int64_t t = i / p.channels;
        const int c = (int)(i % p.channels);
        const float *stat = L.sums + 2 * (n * p.groups + c / L.per);
        const float h = (to_f32(static_cast<const T *>(p.x.data)[offset(p.x, n, t, p.width) + c]) - stat[0]) * stat[1];
        const float z = (p.gamma ? p.gamma[c] : 1.f) * h + (p.beta ? p.beta[c] : 0.f);
        static_cast<T *>(p.y.data)[offset(p.y, n, t, p.width) + c] = from_f32<T>(activate(z, p.activation));
    }
}

template <class T>
__device__ __forceinline__ void backward_terms(const NormLaunch &L, int64_t n, int64_t t, int c, float &e, float &h)
{
    const NtGroupNorm &p = L.p;
    const int64_t at = n * p.groups + c / L.per;
    h = (to_f32(static_cast<const T *>(p.x.data)[offset(p.x, n, t, p.width) + c]) - p.mean[at]) * p.rstd[at];
    const float z = (p.gamma ? p.gamma[c] : 1.f) * h + (p.beta ? p.beta[c] : 0.f);
    e = to_f32(static_cast<const T *>(p.dy.data)[offset(p.dy, n, t, p.width) + c]) * activation_slope(z, p.activation);
}

template <class T>
__global__ void __launch_bounds__(kThreads) backward_sums_kernel(const NormLaunch L)
{
    const NtGroupNorm &p = L.p;
    __shared__ float2 part[kThreads];
    const int64_t texels = (int64_t)p.height * p.width, n = blockIdx.y;
    const int64_t lo = texels * blockIdx.x / kSplit, hi = texels * (blockIdx.x + 1) / kSplit;
    const int rows = p.channels < kThreads ? kThreads / p.channels : 1;
    for (int c0 = 0; c0 < p.channels; c0 += kThreads) {
        const int width = min(kThreads, p.channels - c0), c = c0 + threadIdx.x % width, row = threadIdx.x / width;
        float2 s = make_float2(0.f, 0.f);
        if (row < rows)
            for (int64_t t = lo + row; t < hi; t += rows) {
                float e, h;
                backward_terms<T>(L, n, t, c, e, h);
                s.x += e;
                s.y += e * h;
            }
        part[threadIdx.x] = s;
        __syncthreads();
        if (row == 0) {
            for (int r = 1; r < rows; ++r) s.x += part[r * width + threadIdx.x].x, s.y += part[r * width + threadIdx.x].y;
            reinterpret_cast<float2 *>(L.partials)[(n * kSplit + blockIdx.x) * p.channels + c] = s;
        }
        __syncthreads();
    }
}

// grid (group, image): s1, s2 of a group
__global__ void backward_join_kernel(const NormLaunch L)
{
    const NtGroupNorm &p = L.p;
    __shared__ float2 part[kThreads];
    const int64_t n = blockIdx.y;
    float2 s = make_float2(0.f, 0.f);
    for (int i = threadIdx.x; i < kSplit * L.per; i += kThreads) {
        const int c = blockIdx.x * L.per + i % L.per;
        const float g = p.gamma ? p.gamma[c] : 1.f;
        const float2 v = reinterpret_cast<const float2 *>(L.partials)[(n * kSplit + i / L.per) * p.channels + c];
        s.x += g * v.x;
        s.y += g * v.y;
    }
    part[threadIdx.x] = s;
    for (int w = kThreads / 2; w > 0; w >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < w)
            part[threadIdx.x].x += part[threadIdx.x + w].x, part[threadIdx.x].y += part[threadIdx.x + w].y;
    }
    if (threadIdx.x == 0) reinterpret_cast<float2 *>(L.sums)[n * p.groups + blockIdx.x] = part[0];
}

// grid (channel): dgamma, dbeta
__global__ void backward_params_kernel(const NormLaunch L)
{
    const NtGroupNorm &p = L.p;
    __shared__ float2 part[kThreads];
    float2 s = make_float2(0.f, 0.f);
    for (int64_t i = threadIdx.x; i < (int64_t)p.images * kSplit; i += kThreads) {
        const float2 v = reinterpret_cast<const float2 *>(L.partials)[i * p.channels + blockIdx.x];
        s.x += v.x;
        s.y += v.y;
    }
    part[threadIdx.x] = s;
    for (int w = kThreads / 2; w > 0; w >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < w)
            part[threadIdx.x].x += part[threadIdx.x + w].x, part[threadIdx.x].y += part[threadIdx.x + w].y;
    }
    if (threadIdx.x == 0) {
        if (p.dbeta) p.dbeta[blockIdx.x] = part[0].x;
        if (p.dgamma) p.dgamma[blockIdx.x] = part[0].y;
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) backward_apply_kernel(const NormLaunch L)
{
    const NtGroupNorm &p = L.p;
    const int64_t texels = (int64_t)p.height * p.width, count = texels * p.channels, n = blockIdx.y;
    const float inv = 1.f / ((float)texels * (float)L.per);
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += (int64_t)gridDim.x * kThreads) {
        const int64_t t = i / p.channels;
        const int c = (int)(i % p.channels);
        float e, h;
        backward_terms<T>(L, n, t, c, e, h);
        const int64_t at = n * p.groups + c / L.per;
        const float2 s = reinterpret_cast<const float2 *>(L.sums)[at];
        const float dx = p.rstd[at] * ((p.gamma ? p.gamma[c] : 1.f) * e - (s.x + h * s.y) * inv);
        static_cast<T *>(p.dx.data)[offset(p.dx, n, t, p.width) + c] = from_f32<T>(dx);
    }
}

size_t partial_floats(const NtGroupNorm *p) { return (size_t)p->images * kSplit * p->channels * 2; }

template <class T>
cudaError_t launch(const NormLaunch &L, bool backward, cudaStream_t st)
{
    const NtGroupNorm &p = L.p;
    const dim3 split(kSplit, p.images), group(p.groups, p.images);
    const int64_t count = (int64_t)p.height * p.width * p.channels;
    const dim3 apply((unsigned)std::min<int64_t>((count + kThreads - 1) / kThreads, 8 * sm_count()), p.images);
    if (!backward) {
        forward_stats_kernel<T><<<split, kThreads, 0, st>>>(L);
        forward_join_kernel<<<group, kThreads, 0, st>>>(L);
        forward_apply_kernel<T><<<apply, kThreads, 0, st>>>(L);
    } else {
        backward_sums_kernel<T><<<split, kThreads, 0, st>>>(L);
        backward_join_kernel<<<group, kThreads, 0, st>>>(L);
        backward_apply_kernel<T><<<apply, kThreads, 0, st>>>(L);
        if (p.dgamma || p.dbeta) {
            backward_params_kernel<<<p.channels, kThreads, 0, st>>>(L);
            count_launch();
        }
    }
    for (int i = 0; i < 3; ++i) count_launch();
    return cudaGetLastError();
}

nt_status check_map(const NtFeatureMap &f, const char *name, const NtGroupNorm *p, int size, bool written)
{
    NT_LAYER_REQUIRE(f.data && is_aligned(f.data, size), "%s must be a non-null device pointer aligned to its element", name);
    NT_LAYER_REQUIRE(f.image_stride >= 0 && f.row_stride >= 0 && f.texel_stride >= 0, "%s: strides must be non-negative", name);
    if (written) {
        // each axis steps over everything inside it
        int64_t inner = p->channels;
        NT_LAYER_REQUIRE(p->width == 1 || f.texel_stride >= inner, "%s: texels overlap", name);
        if (p->width > 1) inner += (p->width - 1) * f.texel_stride;
        NT_LAYER_REQUIRE(p->height == 1 || f.row_stride >= inner, "%s: rows overlap", name);
        if (p->height > 1) inner += (p->height - 1) * f.row_stride;
        NT_LAYER_REQUIRE(p->images <= 1 || f.image_stride >= inner, "%s: images overlap", name);
    }
    return NT_OK;
}

// Sizes and enumerations, without the pointers.
nt_status check_shape(const NtGroupNorm *p)
{
    NT_LAYER_REQUIRE(p, "params is null");
    NT_LAYER_REQUIRE(p->images >= 0 && p->images <= 65535, "images must be in [0, 65535] (got %d)", p->images);
    NT_LAYER_REQUIRE(p->height >= 1 && p->width >= 1 && (int64_t)p->height * p->width < (int64_t)1 << 31,
                     "image size %d x %d must be positive and below 2^31 texels", p->width, p->height);
    NT_LAYER_REQUIRE(p->channels >= 1 && p->channels <= NT_GROUP_NORM_MAX_CHANNELS, "channels must be in [1, %d] (got %d)",
                     NT_GROUP_NORM_MAX_CHANNELS, p->channels);
    NT_LAYER_REQUIRE(p->groups >= 1 && p->channels % p->groups == 0, "channels (%d) must be a multiple of groups (%d)",
                     p->channels, p->groups);
    NT_LAYER_REQUIRE(layer_dtype_size(p->dtype), "dtype must be NT_DTYPE_F16, NT_DTYPE_BF16 or NT_DTYPE_F32 (got %d)", p->dtype);
    NT_LAYER_REQUIRE(p->activation >= NT_ACT_NONE && p->activation <= NT_ACT_GELU, "unknown activation %d", p->activation);
    NT_LAYER_REQUIRE(p->epsilon > 0.f, "epsilon must be positive");
    return NT_OK;
}

size_t workspace_bytes(const NtGroupNorm *p, bool)
{
    return p->images ? (partial_floats(p) + (size_t)p->images * p->groups * 2) * sizeof(float) : 0;
}

nt_status run(const NtGroupNorm *p, bool backward, nt_stream_t stream)
{
    nt_status st = check_shape(p);
    if (st != NT_OK) return st;
    const int size = layer_dtype_size(p->dtype);
    const cudaStream_t s = (cudaStream_t)stream;
    NT_LAYER_REQUIRE(is_aligned(p->gamma, 4) && is_aligned(p->beta, 4) && is_aligned(p->mean, 4) && is_aligned(p->rstd, 4) &&
                         is_aligned(p->dgamma, 4) && is_aligned(p->dbeta, 4),
                     "gamma, beta, mean, rstd, dgamma and dbeta must be 4-byte aligned device pointers");
    if (p->images == 0) {
        if (backward)
            for (float *g : {p->dgamma, p->dbeta})
                if (g) {
                    const cudaError_t e = cudaMemsetAsync(g, 0, sizeof(float) * p->channels, s);
                    if (e != cudaSuccess) return set_error(NT_ERR_CUDA, "group norm: %s", cudaGetErrorString(e));
                }
        return NT_OK;
    }
    if ((st = check_map(p->x, "x", p, size, false)) != NT_OK) return st;
    if (backward) {
        if ((st = check_map(p->dy, "dy", p, size, false)) != NT_OK) return st;
        if ((st = check_map(p->dx, "dx", p, size, true)) != NT_OK) return st;
        NT_LAYER_REQUIRE(p->mean && p->rstd, "mean and rstd of the forward call are required");
    } else if ((st = check_map(p->y, "y", p, size, true)) != NT_OK) {
        return st;
    }
    const size_t need = workspace_bytes(p, backward);
    NT_LAYER_REQUIRE(need == 0 || (p->workspace && is_aligned(p->workspace, 16) && p->workspace_bytes >= (int64_t)need),
                     "workspace must be 16-byte aligned and hold %zu bytes (got %lld)", need, (long long)p->workspace_bytes);
    NormLaunch L;
    L.p = *p;
    L.per = p->channels / p->groups;
    L.partials = static_cast<float *>(p->workspace);
    L.sums = L.partials + partial_floats(p);
    const cudaError_t e = p->dtype == NT_DTYPE_F16    ? launch<__half>(L, backward, s)
                          : p->dtype == NT_DTYPE_BF16 ? launch<__nv_bfloat16>(L, backward, s)
                                                      : launch<float>(L, backward, s);
    return e == cudaSuccess ? NT_OK : set_error(NT_ERR_CUDA, "group norm: %s", cudaGetErrorString(e));
}

}  // namespace norm
}  // namespace nt

using namespace nt;

extern "C" {

size_t nt_group_norm_workspace_bytes(const NtGroupNorm *p, int32_t backward)
{
    return p && norm::check_shape(p) == NT_OK ? norm::workspace_bytes(p, backward != 0) : 0;
}

nt_status nt_group_norm_forward(const NtGroupNorm *p, nt_stream_t stream) { return norm::run(p, false, stream); }

nt_status nt_group_norm_backward(const NtGroupNorm *p, nt_stream_t stream) { return norm::run(p, true, stream); }

}  // extern "C"
