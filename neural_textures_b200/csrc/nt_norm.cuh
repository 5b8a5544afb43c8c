// nt_norm.cuh -- the group-norm kernel, forward and backward (nt_group_norm_forward,
// nt_group_norm_backward); nt_norm_forward.cu and nt_norm_backward.cu instantiate it, nt_norm.cu
// checks arguments and plans the launch.
//
// One launch makes two passes over a map, with a barrier between them:
//   1. sums.  `splits` thread blocks share an image; a thread keeps one vector of V channels and
//      strides over texels.  Forward: count, mean and centred squares, each thread about its own
//      first value and joined pairwise after that, so that a common offset costs no digits.
//      Backward: per channel sums of e = dy act'(z) and e h.
//   2. the result, from the image's joined sums.
// What the first pass read is kept in shared memory as far as it goes (the oldest part), and the
// second pass starts with the texels read last, which are still in L2.
// Blocks of an image meet in a cluster (up to 8), where they read each other's sums from shared memory, or,
// for large maps, at a barrier of the whole cooperative grid, with the sums in the workspace.
// All sums are joined in a fixed order.
#pragma once

#include "nt_layer_common.cuh"

namespace nt {
namespace norm {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr uint32_t kSpinLimit = 1u << 24;

struct NormLaunch {
    NtGroupNorm p;
    int32_t per;        // channels of a group
    int32_t splits;     // thread blocks of an image
    int32_t cluster;    // 1: they form a cluster; 0: the grid meets at *barrier
    int32_t flat;       // texels of every map are evenly spaced
    int32_t texels, vectors;  // vectors of V channels in a texel
    int32_t tx, ty;     // threads along channels and texels
    int32_t keep;       // vectors of a thread (of x, and of dy) that stay in shared memory
    int32_t scratch;    // bytes of shared memory in front of them
    float inv_count;    // 1 / values of a group
    float2 *groups_part;    // [image][group][split]
    float2 *channels_part;  // [channel][image * split], backward
    unsigned int *barrier;
};

// V consecutive channels.
template <class T, int V>
struct alignas(V * sizeof(T) > 16 ? 16 : V * sizeof(T)) Vec {
    T v[V];
};

// Streaming: read once (its second reading comes from shared memory).
template <class T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T *p, bool stream)
{
    Vec<T, V> r;
    constexpr int bytes = V * sizeof(T);
    if constexpr (bytes == 16) *reinterpret_cast<uint4 *>(&r) = stream ? __ldcs(reinterpret_cast<const uint4 *>(p)) : *reinterpret_cast<const uint4 *>(p);
    else if constexpr (bytes == 8) *reinterpret_cast<uint2 *>(&r) = stream ? __ldcs(reinterpret_cast<const uint2 *>(p)) : *reinterpret_cast<const uint2 *>(p);
    else if constexpr (bytes == 4) *reinterpret_cast<uint32_t *>(&r) = stream ? __ldcs(reinterpret_cast<const uint32_t *>(p)) : *reinterpret_cast<const uint32_t *>(p);
    else *reinterpret_cast<uint16_t *>(&r) = stream ? __ldcs(reinterpret_cast<const uint16_t *>(p)) : *reinterpret_cast<const uint16_t *>(p);
    return r;
}

template <class T, int V>
__device__ __forceinline__ void store_vec(T *p, const Vec<T, V> &r)
{
    constexpr int bytes = V * sizeof(T);
    if constexpr (bytes == 16) __stcs(reinterpret_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(&r));
    else if constexpr (bytes == 8) __stcs(reinterpret_cast<uint2 *>(p), *reinterpret_cast<const uint2 *>(&r));
    else if constexpr (bytes == 4) __stcs(reinterpret_cast<uint32_t *>(p), *reinterpret_cast<const uint32_t *>(&r));
    else __stcs(reinterpret_cast<uint16_t *>(p), *reinterpret_cast<const uint16_t *>(&r));
}

template <int V>
__device__ __forceinline__ void activate_all(float (&z)[V], int act)
{
    switch (act) {
    case NT_ACT_RELU:
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = activate(z[i], NT_ACT_RELU);
        break;
    case NT_ACT_SILU:
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = activate(z[i], NT_ACT_SILU);
        break;
    case NT_ACT_GELU:
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = activate(z[i], NT_ACT_GELU);
        break;
    default: break;
    }
}

// e = dy act'(z)
template <int V>
__device__ __forceinline__ void times_slope(float (&e)[V], const float (&z)[V], int act)
{
    switch (act) {
    case NT_ACT_RELU:
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] *= activation_slope(z[i], NT_ACT_RELU);
        break;
    case NT_ACT_SILU:
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] *= activation_slope(z[i], NT_ACT_SILU);
        break;
    case NT_ACT_GELU:
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] *= activation_slope(z[i], NT_ACT_GELU);
        break;
    default: break;
    }
}

// Count, mean and sum of squares about the mean.
struct Stats {
    float count, mean, m2;
};

__device__ __forceinline__ Stats join(const Stats &a, const Stats &b)
{
    if (b.count == 0.f) return a;
    if (a.count == 0.f) return b;
    const float n = a.count + b.count, d = b.mean - a.mean, w = __fdividef(b.count, n);
    return {n, fmaf(d, w, a.mean), a.m2 + b.m2 + d * d * a.count * w};
}

__device__ __forceinline__ Stats warp_join(Stats s)
{
#pragma unroll
    for (int w = 16; w > 0; w >>= 1)
        s = join(s, {__shfl_down_sync(0xffffffffu, s.count, w), __shfl_down_sync(0xffffffffu, s.mean, w),
                     __shfl_down_sync(0xffffffffu, s.m2, w)});
    return s;
}

__device__ __forceinline__ float2 warp_sum(float2 s)
{
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) {
        s.x += __shfl_down_sync(0xffffffffu, s.x, w);
        s.y += __shfl_down_sync(0xffffffffu, s.y, w);
    }
    return s;
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

__device__ __forceinline__ float2 peer_f2(const float2 *mine, uint32_t rank)
{
    uint32_t remote;
    float2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(remote) : "memory");
    return v;
}

// All blocks of a cooperative launch; *counter is zero before it.
__device__ __forceinline__ void grid_sync(unsigned int *counter, unsigned int *status)
{
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(counter, 1u);
        uint32_t seen = 0;
        for (uint32_t i = 0; i < kSpinLimit; ++i) {
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
            if (seen >= gridDim.x) break;
        }
        if (seen < gridDim.x) atomicOr(status, 1u);
    }
    __syncthreads();
}

// dgamma, dbeta of one channel from the blocks' sums: a warp.
__device__ __forceinline__ void join_channel(const NormLaunch &L, int c)
{
    const int lane = threadIdx.x & 31, parts = L.p.images * L.splits;
    float2 s = make_float2(0.f, 0.f);
    for (int i = lane; i < parts; i += 32) {
        const float2 v = __ldcg(L.channels_part + (int64_t)c * parts + i);
        s.x += v.x;
        s.y += v.y;
    }
    s = warp_sum(s);
    if (lane == 0) {
        if (L.p.dbeta) L.p.dbeta[c] = s.x;
        if (L.p.dgamma) L.p.dgamma[c] = s.y;
    }
}

// WHOLE: a vector lies in one group.
template <class T, int V, bool WHOLE, bool BACKWARD>
__global__ void __launch_bounds__(kThreads, WHOLE ? 2 : 1) norm_kernel(const __grid_constant__ NormLaunch L, unsigned int *status)
{
    constexpr int U = BACKWARD ? 2 : 4;  // texels in flight
    using Vec = norm::Vec<T, V>;
    extern __shared__ __align__(16) uint8_t smem[];
    const NtGroupNorm &p = L.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t n = blockIdx.x / L.splits;
    const int split = blockIdx.x % L.splits;
    const int lo = (int)((int64_t)L.texels * split / L.splits), hi = (int)((int64_t)L.texels * (split + 1) / L.splits);
    const int row = tid / L.tx, col = tid % L.tx;
    const int mine = row < L.ty && lo + row < hi ? (hi - lo - row + L.ty - 1) / L.ty : 0;  // texels of this thread
    // shared memory: group results [groups], group partials [groups], scratch, kept vectors
    float2 *stat = reinterpret_cast<float2 *>(smem), *part = stat + p.groups, *scratch = part + p.groups;
    Vec *kept = reinterpret_cast<Vec *>(smem + L.scratch);

    const T *x = static_cast<const T *>(p.x.data) + n * p.x.image_stride;
    const T *dy = BACKWARD ? static_cast<const T *>(p.dy.data) + n * p.dy.image_stride : nullptr;
    const NtFeatureMap &out_map = BACKWARD ? p.dx : p.y;
    T *out = static_cast<T *>(out_map.data) + n * out_map.image_stride;
    auto texel = [&](const NtFeatureMap &f, int i) -> int64_t {
        const int t = lo + row + i * L.ty;
        if (L.flat) return t * f.texel_stride;
        const int y = t / p.width;
        return y * f.row_stride + (t - y * p.width) * f.texel_stride;
    };

    // ---- pass 1 ----
    int slot0 = 0;
    for (int v0 = 0; v0 < L.vectors; v0 += L.tx) {
        const int vec = v0 + col, c = vec * V;
        const int count = vec < L.vectors ? mine : 0;
        float s1[V] = {}, s2[V] = {};
        if constexpr (!BACKWARD) {
            float pivot[V] = {};
            for (int i = 0; i < count; i += U) {
                Vec a[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i + u < count) a[u] = load_vec<T, V>(x + texel(p.x, i + u) + c, slot0 + i + u < L.keep);
                if (i == 0)
#pragma unroll
                    for (int j = 0; j < V; ++j) pivot[j] = to_f32(a[0].v[j]);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i + u >= count) break;
                    if (slot0 + i + u < L.keep) kept[(slot0 + i + u) * kThreads + tid] = a[u];
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float d = to_f32(a[u].v[j]) - pivot[j];
                        s1[j] += d;
                        s2[j] = fmaf(d, d, s2[j]);
                    }
                }
            }
            if (vec < L.vectors && row < L.ty) {
                const float inv = count ? __fdividef(1.f, (float)count) : 0.f;
                Stats all = {0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const Stats one = {(float)count, fmaf(s1[j], inv, pivot[j]), fmaxf(s2[j] - s1[j] * s1[j] * inv, 0.f)};
                    if (WHOLE) all = join(all, one);
                    else scratch[row * p.channels + c + j] = make_float2(one.mean, one.m2);
                }
                if (WHOLE) scratch[row * L.vectors + vec] = make_float2(all.mean, all.m2);
            }
        } else {
            float mean[V], rstd[V], gamma[V], beta[V];
            if (vec < L.vectors)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int64_t g = n * p.groups + (c + (WHOLE ? 0 : j)) / L.per;
                    mean[j] = WHOLE && j ? mean[0] : __ldg(p.mean + g);
                    rstd[j] = WHOLE && j ? rstd[0] : __ldg(p.rstd + g);
                    gamma[j] = p.gamma ? __ldg(p.gamma + c + j) : 1.f;
                    beta[j] = p.beta ? __ldg(p.beta + c + j) : 0.f;
                }
            for (int i = 0; i < count; i += U) {
                Vec a[U], b[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i + u < count) {
                        a[u] = load_vec<T, V>(x + texel(p.x, i + u) + c, slot0 + i + u < L.keep);
                        b[u] = load_vec<T, V>(dy + texel(p.dy, i + u) + c, slot0 + i + u < L.keep);
                    }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i + u >= count) break;
                    if (slot0 + i + u < L.keep) {
                        kept[(2 * (slot0 + i + u)) * kThreads + tid] = a[u];
                        kept[(2 * (slot0 + i + u) + 1) * kThreads + tid] = b[u];
                    }
                    float e[V], h[V], z[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        h[j] = (to_f32(a[u].v[j]) - mean[j]) * rstd[j];
                        z[j] = fmaf(gamma[j], h[j], beta[j]);
                        e[j] = to_f32(b[u].v[j]);
                    }
                    times_slope<V>(e, z, p.activation);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        s1[j] += e[j];
                        s2[j] = fmaf(e[j], h[j], s2[j]);
                    }
                }
            }
            if (vec < L.vectors && row < L.ty)
#pragma unroll
                for (int j = 0; j < V; ++j) scratch[row * p.channels + c + j] = make_float2(s1[j], s2[j]);
        }
        slot0 += (hi - lo + L.ty - 1) / L.ty;
    }
    __syncthreads();

    // ---- the block's sums, per group (and per channel) ----
    float2 *const shared_out = L.cluster ? part : nullptr;
    const int parts = p.images * L.splits;
    if constexpr (!BACKWARD) {
        const int step = WHOLE ? V : 1, entries = L.per / step, width = p.channels / step;
        for (int g = warp; g < p.groups; g += kWarps) {
            Stats s = {0.f, 0.f, 0.f};
            for (int e = lane; e < L.ty * entries; e += 32) {
                const int r = e / entries;
                const float2 v = scratch[r * width + g * entries + e - r * entries];
                const int texels = lo + r < hi ? (hi - lo - r + L.ty - 1) / L.ty : 0;
                s = join(s, {(float)texels * step, v.x, v.y});
            }
            s = warp_join(s);
            if (lane == 0) {
                if (shared_out) shared_out[g] = make_float2(s.mean, s.m2);
                else L.groups_part[(n * p.groups + g) * L.splits + split] = make_float2(s.mean, s.m2);
            }
        }
    } else {
        // the rows of each channel, folded in halves
        for (int rows = L.ty; rows > 1; rows = (rows + 1) >> 1) {
            const int half = (rows + 1) >> 1;
            for (int i = tid; i < (rows - half) * p.channels; i += kThreads) {
                const float2 v = scratch[half * p.channels + i];
                scratch[i].x += v.x;
                scratch[i].y += v.y;
            }
            __syncthreads();
        }
        if (p.dgamma || p.dbeta)
            for (int c = tid; c < p.channels; c += kThreads) L.channels_part[(int64_t)c * parts + blockIdx.x] = scratch[c];
        for (int g = warp; g < p.groups; g += kWarps) {
            float2 s = make_float2(0.f, 0.f);
            for (int e = lane; e < L.per; e += 32) {
                const int c = g * L.per + e;
                const float w = p.gamma ? __ldg(p.gamma + c) : 1.f;
                s.x = fmaf(w, scratch[c].x, s.x);
                s.y = fmaf(w, scratch[c].y, s.y);
            }
            s = warp_sum(s);
            if (lane == 0) {
                if (shared_out) shared_out[g] = s;
                else L.groups_part[(n * p.groups + g) * L.splits + split] = s;
            }
        }
    }
    if (!L.cluster) grid_sync(L.barrier, status);
    else if (L.splits > 1) cluster_sync();
    else __syncthreads();

    // ---- the image's sums ----
    for (int g = warp; g < p.groups; g += kWarps) {
        Stats s = {0.f, 0.f, 0.f};
        float2 sum = make_float2(0.f, 0.f);
        for (int i = lane; i < L.splits; i += 32) {
            const float2 v = L.cluster ? (L.splits > 1 ? peer_f2(part + g, i) : part[g])
                                       : __ldcg(L.groups_part + (n * p.groups + g) * L.splits + i);
            if (BACKWARD) {
                sum.x += v.x;
                sum.y += v.y;
            } else {
                const int64_t texels = (int64_t)L.texels * (i + 1) / L.splits - (int64_t)L.texels * i / L.splits;
                s = join(s, {(float)texels * L.per, v.x, v.y});
            }
        }
        if (BACKWARD) {
            sum = warp_sum(sum);
            if (lane == 0) stat[g] = sum;
        } else {
            s = warp_join(s);
            if (lane == 0) {
                const float rstd = 1.f / sqrtf(s.m2 * L.inv_count + p.epsilon);
                stat[g] = make_float2(s.mean, rstd);
                if (split == 0) {
                    if (p.mean) p.mean[n * p.groups + g] = s.mean;
                    if (p.rstd) p.rstd[n * p.groups + g] = rstd;
                }
            }
        }
    }
    if (L.cluster && L.splits > 1) cluster_sync();  // a block's sums stay until its peers have read them
    else __syncthreads();
    if (BACKWARD && !L.cluster && (p.dgamma || p.dbeta))
        for (int64_t c = (int64_t)warp * gridDim.x + blockIdx.x; c < p.channels; c += (int64_t)kWarps * gridDim.x) join_channel(L, (int)c);

    // ---- pass 2, the texels read last first ----
    for (int v0 = (L.vectors - 1) / L.tx * L.tx; v0 >= 0; v0 -= L.tx) {
        slot0 -= (hi - lo + L.ty - 1) / L.ty;
        const int vec = v0 + col, c = vec * V;
        if (vec >= L.vectors) continue;
        float mean[V], scale[V], gamma[V], beta[V], k1[V], k2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int g = (c + (WHOLE ? 0 : j)) / L.per;
            gamma[j] = p.gamma ? __ldg(p.gamma + c + j) : 1.f;
            beta[j] = p.beta ? __ldg(p.beta + c + j) : 0.f;
            if constexpr (!BACKWARD) {
                mean[j] = stat[g].x;
                scale[j] = stat[g].y * gamma[j];
            } else {
                mean[j] = WHOLE && j ? mean[0] : __ldg(p.mean + n * p.groups + g);
                scale[j] = WHOLE && j ? scale[0] : __ldg(p.rstd + n * p.groups + g);
                k1[j] = stat[g].x * L.inv_count;
                k2[j] = stat[g].y * L.inv_count;
            }
        }
        for (int i = mine - 1; i >= 0; i -= U) {
            Vec a[U], b[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = i - u, slot = slot0 + k;
                if (k < 0) continue;
                const bool near = slot < L.keep;
                if constexpr (!BACKWARD) {
                    a[u] = near ? kept[slot * kThreads + tid] : load_vec<T, V>(x + texel(p.x, k) + c, true);
                } else {
                    a[u] = near ? kept[2 * slot * kThreads + tid] : load_vec<T, V>(x + texel(p.x, k) + c, true);
                    b[u] = near ? kept[(2 * slot + 1) * kThreads + tid] : load_vec<T, V>(dy + texel(p.dy, k) + c, true);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = i - u;
                if (k < 0) continue;
                Vec r;
                float z[V];
                if constexpr (!BACKWARD) {
#pragma unroll
                    for (int j = 0; j < V; ++j) z[j] = fmaf(to_f32(a[u].v[j]) - mean[j], scale[j], beta[j]);
                    activate_all<V>(z, p.activation);
#pragma unroll
                    for (int j = 0; j < V; ++j) r.v[j] = from_f32<T>(z[j]);
                } else {
                    float e[V], h[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        h[j] = (to_f32(a[u].v[j]) - mean[j]) * scale[j];
                        z[j] = fmaf(gamma[j], h[j], beta[j]);
                        e[j] = to_f32(b[u].v[j]);
                    }
                    times_slope<V>(e, z, p.activation);
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        r.v[j] = from_f32<T>(scale[j] * (fmaf(gamma[j], e[j], -k1[j]) - h[j] * k2[j]));
                }
                store_vec<T, V>(out + texel(out_map, k) + c, r);
            }
        }
    }
}

using NormKernel = void (*)(NormLaunch, unsigned int *);

template <class T, int V, bool BACKWARD>
NormKernel pick_whole(bool whole)
{
    if constexpr (V == 1) return norm_kernel<T, 1, true, BACKWARD>;
    else return whole ? (NormKernel)norm_kernel<T, V, true, BACKWARD> : (NormKernel)norm_kernel<T, V, false, BACKWARD>;
}

template <class T, bool BACKWARD>
NormKernel pick_width(int v, bool whole)
{
    if constexpr (sizeof(T) == 2)
        if (v == 8) return pick_whole<T, 8, BACKWARD>(whole);
    return v == 4 ? pick_whole<T, 4, BACKWARD>(whole) : v == 2 ? pick_whole<T, 2, BACKWARD>(whole) : pick_whole<T, 1, BACKWARD>(true);
}

template <bool BACKWARD>
NormKernel pick_kernel(int32_t dtype, int v, bool whole)
{
    return dtype == NT_DTYPE_F16    ? pick_width<__half, BACKWARD>(v, whole)
           : dtype == NT_DTYPE_BF16 ? pick_width<__nv_bfloat16, BACKWARD>(v, whole)
                                    : pick_width<float, BACKWARD>(v, whole);
}

NormKernel forward_kernel(int32_t dtype, int v, bool whole);
NormKernel backward_kernel(int32_t dtype, int v, bool whole);

}  // namespace norm
}  // namespace nt
