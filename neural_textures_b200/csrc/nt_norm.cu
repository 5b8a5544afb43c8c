// nt_norm.cu -- channels-last group normalisation with an activation: argument checks and launch
// plan of nt_group_norm_forward and nt_group_norm_backward (the kernel is in nt_norm.cuh).
#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

#include "nt_norm.cuh"

namespace nt {
namespace norm {

constexpr int kJoinWarps = 8;

__global__ void __launch_bounds__(32 * kJoinWarps) join_channels_kernel(const NormLaunch L)
{
    after_previous();
    const int c = blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
    if (c < L.p.channels) join_channel(L, c);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Thread blocks of an image.  A function of the sizes alone, so that the caller's workspace does not depend on
// addresses.
struct Plan {
    bool cluster;  // one launch
    int splits;    // blocks of an image, in the launch that makes the sums
    int applies;   // and in the one that makes the result
    int per_sm;    // blocks that share an SM's shared memory: one where the sums of a texel need the room
};

// A cluster costs about 1 us over a single block; two launches let every SM compute, but take the host 3 us more.  A
// turn of a block (a vector for each of its threads, both passes) takes about 0.35 us forward and 0.6 us backward.
// So an image is split until a block has four turns, and takes two launches where the largest cluster would
// leave it more than kTurns.  On the device, fp16, forward: 64 x 64 x 64 (4 turns) 7.4 us in a cluster of 16 and 6.8 us in two
// launches, 96 x 96 x 64 (9 turns) 9.5 and 6.9 us; backward: 64 x 64 x 64 (5.3 turns) 10.8 and 9.3 us.
constexpr int kForwardTurns = 8, kBackwardTurns = 4;
constexpr int kApplyTurns = 16;  // of a block of the second launch: enough of them that fast SMs take more

// Channels of a vector: up to 16 bytes of them, and up to 4 where vectors cross groups, whose per-channel values take
// the registers of a second block on the SM otherwise (3x83x138x48 fp16 of 8 groups: 14.2 us in vectors of 8, 9.4 in 4).
int vector_width(const NtGroupNorm *p)
{
    int v = 16 / layer_dtype_size(p->dtype);
    while (p->channels % v) v /= 2;
    return v == 8 && p->channels / p->groups % 8 ? 4 : v;
}

Plan plan(const NtGroupNorm *p, bool backward)
{
    const int sms = sm_count(), threads = backward ? kBackwardThreads : kForwardThreads, v = vector_width(p);
    const int per_sm = p->channels <= 2048 ? 2 : 1;
    const int64_t texels = (int64_t)p->height * p->width, turns = ceil_div(texels * (p->channels / v), threads);
    const int64_t most = std::min<int64_t>(texels, kMaxSplits);
    const int largest = (int64_t)p->images * kMaxCluster <= sms * 7 / 8 ? kMaxCluster : 8;  // of 16: one in most of the GPCs
    int64_t splits = 1;
    while (splits < largest && splits * 2 <= most && turns > 4 * splits && splits * p->images <= sms) splits *= 2;
    const int64_t resident = (int64_t)per_sm * sms / p->images;
    if (turns <= (backward ? kBackwardTurns : kForwardTurns) * splits || resident <= splits)
        return {true, (int)splits, (int)splits, splits * p->images <= sms ? 1 : per_sm};
    splits = std::min({ceil_div(turns, 4), resident, most});
    return {false, (int)splits, (int)std::min(std::max(splits, ceil_div(turns, kApplyTurns)), texels), per_sm};
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

// Workspace: group partials, channel partials.
struct Layout {
    size_t channels_at, total;
};

Layout layout(const NtGroupNorm *p, const Plan &pl, bool backward)
{
    Layout l;
    l.channels_at = pl.cluster ? 0 : align16((size_t)p->images * p->groups * pl.splits * sizeof(float2));
    l.total = l.channels_at + (backward ? (size_t)p->images * pl.splits * p->channels * sizeof(float2) : 0);
    return l;
}

// Whether vectors of v channels are aligned in a map.
bool vectors_aligned(const NtFeatureMap &f, int v, int size)
{
    return is_aligned(f.data, v * size) && f.image_stride % v == 0 && f.row_stride % v == 0 && f.texel_stride % v == 0;
}

// Whether a map's texels are evenly spaced, `ty` of them by less than 2^31 bytes.
bool flat(const NtFeatureMap &f, const NtGroupNorm *p, int size)
{
    return (p->height == 1 || f.row_stride == p->width * f.texel_stride) && f.texel_stride < ((int64_t)1 << 31) / (512 * size);
}

// Once per kernel and device.
cudaError_t allow_large_clusters(const void *kernel)
{
    static std::mutex mu;
    static std::set<std::pair<const void *, int>> done;
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> lock(mu);
    if (done.count({kernel, dev})) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) done.insert({kernel, dev});
    return e;
}

cudaError_t launch(const NtGroupNorm *p, bool backward, cudaStream_t st)
{
    const int size = layer_dtype_size(p->dtype);
    const Plan pl = plan(p, backward);
    const Layout at = layout(p, pl, backward);
    char *ws = static_cast<char *>(p->workspace);
    NormLaunch L = {};
    L.p = *p;
    const int threads = backward ? kBackwardThreads : kForwardThreads, ring = backward ? kBackwardRing : kForwardRing;
    L.per = p->channels / p->groups;
    L.parts = pl.splits;
    const bool even = flat(p->x, p, size) && flat(backward ? p->dy : p->y, p, size) && flat(backward ? p->dx : p->y, p, size);
    L.texels = p->height * p->width;
    L.part_share = L.texels / L.parts;
    L.part_extra = L.texels % L.parts;
    L.inv_count = 1.f / ((float)L.texels * (float)L.per);
    L.groups_part = reinterpret_cast<float2 *>(ws);
    L.channels_part = reinterpret_cast<float2 *>(ws + at.channels_at);
    const size_t most = 227 * 1024 / pl.per_sm - 1024;
    size_t smem = 0;
    // vectors that are not aligned are put together from their elements, unless half of one is aligned
    int v = vector_width(p);
    auto all_aligned = [&](int w) {
        return vectors_aligned(p->x, w, size) && vectors_aligned(backward ? p->dy : p->y, w, size) &&
               vectors_aligned(backward ? p->dx : p->y, w, size);
    };
    if (v * size == 16 && !all_aligned(v) && all_aligned(v / 2)) v /= 2;
    bool whole = true;
    for (;; v /= 2) {  // narrower vectors where the sums of very many groups leave no room for the ring
        whole = L.per % v == 0;
        L.vectors = p->channels / v;
        // threads along a texel's vectors: all of them, or the number of turns that leaves the fewest threads idle
        double used = 0;
        for (int turns = (int)ceil_div(L.vectors, threads), last = turns + 3; turns <= last; ++turns) {
            const int tx = (int)ceil_div(L.vectors, turns), ty = threads / tx;
            const double share = (double)L.vectors * ty / ((double)turns * threads);
            if (share > used + 0.05) used = share, L.tx = tx, L.ty = ty;
        }
        const size_t entries = (size_t)L.ty * (backward || !whole ? p->channels : L.vectors);
        L.scratch = (int32_t)align16((2 * (size_t)p->groups + entries) * sizeof(float2));
        const size_t slot = (size_t)threads * v * size * (backward ? 2 : 1);
        const int64_t room = (int64_t)((most - L.scratch) / slot);
        const int64_t slots = pl.cluster ? ceil_div(ceil_div(L.texels, pl.splits), L.ty) * ceil_div(L.vectors, L.tx) : ring + 1;
        L.keep = !pl.cluster ? 0 : (int32_t)(slots <= room ? slots : std::max<int64_t>(room - ring, 0));
        smem = L.scratch + (pl.cluster && slots <= room ? slots : L.keep + ring) * slot;
        if (smem <= most || v == 1) break;
    }
    L.aligned = (vectors_aligned(p->x, v, size) ? kXAligned : 0) | (!backward || vectors_aligned(p->dy, v, size) ? kDyAligned : 0) |
                (vectors_aligned(backward ? p->dx : p->y, v, size) ? kOutAligned : 0);
    const bool regular = even && L.aligned == (kXAligned | kDyAligned | kOutAligned);
    L.by_tx = (uint32_t)ceil_div(1 << 18, L.tx);
    const int units = whole ? L.per / v : L.per;
    L.by_group = units == 1 ? 0 : (uint32_t)ceil_div((int64_t)1 << 32, units);

    // launches `kernel` with `splits` blocks an image
    auto run = [&](NormKernel kernel, int splits, int cluster) {
        L.splits = splits;
        L.share = L.texels / splits;
        L.extra = L.texels % splits;
        L.turns = L.share / L.ty;
        L.left = L.share % L.ty;
        cudaError_t e = set_smem_limit(reinterpret_cast<const void *>(kernel), 227 * 1024 - 1024);
        if (e == cudaSuccess && cluster > 8) e = allow_large_clusters(reinterpret_cast<const void *>(kernel));
        return e == cudaSuccess ? launch_next(kernel, dim3((unsigned)splits, (unsigned)p->images), threads, smem, st, (unsigned)cluster, L) : e;
    };
    cudaError_t e;
    if (pl.cluster) {
        e = run((backward ? backward_kernel : forward_kernel)(p->dtype, v, whole, regular), pl.splits, pl.splits);
        if (e == cudaSuccess && backward && p->images > 1 && (p->dgamma || p->dbeta))
            e = launch_next(join_channels_kernel, dim3((unsigned)ceil_div(p->channels, kJoinWarps)), 32 * kJoinWarps, 0, st, 1, L);
        return e;
    }
    e = run((backward ? backward_sums_kernel : forward_sums_kernel)(p->dtype, v, whole, regular), pl.splits, 1);
    return e == cudaSuccess ? run((backward ? backward_apply_kernel : forward_apply_kernel)(p->dtype, v, whole, regular), pl.applies, 1) : e;
}

nt_status check_map(const NtFeatureMap &f, const char *name, const NtGroupNorm *p, int size, bool written)
{
    NT_LAYER_REQUIRE(f.data && is_aligned(f.data, size), "%s must be a non-null device pointer aligned to its element", name);
    NT_LAYER_REQUIRE(f.image_stride >= 0 && f.row_stride >= 0 && f.texel_stride >= 0, "%s: strides must be non-negative", name);
    if (written) {
        // each axis steps over everything inside it, whatever their order
        struct Axis {
            int64_t stride;
            int32_t size;
            const char *what;
        } axes[3] = {{f.texel_stride, p->width, "texels"}, {f.row_stride, p->height, "rows"}, {f.image_stride, p->images, "images"}};
        std::stable_sort(axes, axes + 3, [](const Axis &a, const Axis &b) { return a.stride < b.stride; });
        int64_t inner = p->channels;
        for (const Axis &a : axes) {
            if (a.size <= 1) continue;
            NT_LAYER_REQUIRE(a.stride >= inner, "%s: %s overlap", name, a.what);
            inner += (a.size - 1) * a.stride;
        }
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

size_t workspace_bytes(const NtGroupNorm *p, bool backward)
{
    return p->images ? layout(p, plan(p, backward), backward).total : 0;
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
    NT_LAYER_REQUIRE(is_aligned(p->workspace, 16) && (need == 0 || (p->workspace && p->workspace_bytes >= (int64_t)need)),
                     "workspace must be 16-byte aligned and hold %zu bytes (got %lld)", need, (long long)p->workspace_bytes);
    const cudaError_t e = launch(p, backward, s);
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
