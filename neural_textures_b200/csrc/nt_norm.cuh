// nt_norm.cuh -- the group-norm kernel, forward and backward (nt_group_norm_forward,
// nt_group_norm_backward); nt_norm_{forward,backward}{,_sums,_apply}.cu instantiate it, nt_norm.cu
// checks arguments and plans the launches.
//
// Two passes over a map:
//   1. sums.  `splits` thread blocks share an image; a thread keeps one vector of V channels and
//      strides over texels.  Forward: count, mean and centred squares, each thread about the mean
//      of its first values and joined about common means after that, so that a common offset costs no digits.
//      Backward: per channel sums of e = dy act'(z) and e h.
//   2. the result, from the image's joined sums.
// An image that a cluster of up to 16 blocks gets through quickly takes one launch: the blocks read each
// other's sums from shared memory, and keep there what the first pass read as far as it goes.  Larger
// ones take a launch for each pass, with the blocks' sums in the workspace; the second is set up under the
// first, and starts with the texels read last, which are still in L2.  (One cooperative launch for both
// passes, the blocks meeting at a barrier of the grid with 24 MB kept on chip, was slower: SMs of
// different GPCs differ by half in bandwidth, and all waited for the slowest twice: 73 us against 68 us for
// 1024 x 1024 x 64 fp16, 17.6 against 9.8 us for 256 x 256 x 64.)
// A thread's vectors arrive by asynchronous copies in its own slots of shared memory, so that loads stay in
// flight while it computes and no barrier is needed: a ring of a few vectors, and in front of it what is kept.
// All sums are joined in a fixed order.
//
// Bound by HBM (2 to 3 readings of a map in all) and, in the second pass, by issue slots and the special-function unit.
// 1024 x 1024 x 64 fp16 with SiLU, one B200: 68.5 us forward (25 sums, 5.3 TB/s; 43 result), 117 us backward.
#pragma once

#include "nt_layer_common.cuh"

namespace nt {
namespace norm {

constexpr int kForwardThreads = 512;
// Vectors in flight for each thread, 64 and 72 KB on an SM; 8 and 6 of them for the sums changed nothing.
constexpr int kForwardRing = 4, kBackwardRing = 4;
constexpr int kBackwardThreads = 384;  // 84 registers a thread with two blocks on an SM: 64 spill
constexpr int kMaxCluster = 16;
constexpr int kMaxSplits = 320;  // thread blocks of an image

enum { kXAligned = 1, kDyAligned = 2, kOutAligned = 4 };  // NormLaunch.aligned

// Both passes in one launch by a cluster, or a launch for each.
enum Phase { kBoth, kSums, kApply };

struct NormLaunch {
    NtGroupNorm p;
    int32_t per;        // channels of a group
    int32_t splits;     // thread blocks of an image, in this launch
    int32_t parts, part_share, part_extra;  // blocks of an image that made the sums, and their texels
    int32_t aligned;    // maps whose vectors are aligned
    int32_t texels, vectors;  // vectors of V channels in a texel
    int32_t tx, ty;     // threads along channels and texels
    int32_t share, extra;   // texels of a block: share, the first `extra` blocks one more
    int32_t turns, left;    // share / ty and its remainder
    uint32_t by_tx;         // ceil(2^18 / tx): thread / tx without a division
    uint32_t by_group;      // ceil(2^32 / (units of a group)), 0 for one; a unit is a vector, or a channel where vectors cross groups
    int32_t keep;       // vectors of a thread (of x, and of dy) that stay in shared memory, in front of its ring
    int32_t scratch;    // bytes of shared memory in front of them
    float inv_count;    // 1 / values of a group
    float2 *groups_part;    // [image][group][part]
    float2 *channels_part;  // [channel][image * part], backward
};

// V consecutive channels.
template <class T, int V>
struct alignas(V * sizeof(T) > 16 ? 16 : V * sizeof(T)) Vec {
    T v[V];
};

// A vector from global to shared memory: asynchronous, but for 2-byte vectors.
template <class T, int V>
__device__ __forceinline__ void fetch(uint32_t to, const char *p, uint64_t policy)
{
    constexpr int bytes = V * sizeof(T);
    if constexpr (bytes == 16)
        asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to), "l"(p), "l"(policy) : "memory");
    else if constexpr (bytes >= 4)
        asm volatile("cp.async.ca.shared.global.L2::cache_hint [%0], [%1], %2, %3;" ::"r"(to), "l"(p), "n"(bytes), "l"(policy) : "memory");
    else
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(*reinterpret_cast<const uint16_t *>(p)) : "memory");
}

// The same of a vector that is aligned to its elements only.
template <class T, int V>
__device__ __forceinline__ void fetch_each(uint32_t to, const char *p, uint64_t policy)
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) fetch<T, 1>(to + 4 * i, p + 4 * i, policy);
    } else {
        uint16_t v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = reinterpret_cast<const uint16_t *>(p)[i];
#pragma unroll
        for (int i = 0; i < V; ++i) asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + 2 * i), "h"(v[i]) : "memory");
    }
}

template <class T, int V>
__device__ __forceinline__ Vec<T, V> read_slot(uint32_t at)
{
    Vec<T, V> r;
    constexpr int bytes = V * sizeof(T);
    if constexpr (bytes == 16) {
        uint4 &v = *reinterpret_cast<uint4 *>(&r);
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    } else if constexpr (bytes == 8) {
        uint2 &v = *reinterpret_cast<uint2 *>(&r);
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    } else if constexpr (bytes == 4) {
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(*reinterpret_cast<uint32_t *>(&r)) : "r"(at) : "memory");
    } else {
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(*reinterpret_cast<uint16_t *>(&r)) : "r"(at) : "memory");
    }
    return r;
}

// L2 policies: what is read once (again), and what the second pass will read.
__device__ __forceinline__ uint64_t policy_once()
{
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint64_t policy_again()
{
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
    return p;
}

__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <class T, int V>
__device__ __forceinline__ void store_vec(T *p, const Vec<T, V> &r)
{
    constexpr int bytes = V * sizeof(T);
    if constexpr (bytes == 16) __stcs(reinterpret_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(&r));
    else if constexpr (bytes == 8) __stcs(reinterpret_cast<uint2 *>(p), *reinterpret_cast<const uint2 *>(&r));
    else if constexpr (bytes == 4) __stcs(reinterpret_cast<uint32_t *>(p), *reinterpret_cast<const uint32_t *>(&r));
    else __stcs(reinterpret_cast<uint16_t *>(p), *reinterpret_cast<const uint16_t *>(&r));
}

// A vector's values in pairs, for packed fp32 arithmetic (of a single value, beside a zero).
template <class T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V> &a, float2 (&f)[(V + 1) / 2])
{
#pragma unroll
    for (int j = 0; j < (V + 1) / 2; ++j) {
        if constexpr (V == 1) f[j] = make_float2(to_f32(a.v[0]), 0.f);
        else if constexpr (sizeof(T) == 4) f[j] = make_float2(a.v[2 * j], a.v[2 * j + 1]);
        else f[j] = pair_f32(reinterpret_cast<const typename Pair<T>::type *>(&a)[j]);
    }
}

template <class T, int V>
__device__ __forceinline__ Vec<T, V> pack(const float2 (&f)[(V + 1) / 2])
{
    Vec<T, V> r;
#pragma unroll
    for (int j = 0; j < (V + 1) / 2; ++j) {
        if constexpr (V == 1) r.v[0] = from_f32<T>(f[0].x);
        else if constexpr (sizeof(T) == 4) r.v[2 * j] = f[j].x, r.v[2 * j + 1] = f[j].y;
        else reinterpret_cast<typename Pair<T>::type *>(&r)[j] = f32_pair<T>(f[j]);
    }
    return r;
}

__device__ __forceinline__ float warp_sum_all(float s)
{
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
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

__device__ __forceinline__ void prefetch(const void *p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

// dgamma, dbeta of one channel from the blocks' sums: a warp.
__device__ __forceinline__ void join_channel(const NormLaunch &L, int c)
{
    const int lane = threadIdx.x & 31, parts = L.p.images * L.parts;
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

// What a thread's passes share.
template <class T, int V, bool WHOLE, bool REGULAR, bool BACKWARD, Phase PHASE>
struct Threads {
    static constexpr int P = (V + 1) / 2;
    static constexpr int NT = BACKWARD ? kBackwardThreads : kForwardThreads;
    const NormLaunch &L;
    int64_t n;
    int lo, row, col, mine;  // first texel of the block; place of the thread; its texels
    const float2 *stat;
    float2 *scratch;
    uint32_t kept;  // shared-memory address of the thread's first slot

    // Texel i of this thread in a map, from channel c.
    struct Path {
        const Threads &t;
        const NtFeatureMap &f;
        char *at;
        int step;  // bytes
        __device__ __forceinline__ Path(const Threads &t, const NtFeatureMap &f, int c) : t(t), f(f)
        {
            at = static_cast<char *>(f.data) + (t.n * f.image_stride + c) * (int64_t)sizeof(T);
            if (REGULAR) at += (t.lo + t.row) * f.texel_stride * (int64_t)sizeof(T);
            step = (int)(t.L.ty * f.texel_stride * (int64_t)sizeof(T));
        }
        __device__ __forceinline__ char *operator()(int i) const
        {
            if (REGULAR) return at + (int64_t)i * step;
            const int k = t.lo + t.row + i * t.L.ty, y = k / t.L.p.width, x = k - y * t.L.p.width;
            return at + (y * f.row_stride + x * f.texel_stride) * (int64_t)sizeof(T);
        }
    };
    // Per-channel values of a parameter, in pairs.
    __device__ __forceinline__ void channels(const float *param, float other, int c, float2 (&v)[P]) const
    {
        if (param && V >= 4 && (reinterpret_cast<uintptr_t>(param) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < P; j += 2) {
                const float4 q = __ldg(reinterpret_cast<const float4 *>(param + c) + j / 2);
                v[j] = make_float2(q.x, q.y);
                if (j + 1 < P) v[j + 1] = make_float2(q.z, q.w);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < P; ++j)
            v[j] = make_float2(param ? __ldg(param + c + 2 * j) : other, V > 1 && param ? __ldg(param + c + 2 * j + 1) : other);
    }
    // Group of channel c + i (of the whole vector, when it lies in one).
    __device__ __forceinline__ int group(int c, int i) const
    {
        const uint32_t unit = WHOLE ? (uint32_t)c / V : (uint32_t)(c + (i >= V ? 0 : i));
        return (int)(L.by_group ? __umulhi(unit, L.by_group) : unit);
    }

    // The slots of this thread: kept vectors, then a ring of kDepth (a power of two).  In the backward pass a
    // slot holds x and, kNext bytes on, dy.
    static constexpr uint32_t kNext = NT * sizeof(Vec<T, V>), kSlot = kNext * (BACKWARD ? 2 : 1);
    static constexpr int kDepth = BACKWARD ? kBackwardRing : kForwardRing;
    struct Source {
        Path x, dy;
        __device__ __forceinline__ Source(const Threads &t, int c) : x(t, t.L.p.x, c), dy(t, t.L.p.dy, c) {}
        __device__ __forceinline__ void get(uint32_t slot, int i, uint64_t policy) const
        {
            one(slot, x(i), policy, kXAligned);
            if (BACKWARD) one(slot + kNext, dy(i), policy, kDyAligned);
        }
        __device__ __forceinline__ void one(uint32_t slot, const char *p, uint64_t policy, int bit) const
        {
            if (REGULAR || V == 1 || (x.t.L.aligned & bit)) fetch<T, V>(slot, p, policy);
            else fetch_each<T, V>(slot, p, policy);
        }
    };

    // use(slot, i) for texels 0 .. count - 1.  In front of texel `stop`, a multiple of 4, stop = pause(stop).  Afterwards the
    // last kDepth texels are still in the ring, texel i in slot (i - near) % kDepth.
    template <class Use, class Pause>
    __device__ __forceinline__ void each_forth(int c, int count, int near, int slot0, Use use, int stop, Pause pause) const
    {
        const uint32_t keep = kept + slot0 * kSlot, ring = kept + L.keep * kSlot;
        const Source src(*this, c);
        const uint64_t once = policy_once(), again = policy_again();
        for (int i = 0; i < near; ++i) src.get(keep + i * kSlot, i, once);
        fetch_commit();
#pragma unroll
        for (int u = 0; u < kDepth; ++u) {
            if (near + u < count) src.get(ring + u * kSlot, near + u, again);
            fetch_commit();
        }
        fetch_wait<kDepth>();
        int i = 0;
        while (i < near) {  // runs between two stops: looking for one at every texel cost 17% of 200 x 64 x 64 x 32 fp16
            const int end = min(near, stop);
#pragma unroll 2
            for (; i < end; ++i) use(keep + i * kSlot, i);
            if (i == stop && i < count) stop = pause(i);
        }
        while (i < count) {
            const int end = min(count, stop);
#pragma unroll 2
            for (; i < end; ++i) {
                const uint32_t slot = ring + ((i - near) & (kDepth - 1)) * kSlot;
                fetch_wait<kDepth - 1>();
                use(slot, i);
                if (i + kDepth < count) src.get(slot, i + kDepth, again);
                fetch_commit();
            }
            if (i == stop && i < count) stop = pause(i);
        }
    }

    // The same from count - 1 down to 0, the ring as each_forth left it for this column, or `fresh`.
    template <class Use>
    __device__ __forceinline__ void each_back(int c, int count, int near, int slot0, bool fresh, Use use) const
    {
        const uint32_t keep = kept + slot0 * kSlot, ring = kept + L.keep * kSlot;
        if (count > near) {
            const Source src(*this, c);
            const uint64_t once = policy_once();
#pragma unroll
            for (int u = 0; u < kDepth; ++u) {
                const int i = count - 1 - u;
                if (fresh && i >= near) src.get(ring + ((i - near) & (kDepth - 1)) * kSlot, i, once);
                fetch_commit();
            }
#pragma unroll 2
            for (int i = count - 1; i >= near; --i) {
                const uint32_t slot = ring + ((i - near) & (kDepth - 1)) * kSlot;
                fetch_wait<kDepth - 1>();
                use(slot, i);
                if (i - kDepth >= near) src.get(slot, i - kDepth, once);
                fetch_commit();
            }
        }
#pragma unroll 2
        for (int i = near - 1; i >= 0; --i) use(keep + i * kSlot, i);
    }

    // use(slot, i) for every texel, nothing kept: texels 0 .. count - 1 (with stops as above), or backwards.  The ring's slots
    // are constants of an unrolled loop.
    template <bool REVERSED, class Use, class Pause>
    __device__ __forceinline__ void each_fresh(int c, int count, Use use, int stop, Pause pause) const
    {
        const Source src(*this, c);
        const uint64_t policy = REVERSED ? policy_once() : policy_again();
        auto texel = [&](int i) { return REVERSED ? count - 1 - i : i; };
#pragma unroll
        for (int u = 0; u < kDepth; ++u) {
            if (u < count) src.get(kept + u * kSlot, texel(u), policy);
            fetch_commit();
        }
        int i = 0;
        static_assert(kDepth == 4, "a stop is a multiple of it");
        for (; i + 2 * kDepth <= count; i += kDepth) {
            if (i == stop) stop = pause(i);
#pragma unroll
            for (int u = 0; u < kDepth; ++u) {
                fetch_wait<kDepth - 1>();
                use(kept + u * kSlot, texel(i + u));
                src.get(kept + u * kSlot, texel(i + u + kDepth), policy);
                fetch_commit();
            }
        }
#pragma unroll 1
        for (; i < count; i += kDepth) {
            if (i == stop) stop = pause(i);
#pragma unroll
            for (int u = 0; u < kDepth; ++u) {
                fetch_wait<kDepth - 1>();
                if (i + u < count) use(kept + u * kSlot, texel(i + u));
                if (i + u + kDepth < count) src.get(kept + u * kSlot, texel(i + u + kDepth), policy);
                fetch_commit();
            }
        }
    }

    template <class Use, class Pause>
    __device__ __forceinline__ void every_forth(int c, int count, int near, int slot0, Use use, int stop, Pause pause) const
    {
        if constexpr (PHASE == kSums) each_fresh<false>(c, count, use, stop, pause);
        else each_forth(c, count, near, slot0, use, stop, pause);
    }
    template <class Use>
    __device__ __forceinline__ void every_back(int c, int count, int near, int slot0, bool fresh, Use use) const
    {
        if constexpr (PHASE == kApply) each_fresh<true>(c, count, use, -1, [](int) { return -1; });
        else each_back(c, count, near, slot0, fresh, use);
    }

    // ---- pass 1 ----
    __device__ __forceinline__ void forward_sums(int c, int count, int near, int slot0) const
    {
        // Sums about a pivot: the first value, then, after 4, 16, 64, 128, 192, ... texels, the mean of all so far, so that
        // the squares are at most 4 times the centred ones.  About the first value alone, a black border in front of 8,000
        // texels cost 2.5% of the variance.  The squares of 64 texels are added to those before them at once: long
        // chains of equal terms round one way.
        float2 pivot[P] = {}, s1[P] = {}, s2[P] = {}, before[P] = {};  // pivot: its negative; before: squares
        bool begun = false;
        auto add = [&](uint32_t slot, int) {
            float2 f[P];
            unpack<T, V>(read_slot<T, V>(slot), f);
            if (!begun) {
                begun = true;
#pragma unroll
                for (int j = 0; j < P; ++j) pivot[j] = make_float2(-f[j].x, -f[j].y);
            }
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const float2 d = __fadd2_rn(f[j], pivot[j]);
                s1[j] = __fadd2_rn(s1[j], d);
                s2[j] = __ffma2_rn(d, d, s2[j]);
            }
        };
        every_forth(c, count, near, slot0, add, 4, [&](int i) {
            const float inv = __fdividef(-1.f, (float)i);
#pragma unroll
            for (int j = 0; j < P; ++j) {  // up by -d: s1' = s1 + i d, s2' = s2 + 2 d s1 + i d^2 = s2 + d (s1 + s1')
                const float2 to = __ffma2_rn(s1[j], f2(inv), pivot[j]), d = __ffma2_rn(pivot[j], f2(-1.f), to);
                const float2 t = __ffma2_rn(d, f2((float)i), s1[j]);
                before[j] = __fadd2_rn(before[j], __ffma2_rn(d, __fadd2_rn(s1[j], t), s2[j]));
                s2[j] = f2(0.f);
                s1[j] = t;
                pivot[j] = to;
            }
            return i < 64 ? 4 * i : i + 64;
        });
        // (mean, centred squares) of each channel, or of the vector about the mean of its channels
        const float inv = count > 0 ? __fdividef(1.f, (float)count) : 0.f;
        float mean[V], m2[V], shift = 0.f, sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float a = j & 1 ? s1[j / 2].y : s1[j / 2].x, b = j & 1 ? s2[j / 2].y + before[j / 2].y : s2[j / 2].x + before[j / 2].x;
            mean[j] = fmaf(a, inv, -(j & 1 ? pivot[j / 2].y : pivot[j / 2].x));
            const float squares = fmaf(-a * inv, a, b);
            m2[j] = squares < 0.f ? 0.f : squares == squares ? squares : b;  // b: infinite where the squares overflow
            if (!WHOLE) scratch[row * L.p.channels + c + j] = make_float2(mean[j], m2[j]);
            shift += mean[j] - mean[0];
        }
        if (!WHOLE) return;
        const float all = fmaf(shift, 1.f / V, mean[0]);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += fmaf((float)count * (mean[j] - all), mean[j] - all, m2[j]);
        scratch[row * L.vectors + c / V] = make_float2(all, sum);
    }

    // Terms of the backward pass: h and e = dy act'(z).
    template <int ACT>
    __device__ __forceinline__ static void terms(float2 x, float2 dy, float2 shift, float2 rstd, float2 gamma, float2 beta, float2 &h,
                                                 float2 &e)
    {
        h = __fmul2_rn(__fadd2_rn(x, shift), rstd);
        e = ACT == NT_ACT_NONE ? dy : times_slope2<ACT>(dy, __ffma2_rn(gamma, h, beta));
    }

    __device__ __forceinline__ void statistics(int c, float2 (&shift)[P], float2 (&rstd)[P]) const
    {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            if (WHOLE && j) break;
            const int64_t g0 = n * L.p.groups + group(c, 2 * j), g1 = n * L.p.groups + group(c, 2 * j + 1);
            shift[j] = make_float2(-__ldg(L.p.mean + g0), -__ldg(L.p.mean + g1));
            rstd[j] = make_float2(__ldg(L.p.rstd + g0), __ldg(L.p.rstd + g1));
        }
    }

    template <int ACT>
    __device__ __forceinline__ void backward_sums(int c, int count, int near, int slot0) const
    {
        float2 s1[P] = {}, s2[P] = {}, shift[P], rstd[P], gamma[P], beta[P];
        // In chains of 256, added up in shared memory, as long chains of equal terms (a broadcast dy) round one way: 11,000
        // of them cost 10^-4.  Chains of 64 cost 1024 x 1024 x 64 fp16 another 0.5 us: the stores conflict in their banks.
        float2 *const sums = scratch + row * L.p.channels + c;
        auto put_sums = [&](bool add) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float2 s = j & 1 ? make_float2(s1[j / 2].y, s2[j / 2].y) : make_float2(s1[j / 2].x, s2[j / 2].x);
                if (add) s = __fadd2_rn(s, sums[j]);
                sums[j] = s;
            }
        };
        statistics(c, shift, rstd);
        channels(L.p.gamma, 1.f, c, gamma);
        channels(L.p.beta, 0.f, c, beta);
        every_forth(c, count, near, slot0, [&](uint32_t slot, int) {
            float2 fa[P], fb[P];
            unpack<T, V>(read_slot<T, V>(slot), fa);
            unpack<T, V>(read_slot<T, V>(slot + kNext), fb);
#pragma unroll
            for (int j = 0; j < P; ++j) {
                float2 h, e;
                terms<ACT>(fa[j], fb[j], shift[WHOLE ? 0 : j], rstd[WHOLE ? 0 : j], gamma[j], beta[j], h, e);
                s1[j] = __fadd2_rn(s1[j], e);
                s2[j] = __ffma2_rn(e, h, s2[j]);
            }
        }, 256, [&](int i) {
            put_sums(i > 256);
#pragma unroll
            for (int j = 0; j < P; ++j) s1[j] = s2[j] = f2(0.f);
            return i + 256;
        });
        put_sums(count > 256);
    }

    // ---- pass 2, the texels read last first ----
    __device__ __forceinline__ void put(char *at, const Vec<T, V> &v) const
    {
        T *p = reinterpret_cast<T *>(at);
        if (REGULAR || V == 1 || (L.aligned & kOutAligned)) {
            store_vec<T, V>(p, v);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) p[i] = v.v[i];
        }
    }

    template <int ACT>
    __device__ __forceinline__ void forward_apply(int c, int count, int near, int slot0, bool fresh) const
    {
        float2 shift[P], scale[P], beta[P];
        channels(L.p.gamma, 1.f, c, scale);
        channels(L.p.beta, 0.f, c, beta);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const float2 a = stat[group(c, 2 * j)], b = stat[group(c, 2 * j + 1)];
            shift[j] = make_float2(-a.x, -b.x);
            scale[j] = __fmul2_rn(scale[j], make_float2(a.y, b.y));
        }
        const Path out(*this, L.p.y, c);
        every_back(c, count, near, slot0, fresh, [&](uint32_t slot, int i) {
            float2 f[P];
            unpack<T, V>(read_slot<T, V>(slot), f);
#pragma unroll
            for (int j = 0; j < P; ++j)
                f[j] = activate2<ACT>(__ffma2_rn(__fadd2_rn(f[j], shift[WHOLE ? 0 : j]), scale[j], beta[j]));
            put(out(i), norm::pack<T, V>(f));
        });
    }

    template <int ACT>
    __device__ __forceinline__ void backward_apply(int c, int count, int near, int slot0, bool fresh) const
    {
        float2 shift[P], rstd[P], gamma[P], beta[P], k1[P], k2[P];
        statistics(c, shift, rstd);
        channels(L.p.gamma, 1.f, c, gamma);
        channels(L.p.beta, 0.f, c, beta);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            if (WHOLE && j) break;
            const float2 a = stat[group(c, 2 * j)], b = stat[group(c, 2 * j + 1)];
            k1[j] = make_float2(-a.x * L.inv_count, -b.x * L.inv_count);
            k2[j] = make_float2(-a.y * L.inv_count, -b.y * L.inv_count);
        }
        const Path out(*this, L.p.dx, c);
        every_back(c, count, near, slot0, fresh, [&](uint32_t slot, int i) {
            float2 fa[P], fb[P];
            unpack<T, V>(read_slot<T, V>(slot), fa);
            unpack<T, V>(read_slot<T, V>(slot + kNext), fb);
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const int s = WHOLE ? 0 : j;
                float2 h, e;
                terms<ACT>(fa[j], fb[j], shift[s], rstd[s], gamma[j], beta[j], h, e);
                fa[j] = __fmul2_rn(rstd[s], __ffma2_rn(gamma[j], e, __ffma2_rn(h, k2[s], k1[s])));
            }
            put(out(i), norm::pack<T, V>(fa));
        });
    }

    template <int ACT>
    __device__ __forceinline__ void first(int c, int count, int near, int slot0) const
    {
        if constexpr (BACKWARD) backward_sums<ACT>(c, count, near, slot0);
        else forward_sums(c, count, near, slot0);
    }
    template <int ACT>
    __device__ __forceinline__ void second(int c, int count, int near, int slot0, bool fresh) const
    {
        if constexpr (BACKWARD) backward_apply<ACT>(c, count, near, slot0, fresh);
        else forward_apply<ACT>(c, count, near, slot0, fresh);
    }
};

// WHOLE: a vector lies in one group.  REGULAR: the texels of every map are evenly spaced and its
// vectors aligned.
template <class T, int V, bool WHOLE, bool REGULAR, bool BACKWARD, Phase PHASE>
__global__ void __launch_bounds__(BACKWARD ? kBackwardThreads : kForwardThreads, 2)
    norm_kernel(const __grid_constant__ NormLaunch L)
{
    constexpr int NT = BACKWARD ? kBackwardThreads : kForwardThreads, kWarps = NT / 32;
    extern __shared__ __align__(16) uint8_t smem[];
    const NtGroupNorm &p = L.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t n = blockIdx.y;
    const int split = PHASE == kApply ? L.splits - 1 - blockIdx.x : blockIdx.x;  // the texels read last first
    const int share = L.share, extra = L.extra;
    const int lo = split * share + min(split, extra), hi = lo + share + (split < extra);
    // shared memory: group results [groups], group partials [groups], scratch, kept vectors
    float2 *stat = reinterpret_cast<float2 *>(smem), *part = stat + p.groups, *scratch = part + p.groups;
    const int row = (int)(tid * L.by_tx >> 18), col = tid - row * L.tx;
    int turn = L.turns, left = L.left + (split < extra);
    if (left == L.ty) ++turn, left = 0;
    const int mine = row < L.ty ? turn + (row < left) : 0;  // texels of this thread
    const int most = turn + (left > 0);                     // and of any
    const Threads<T, V, WHOLE, REGULAR, BACKWARD, PHASE> th = {L,    n,       lo, row, col, mine,
                                               stat, scratch,
                                               (uint32_t)__cvta_generic_to_shared(smem + L.scratch) + tid * (uint32_t)sizeof(Vec<T, V>)};
    after_previous();
    int slot0 = 0;
    for (int v0 = 0; PHASE != kApply && v0 < L.vectors; v0 += L.tx, slot0 += most) {
        const int vec = v0 + col;
        if (vec >= L.vectors || row >= L.ty) continue;
        const int near = min(max(L.keep - slot0, 0), mine);
        if (!BACKWARD && PHASE == kBoth) {  // the second pass wants them soon
            if (p.gamma) prefetch(p.gamma + vec * V);
            if (p.beta) prefetch(p.beta + vec * V);
        }
        switch (BACKWARD ? p.activation : NT_ACT_NONE) {
        case NT_ACT_RELU: th.template first<NT_ACT_RELU>(vec * V, mine, near, slot0); break;
        case NT_ACT_SILU: th.template first<NT_ACT_SILU>(vec * V, mine, near, slot0); break;
        case NT_ACT_GELU: th.template first<NT_ACT_GELU>(vec * V, mine, near, slot0); break;
        default: th.template first<NT_ACT_NONE>(vec * V, mine, near, slot0); break;
        }
    }
    __syncthreads();

    // ---- the block's sums, per group (and per channel) ----
    auto finish = [&](int g, float mean, float squares) {
        const float rstd = rsqrtf(fmaf(squares, L.inv_count, p.epsilon));
        stat[g] = make_float2(mean, rstd);
        if (split == 0) {
            if (p.mean) p.mean[n * p.groups + g] = mean;
            if (p.rstd) p.rstd[n * p.groups + g] = rstd;
        }
    };
    const int blocks = p.images * L.splits;
    if constexpr (PHASE != kApply) {
        if constexpr (!BACKWARD) {
            const int step = WHOLE ? V : 1, entries = L.per / step, width = p.channels / step;
            for (int g = warp; g < p.groups; g += kWarps) {
                // two passes over the group's entries: the mean, from differences to one of them; the squares about it
                const float2 *const of = scratch + g * entries;
                const float origin = of[0].x;
                float shift = 0.f, sum = 0.f;
                for (int e = lane; e < L.ty * entries; e += 32) {
                    const int r = entries == 1 ? e : e / entries;
                    shift = fmaf((float)(turn + (r < left)) * step, of[r * (width - entries) + e].x - origin, shift);
                }
                const float mean = origin + __fdividef(warp_sum_all(shift), (float)(hi - lo) * L.per);
                for (int e = lane; e < L.ty * entries; e += 32) {
                    const int r = entries == 1 ? e : e / entries;
                    const float2 v = of[r * (width - entries) + e];
                    sum += fmaf((float)(turn + (r < left)) * step * (v.x - mean), v.x - mean, v.y);
                }
                sum = warp_sum_all(sum);
                if (lane == 0) {
                    if (PHASE == kBoth && L.splits == 1) finish(g, mean, sum);
                    else if (PHASE == kBoth) part[g] = make_float2(mean, sum);
                    else L.groups_part[(n * p.groups + g) * L.splits + split] = make_float2(mean, sum);
                }
            }
        } else {
            // the rows of each channel, folded in halves
            for (int rows = L.ty; rows > 1; rows = (rows + 1) >> 1) {
                const int half = (rows + 1) >> 1;
                for (int i = tid; i < (rows - half) * p.channels; i += NT) {
                    const float2 v = scratch[half * p.channels + i];
                    scratch[i].x += v.x;
                    scratch[i].y += v.y;
                }
                __syncthreads();
            }
            if ((p.dgamma || p.dbeta) && (p.images > 1 || PHASE == kSums))
                for (int c = tid; c < p.channels; c += NT) L.channels_part[(int64_t)c * blocks + blockIdx.y * L.splits + blockIdx.x] = scratch[c];
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
                    if (PHASE == kBoth && L.splits == 1) stat[g] = s;
                    else if (PHASE == kBoth) part[g] = s;
                    else L.groups_part[(n * p.groups + g) * L.splits + split] = s;
                }
            }
        }
    }
    if constexpr (PHASE == kSums) return;
    if (PHASE == kBoth && L.splits > 1) cluster_sync();
    else if (PHASE == kBoth) __syncthreads();

    // ---- the image's sums ----
    const int parts = L.parts;
    for (int g = warp; g < p.groups && (PHASE == kApply || parts > 1); g += kWarps) {
        float2 v[kMaxSplits / 32];
#pragma unroll
        for (int k = 0; k < kMaxSplits / 32; ++k) {
            const int i = lane + 32 * k;
            v[k] = make_float2(0.f, 0.f);
            if (i < parts) v[k] = PHASE == kBoth ? peer_f2(part + g, i) : __ldcg(L.groups_part + (n * p.groups + g) * parts + i);
        }
        float a = 0.f, b = 0.f;
        if (BACKWARD) {
#pragma unroll
            for (int k = 0; k < kMaxSplits / 32; ++k) a += v[k].x, b += v[k].y;
            a = warp_sum_all(a);
            b = warp_sum_all(b);
            if (lane == 0) stat[g] = make_float2(a, b);
        } else {
            const float origin = __shfl_sync(0xffffffffu, v[0].x, 0);
#pragma unroll
            for (int k = 0; k < kMaxSplits / 32; ++k)
                if (lane + 32 * k < parts) a = fmaf((float)(L.part_share + (lane + 32 * k < L.part_extra)), v[k].x - origin, a);
            const float mean = origin + __fdividef(warp_sum_all(a), (float)L.texels);
#pragma unroll
            for (int k = 0; k < kMaxSplits / 32; ++k)
                if (lane + 32 * k < parts)
                    b += fmaf((float)(L.part_share + (lane + 32 * k < L.part_extra)) * L.per * (v[k].x - mean), v[k].x - mean, v[k].y);
            b = warp_sum_all(b);
            if (lane == 0) finish(g, mean, b);
        }
    }
    if (BACKWARD && PHASE == kBoth && p.images == 1 && (p.dgamma || p.dbeta))
        for (int c = split * NT + tid; c < p.channels; c += L.splits * NT) {
            float2 s = scratch[c];
            if (L.splits > 1) {
                s = make_float2(0.f, 0.f);
                for (int i = 0; i < L.splits; ++i) {
                    const float2 v = peer_f2(scratch + c, i);
                    s.x += v.x;
                    s.y += v.y;
                }
            }
            if (p.dbeta) p.dbeta[c] = s.x;
            if (p.dgamma) p.dgamma[c] = s.y;
        }
    if (PHASE == kBoth && L.splits > 1) cluster_sync();  // a block's sums stay until its peers have read them
    else if (PHASE == kApply) __syncthreads();
    if (BACKWARD && PHASE == kApply && (p.dgamma || p.dbeta))
        for (int c = warp * blocks + blockIdx.y * L.splits + blockIdx.x; c < p.channels; c += kWarps * blocks) join_channel(L, c);

    for (int v0 = (L.vectors - 1) / L.tx * L.tx; v0 >= 0; v0 -= L.tx) {
        if (PHASE == kBoth) slot0 -= most;
        const int vec = v0 + col;
        if (vec >= L.vectors || mine == 0) continue;
        const int near = min(max(L.keep - slot0, 0), mine);
        const bool fresh = PHASE == kApply || v0 + L.tx < L.vectors;  // else the ring holds the last columns of pass 1
        switch (p.activation) {
        case NT_ACT_RELU: th.template second<NT_ACT_RELU>(vec * V, mine, near, slot0, fresh); break;
        case NT_ACT_SILU: th.template second<NT_ACT_SILU>(vec * V, mine, near, slot0, fresh); break;
        case NT_ACT_GELU: th.template second<NT_ACT_GELU>(vec * V, mine, near, slot0, fresh); break;
        default: th.template second<NT_ACT_NONE>(vec * V, mine, near, slot0, fresh); break;
        }
    }
}

using NormKernel = void (*)(NormLaunch);

template <class T, int V, bool BACKWARD, Phase PHASE>
NormKernel pick_whole(bool whole, bool regular)
{
    if constexpr (V > 1 && V < 8)
        if (!whole) return regular ? norm_kernel<T, V, false, true, BACKWARD, PHASE> : norm_kernel<T, V, false, false, BACKWARD, PHASE>;
    return regular ? norm_kernel<T, V, true, true, BACKWARD, PHASE> : norm_kernel<T, V, true, false, BACKWARD, PHASE>;
}

template <class T, bool BACKWARD, Phase PHASE>
NormKernel pick_width(int v, bool whole, bool regular)
{
    if constexpr (sizeof(T) == 2)
        if (v == 8) return pick_whole<T, 8, BACKWARD, PHASE>(whole, regular);
    return v == 4   ? pick_whole<T, 4, BACKWARD, PHASE>(whole, regular)
           : v == 2 ? pick_whole<T, 2, BACKWARD, PHASE>(whole, regular)
                    : pick_whole<T, 1, BACKWARD, PHASE>(whole, regular);
}

template <bool BACKWARD, Phase PHASE>
NormKernel pick_kernel(int32_t dtype, int v, bool whole, bool regular)
{
    return dtype == NT_DTYPE_F16    ? pick_width<__half, BACKWARD, PHASE>(v, whole, regular)
           : dtype == NT_DTYPE_BF16 ? pick_width<__nv_bfloat16, BACKWARD, PHASE>(v, whole, regular)
                                    : pick_width<float, BACKWARD, PHASE>(v, whole, regular);
}

// One per file that instantiates kernels: [forward, backward] x [both passes, sums, result].
NormKernel forward_kernel(int32_t dtype, int v, bool whole, bool regular);
NormKernel forward_sums_kernel(int32_t dtype, int v, bool whole, bool regular);
NormKernel forward_apply_kernel(int32_t dtype, int v, bool whole, bool regular);
NormKernel backward_kernel(int32_t dtype, int v, bool whole, bool regular);
NormKernel backward_sums_kernel(int32_t dtype, int v, bool whole, bool regular);
NormKernel backward_apply_kernel(int32_t dtype, int v, bool whole, bool regular);

}  // namespace norm
}  // namespace nt
