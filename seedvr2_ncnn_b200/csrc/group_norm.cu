// Group norm with an activation, channels last, on sm_100a:
//   y[i][r][c] = act((x[i][r][c] - mean(i, g)) * rstd(i, g) * gamma[c] + beta[c]),
// g = c / (C / groups), statistics over the instance's rows and the group's
// channels, rstd = 1 / sqrt(var + eps) with the biased variance.
//
// HBM-bound at best: x read once, y written once.  Two forms:
//   * slab kernel (small x): a slab -- one instance, a slice of whole groups --
//     stays in the registers of one thread-block cluster from its only read to
//     its write; the CTAs push their groups' (count, mean, M2) into each
//     other's shared memory and meet at one cluster barrier.
//   * sums + apply kernels (large x): every SM streams whole rows; the first
//     leaves (mean, M2) per part of an instance's rows and group in the
//     caller's workspace, the second joins them and normalises, reading each
//     part last row first, so that what the first read last comes from L2.
//
// Statistics: each thread sums d = x - p and d^2 per channel in fp32 around its
// own first value p (no cancellation for channels far from zero), turns them
// into (mean, M2), and these are joined by
//   mean = sum n_k mean_k / n,  M2 = sum M2_k + n_k (mean_k - mean)^2,
// in a fixed order: results do not depend on the run.
#include <algorithm>
#include <type_traits>

#include "activation.cuh"
#include "s2_common.cuh"
#include "s2_internal.h"
#include "s2_objects.h"

namespace s2 {

namespace {

constexpr int kThreads = 256;
constexpr int kBlocks = 3; // CTAs a SM of the large kernels
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;

struct GroupNormArgs
{
    const void* x;
    void* out;
    const float* gamma;
    const float* beta;
    int64_t ldx, ldo;
    int rows;        // per instance
    int width;       // channels per group
    int slice;       // channels per slab or part (whole groups)
    int slices;      // per instance
    int groups;      // per slice
    int parts;       // runs of rows per instance: CTAs of a slab's cluster, or parts
    int slots;       // rows a CTA works on at once: kThreads / min(kThreads, slice / V)
    uint32_t by_cols; // thread / (slice / V) = umulhi(thread, by_cols) where that is below kThreads
    int part_rows, longer; // the first `longer` parts have part_rows + 1 rows, the others part_rows
    uint32_t by_width;     // c / width = umulhi(c, by_width) for width > 1 and c * width < 2^32
    int sub;         // channels of one group that lie in one thread's vector
    int red_bytes;   // of the sums kernel's reduction, before its ring
    float eps;
    int act;
    float2* partial; // [instances][slices * groups][parts] (mean, M2)
};

// V consecutive channels as they lie in memory.
template <typename T, int V>
struct Raw
{
    T v[V];
};
template <>
struct Raw<__nv_bfloat16, 8>
{
    uint4 q;
};
template <>
struct Raw<float, 4>
{
    uint4 q;
};
template <>
struct Raw<__nv_bfloat16, 4>
{
    uint2 q;
};

// As pairs; V = 1 leaves the second half of its pair zero.
template <int V>
constexpr int kPairs = (V + 1) / 2;

__device__ __forceinline__ float2 bf16_pair(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float2 (&f)[kPairs<V>])
{
    if constexpr (V == 8)
        f[0] = bf16_pair(r.q.x), f[1] = bf16_pair(r.q.y), f[2] = bf16_pair(r.q.z), f[3] = bf16_pair(r.q.w);
    else if constexpr (V == 4 && sizeof(T) == 2)
        f[0] = bf16_pair(r.q.x), f[1] = bf16_pair(r.q.y);
    else if constexpr (V == 4)
    {
        f[0] = make_float2(__uint_as_float(r.q.x), __uint_as_float(r.q.y));
        f[1] = make_float2(__uint_as_float(r.q.z), __uint_as_float(r.q.w));
    }
    else
        f[0] = make_float2(static_cast<float>(r.v[0]), 0.f);
}

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p)
{
    Raw<T, V> r;
    if constexpr (V > 1)
        r.q = __ldcs(reinterpret_cast<const decltype(r.q)*>(p));
    else
        r.v[0] = *p;
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_out(T* p, const float2 (&f)[kPairs<V>])
{
    if constexpr (V == 8 && sizeof(T) == 2)
        __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y),
                                                       pack_bf16x2(f[2].x, f[2].y), pack_bf16x2(f[3].x, f[3].y)));
    else if constexpr (V == 4 && sizeof(T) == 2)
        __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y)));
    else if constexpr (V > 1)
    {
#pragma unroll
        for (int j = 0; j < V / 4; j++)
            __stcs(reinterpret_cast<float4*>(p) + j, make_float4(f[2 * j].x, f[2 * j].y, f[2 * j + 1].x, f[2 * j + 1].y));
    }
    else if constexpr (sizeof(T) == 2)
        *p = __float2bfloat16_rn(f[0].x);
    else
        *p = f[0].x;
}

// max(v, 0), NaN kept
__device__ __forceinline__ float not_negative(float v)
{
    return v < 0.f ? 0.f : v;
}

// Joins (n, mean, M2) entries: `count` groups with slots x units entries each,
// get(group, slot, unit), done(group, joined).  A power of two of lanes works
// on a group, as many as it has entries at most, so that a warp joins several
// small groups at once; the lanes lie over a power of two of units, so no
// index needs a division.
template <class Get, class Done>
__device__ __forceinline__ void join_groups(int first, int count, int slots, int units, Get get, Done done)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int log_u = units > 16 ? 5 : (units > 1 ? 32 - __clz(units - 1) : 0);
    const int want = slots << log_u;
    const int log_l = want > 16 ? 5 : (want > 1 ? 32 - __clz(want - 1) : 0);
    const int in = lane & ((1 << log_l) - 1), seg = lane >> log_l, segs = 32 >> log_l;
    const int u0 = in & ((1 << log_u) - 1), s0 = in >> log_u, s_step = log_l > log_u ? 1 << (log_l - log_u) : 1;
    auto seg_add = [&](float v) {
        for (int m = 1 << log_l >> 1; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
        return v;
    };
    for (int base = first + warp * segs; base < first + count; base += kWarps * segs)
    {
        const int g = base + seg;
        const int live = g < first + count ? slots : 0;
        // around the first entry's mean, so that a mean far from zero loses nothing
        const float p = live > 0 ? get(g, 0, 0).y : 0.f;
        float n = 0.f, s = 0.f;
#pragma unroll 4
        for (int sl = s0; sl < live; sl += s_step)
            for (int u = u0; u < units; u += 1 << log_u)
            {
                const float3 t = get(g, sl, u);
                n += t.x;
                s += t.x * (t.y - p);
            }
        n = seg_add(n);
        s = seg_add(s);
        const float mean = p + (n > 0.f ? __fdividef(s, n) : 0.f);
        float m2 = 0.f;
        for (int sl = s0; sl < live; sl += s_step)
            for (int u = u0; u < units; u += 1 << log_u)
            {
                const float3 t = get(g, sl, u);
                const float d = t.y - mean;
                m2 += t.z + t.x * d * d;
            }
        m2 = seg_add(m2);
        if (in == 0 && live > 0) done(g, make_float3(n, mean, m2));
    }
}

// Two entries.
__device__ __forceinline__ float3 join2(float3 a, float3 b)
{
    const float n = a.x + b.x, mean = a.x > 0.f ? a.y + b.x * (b.y - a.y) / n : b.y;
    const float da = a.y - mean, db = b.y - mean;
    return make_float3(n, mean, a.z + a.x * da * da + (b.z + b.x * db * db));
}

// Sums around p of n values in each of V channels -> (mean, M2), `sub`
// consecutive channels of one group joined: V / sub entries of `red`.
template <int V, int SUB>
__device__ __forceinline__ void merge_channels(const float (&m)[V], const float (&q)[V], float n, float2* red, int pitch)
{
#pragma unroll
    for (int e = 0; e < V / SUB; e++)
    {
        float s = 0.f, m2 = 0.f;
#pragma unroll
        for (int j = 0; j < SUB; j++) s += m[e * SUB + j];
        const float mean = s * (1.f / SUB);
#pragma unroll
        for (int j = 0; j < SUB; j++)
        {
            const float d = m[e * SUB + j] - mean;
            m2 += q[e * SUB + j] + n * d * d;
        }
        red[e * pitch] = make_float2(mean, m2);
    }
}
template <int V>
__device__ __forceinline__ void leave_sums(const float2 (&neg)[kPairs<V>], const float2 (&s1)[kPairs<V>],
                                           const float2 (&s2)[kPairs<V>], int n, int sub, float2* red, int pitch)
{
    const float fn = (float)n, inv = __fdividef(1.f, fn);
    float m[V], q[V];
#pragma unroll
    for (int j = 0; j < V; j++)
    {
        const float a = j & 1 ? s1[j / 2].y : s1[j / 2].x, b = j & 1 ? s2[j / 2].y : s2[j / 2].x;
        const float mean = a * inv;
        m[j] = mean - (j & 1 ? neg[j / 2].y : neg[j / 2].x);
        q[j] = not_negative(b - a * mean);
    }
    if (V == 8 && sub == 8)
        merge_channels<V, V>(m, q, fn, red, pitch);
    else if (V >= 4 && sub == 4)
        merge_channels<V, V >= 4 ? 4 : 1>(m, q, fn, red, pitch);
    else if (V >= 4 && sub == 2)
        merge_channels<V, V >= 4 ? 2 : 1>(m, q, fn, red, pitch);
    else
        merge_channels<V, 1>(m, q, fn, red, pitch);
}

// Thread t of a CTA owns vector column t % cols and rows t / cols, + slots, ...
struct Lanes
{
    int cols, slots, slot, col;
    int rounds, more; // rows of a slot: rounds, and one more below `more`
    __device__ Lanes(const GroupNormArgs& a, int vpr, unsigned rows) : slots(a.slots)
    {
        cols = min(vpr, kThreads);
        slot = cols == 1 ? threadIdx.x : (cols == kThreads ? 0 : (int)__umulhi(threadIdx.x, a.by_cols));
        col = threadIdx.x - slot * cols;
        rounds = rows / (unsigned)slots;
        more = rows - rounds * slots;
    }
    __device__ int rows_of(int s) const { return rounds + (s < more ? 1 : 0); }
    __device__ int mine() const { return slot < slots ? rows_of(slot) : 0; }
    __device__ int live_slots() const { return rounds > 0 ? slots : more; }
    // Entries of the reduction lie unit after unit (a unit: `sub` channels), a
    // unit's slots side by side; the odd pitch keeps both ways of walking them
    // off one bank.
    __device__ int pitch() const { return slots | 1; }
};

template <int V>
struct Sums
{
    float2 neg[kPairs<V>], s1[kPairs<V>], s2[kPairs<V>];
    __device__ void start(const float2 (&p)[kPairs<V>])
    {
#pragma unroll
        for (int j = 0; j < kPairs<V>; j++)
        {
            neg[j] = make_float2(-p[j].x, -p[j].y);
            s1[j] = s2[j] = make_float2(0.f, 0.f);
        }
    }
    __device__ void add(const float2 (&f)[kPairs<V>])
    {
#pragma unroll
        for (int j = 0; j < kPairs<V>; j++)
        {
            const float2 d = __fadd2_rn(f[j], neg[j]);
            s1[j] = __fadd2_rn(s1[j], d);
            s2[j] = __ffma2_rn(d, d, s2[j]);
        }
    }
};

// (x - mean) * mul + add per channel of a thread's vector, then the activation
template <typename TO, int V>
struct Scale
{
    float2 neg[kPairs<V>], mul[kPairs<V>], off[kPairs<V>];
    __device__ void load(const GroupNormArgs& a, const float2* stat, int c0, int col)
    {
#pragma unroll
        for (int j = 0; j < kPairs<V>; j++)
        {
            float v[3][2] = {};
#pragma unroll
            for (int h = 0; h < (V == 1 ? 1 : 2); h++)
            {
                const int c = col * V + 2 * j + h;
                const float2 t = stat[a.width > 1 ? (int)__umulhi(c, a.by_width) : c]; // (mean, rstd)
                v[0][h] = -t.x;
                v[1][h] = t.y * (a.gamma ? __ldg(a.gamma + c0 + c) : 1.f);
                v[2][h] = a.beta ? __ldg(a.beta + c0 + c) : 0.f;
            }
            neg[j] = make_float2(v[0][0], v[0][1]);
            mul[j] = make_float2(v[1][0], v[1][1]);
            off[j] = make_float2(v[2][0], v[2][1]);
        }
    }
    template <int ACT>
    __device__ void row(float2 (&f)[kPairs<V>], TO* out) const
    {
#pragma unroll
        for (int j = 0; j < kPairs<V>; j++) f[j] = __ffma2_rn(__fadd2_rn(f[j], neg[j]), mul[j], off[j]);
        activate<ACT>(f);
        store_out<TO, V>(out, f);
    }
};

template <class F>
__device__ __forceinline__ void with_act(int act, F f)
{
    switch (act)
    {
    case S2_ACT_SILU: f(std::integral_constant<int, S2_ACT_SILU>()); break;
    case S2_ACT_GELU_TANH: f(std::integral_constant<int, S2_ACT_GELU_TANH>()); break;
    case S2_ACT_GELU_ERF: f(std::integral_constant<int, S2_ACT_GELU_ERF>()); break;
    default: f(std::integral_constant<int, S2_ACT_NONE>()); break;
    }
}

__device__ __forceinline__ int part_first(const GroupNormArgs& a, int p)
{
    return p * a.part_rows + min(p, a.longer);
}
__device__ __forceinline__ int part_rows(const GroupNormArgs& a, int p)
{
    return a.part_rows + (p < a.longer ? 1 : 0);
}

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, float4 v)
{
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}

// ---------------------------------------------------------------- slab kernel
// Rows of its vector column per thread, in registers: two forms of the kernel,
// since the longer one's code costs a small x 0.3 us.
constexpr int kHeld = 8, kHeldMost = 12;
constexpr int kSlabBlocks = 2; // CTAs a SM: the registers must leave room for them (see kSlabCtas)

// Bytes of the reduction: units x pitch.
size_t red_bytes(int cols, int per_thread)
{
    return ((size_t)cols * per_thread * ((kThreads / cols) | 1) * 8 + 15) / 16 * 16;
}

size_t slab_smem(int cluster, int groups, int cols, int per_thread)
{
    return (size_t)(cluster + 1) * groups * 16 + (size_t)groups * 8 + red_bytes(cols, per_thread);
}

template <typename TI, typename TO, int V, int K>
__global__ void __launch_bounds__(kThreads, kSlabBlocks) group_norm_slab_kernel(const GroupNormArgs a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    const int G = a.groups, P = a.parts;
    float4* table = reinterpret_cast<float4*>(smem); // [P][G], written by the cluster
    float4* own = table + P * G;
    float2* stat = reinterpret_cast<float2*>(own + G);
    float2* red = stat + G;
    const int per_thread = V / a.sub;

    const int rank = P > 1 ? (int)cluster_ctarank() : 0;
    const int64_t slab = blockIdx.x / P;
    const int64_t inst = slab / a.slices;
    const int c0 = (int)(slab - inst * a.slices) * a.slice;
    const int r0 = part_first(a, rank);
    const Lanes t(a, a.slice / V, part_rows(a, rank));
    const int mine = t.mine();
    const int64_t row0 = inst * a.rows + r0 + t.slot;
    const TI* x = static_cast<const TI*>(a.x) + row0 * a.ldx + c0 + t.col * V;
    const int64_t x_step = t.slots * a.ldx;

    Raw<TI, V> raw[K];
#pragma unroll
    for (int k = 0; k < K; k++)
        if (k < mine) raw[k] = load_raw<TI, V>(x + k * x_step);
    if (mine > 0)
    {
        Sums<V> s;
        float2 f[kPairs<V>];
        unpack<TI, V>(raw[0], f);
        s.start(f);
#pragma unroll
        for (int k = 1; k < K; k++)
            if (k < mine)
            {
                unpack<TI, V>(raw[k], f);
                s.add(f);
            }
        leave_sums<V>(s.neg, s.s1, s.s2, mine, a.sub, red + t.col * per_thread * t.pitch() + t.slot, t.pitch());
    }
    // every CTA of the cluster runs before any writes into its shared memory
    if (P > 1)
        cluster_sync();
    else
        __syncthreads();
    const int units = a.width / a.sub; // entries of a group per row
    auto finish = [&](int g, float3 j) { stat[g] = make_float2(j.y, 1.f / sqrtf(not_negative(j.z / j.x) + a.eps)); };
    join_groups(
        0, G, t.live_slots(), units,
        [&](int g, int sl, int u) {
            const float2 v = red[(g * units + u) * t.pitch() + sl];
            return make_float3((float)(t.rows_of(sl) * a.sub), v.x, v.y);
        },
        [&](int g, float3 j) {
            if (P == 1)
                finish(g, j);
            else
                own[g] = make_float4(j.x, j.y, j.z, 0.f);
        });
    if (P > 1)
    {
        __syncthreads();
        for (int e = threadIdx.x; e < G * P; e += kThreads)
        {
            const int to = e / G, g = e - to * G;
            // a CTA without rows leaves no entries of its own
            st_cluster_v4(mapa_shared(table + rank * G + g, to),
                          t.live_slots() > 0 ? own[g] : make_float4(0.f, 0.f, 0.f, 0.f));
        }
        cluster_sync();
        join_groups(
            0, G, P, 1,
            [&](int g, int k, int) {
                const float4 v = table[k * G + g];
                return make_float3(v.x, v.y, v.z);
            },
            finish);
    }
    __syncthreads();
    if (mine == 0) return;
    Scale<TO, V> sc;
    sc.load(a, stat, c0, t.col);
    TO* out = static_cast<TO*>(a.out) + row0 * a.ldo + c0 + t.col * V;
    const int64_t o_step = t.slots * a.ldo;
    with_act(a.act, [&](auto act) {
#pragma unroll
        for (int k = 0; k < K; k++)
            if (k < mine)
            {
                float2 f[kPairs<V>];
                unpack<TI, V>(raw[k], f);
                sc.template row<decltype(act)::value>(f, out + k * o_step);
            }
    });
}

// ---------------------------------------------------------------- sums, apply
// Rows of a thread's column in order.  Vectors come through a private
// ring of shared memory filled by cp.async: no barrier, since a thread reads
// only what it fetched itself, and no registers held while a row is on its
// way.  kStep rows are fetched and handed out together, kDepth - 1 such steps
// ahead; begin() sends for the first of them.  Single channels are loaded
// plainly, kPlain rows at once.
constexpr int kDepth = 4;
constexpr int kStep = 4;
constexpr int kPlain = 8;
template <typename TI, int V>
constexpr size_t kRingBytes = V > 1 ? (size_t)kThreads * sizeof(Raw<TI, V>) * kStep * kDepth : 0;

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src)
{
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

template <typename TI, int V>
struct RowStream
{
    static constexpr int VB = sizeof(Raw<TI, V>), ROW = kThreads * VB;
    const TI* next;
    int64_t step;
    int n, unfetched;
    uint8_t* mine;

    __device__ void fetch(int slot)
    {
        const uint32_t to = smem_u32(mine) + slot * (kStep * ROW);
        if (unfetched >= kStep)
        {
#pragma unroll
            for (int u = 0; u < kStep; u++) cp_async<VB>(to + u * ROW, next + u * step);
        }
        else
        {
#pragma unroll
            for (int u = 0; u < kStep - 1; u++)
                if (u < unfetched) cp_async<VB>(to + u * ROW, next + u * step);
        }
        unfetched -= kStep;
        next += kStep * step;
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __device__ void begin(const TI* x, int64_t step_, int n_, uint8_t* ring)
    {
        next = x;
        step = step_;
        n = unfetched = n_;
        mine = ring + threadIdx.x * VB;
        if constexpr (V > 1)
        {
#pragma unroll
            for (int d = 0; d < kDepth - 1; d++) fetch(d);
        }
    }
    template <class F>
    __device__ void run(F f)
    {
        if constexpr (V > 1)
        {
            // not unrolled over the ring: with four activations' bodies in it the
            // loop would outgrow the instruction cache
            int slot = 0;
            for (int left = n; left > 0; left -= kStep)
            {
                asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
                Raw<TI, V> r;
                const uint8_t* at = mine + slot * (kStep * ROW);
                if (left >= kStep)
                {
#pragma unroll
                    for (int u = 0; u < kStep; u++)
                    {
                        r.q = *reinterpret_cast<const decltype(r.q)*>(at + u * ROW);
                        f(r);
                    }
                }
                else
                {
#pragma unroll 1
                    for (int u = 0; u < left; u++)
                    {
                        r.q = *reinterpret_cast<const decltype(r.q)*>(at + u * ROW);
                        f(r);
                    }
                }
                fetch(slot == 0 ? kDepth - 1 : slot - 1); // into the slot that the step before has read
                slot = slot == kDepth - 1 ? 0 : slot + 1;
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        else
        {
            int k = 0;
            for (; k + kPlain <= n; k += kPlain, next += kPlain * step)
            {
                Raw<TI, V> r[kPlain];
#pragma unroll
                for (int u = 0; u < kPlain; u++) r[u] = load_raw<TI, V>(next + u * step);
#pragma unroll
                for (int u = 0; u < kPlain; u++) f(r[u]);
            }
            for (; k < n; k++, next += step) f(load_raw<TI, V>(next));
        }
    }
};

struct Part
{
    int64_t inst, row0;
    int c0, part, nrows;
    __device__ Part(const GroupNormArgs& a)
    {
        const unsigned s = blockIdx.x / (unsigned)a.parts;
        part = (int)(blockIdx.x - s * a.parts);
        inst = s / (unsigned)a.slices;
        c0 = (int)(s - inst * a.slices) * a.slice;
        row0 = inst * a.rows + part_first(a, part);
        nrows = part_rows(a, part);
    }
};

template <typename TI, int V>
__global__ void __launch_bounds__(kThreads, kBlocks) group_norm_sums_kernel(const GroupNormArgs a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    const int G = a.groups;
    float4* own = reinterpret_cast<float4*>(smem); // [G]
    float2* red = reinterpret_cast<float2*>(own + G);
    cudaTriggerProgrammaticLaunchCompletion(); // the apply kernel waits for the results itself
    uint8_t* ring = reinterpret_cast<uint8_t*>(red) + a.red_bytes;
    const int per_thread = V / a.sub;
    const Part p(a);
    const int vpr = a.slice / V;
    const Lanes t(a, vpr, p.nrows);
    const int mine = t.mine();
    const int64_t step = t.slots * a.ldx;

    // one block of columns at a time (one block, unless a group is wider than the CTA)
    for (int cb = 0; cb < vpr; cb += t.cols)
    {
        const int col = cb + t.col;
        if (mine > 0 && col < vpr)
        {
            const TI* x = static_cast<const TI*>(a.x) + (p.row0 + t.slot) * a.ldx + p.c0 + col * V;
            Sums<V> s;
            RowStream<TI, V> rows;
            rows.begin(x, step, mine, ring);
            float2 first[kPairs<V>];
            unpack<TI, V>(load_raw<TI, V>(x), first);
            s.start(first);
            rows.run([&](const Raw<TI, V>& raw) {
                float2 f[kPairs<V>];
                unpack<TI, V>(raw, f);
                s.add(f);
            });
            leave_sums<V>(s.neg, s.s1, s.s2, mine, a.sub, red + t.col * per_thread * t.pitch() + t.slot, t.pitch());
        }
        __syncthreads();
        const int ch0 = cb * V, ch1 = min(vpr, cb + t.cols) * V;
        if (vpr <= kThreads)
        {
            const int units = a.width / a.sub;
            join_groups(
                0, G, t.live_slots(), units,
                [&](int g, int sl, int u) {
                    const float2 v = red[(g * units + u) * t.pitch() + sl];
                    return make_float3((float)(t.rows_of(sl) * a.sub), v.x, v.y);
                },
                [&](int g, float3 j) { own[g] = make_float4(j.x, j.y, j.z, 0.f); });
        }
        else
        {
            // several blocks: a group's columns may lie in two of them
            const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
            for (int g = ch0 / a.width + warp; g * a.width < ch1; g += kWarps)
            {
                const int lo = max(g * a.width, ch0), units = (min((g + 1) * a.width, ch1) - lo) / a.sub;
                const float2* entry = red + (lo - ch0) / a.sub * t.pitch();
                float3 j = make_float3(0.f, 0.f, 0.f);
                for (int sl = 0; sl < t.live_slots(); sl++)
                    for (int u = lane; u < units; u += 32)
                    {
                        const float2 v = entry[u * t.pitch() + sl];
                        j = join2(j, make_float3((float)(t.rows_of(sl) * a.sub), v.x, v.y));
                    }
#pragma unroll
                for (int m = 16; m >= 1; m >>= 1)
                    j = join2(j, make_float3(__shfl_xor_sync(0xffffffffu, j.x, m), __shfl_xor_sync(0xffffffffu, j.y, m),
                                             __shfl_xor_sync(0xffffffffu, j.z, m)));
                if (lo > g * a.width) j = join2(make_float3(own[g].x, own[g].y, own[g].z), j);
                __syncwarp();
                if (lane == 0) own[g] = make_float4(j.x, j.y, j.z, 0.f);
            }
        }
        __syncthreads();
    }
    const int64_t g0 = p.inst * a.slices * G + p.c0 / a.width;
    for (int g = threadIdx.x; g < G; g += kThreads)
        a.partial[(g0 + g) * a.parts + p.part] = make_float2(own[g].y, own[g].z);
}

template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(kThreads, kBlocks) group_norm_apply_kernel(const GroupNormArgs a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    const int G = a.groups;
    float2* stat = reinterpret_cast<float2*>(smem); // [G]
    const Part p(a);
    const int vpr = a.slice / V;
    const Lanes t(a, vpr, p.nrows);
    const int mine = t.mine();
    uint8_t* ring = smem + ((size_t)G * 8 + 15) / 16 * 16;
    const int64_t x_step = t.slots * a.ldx, o_step = t.slots * a.ldo;
    const int64_t last = p.row0 + t.slot + (int64_t)(mine - 1) * t.slots; // last row first
    const TI* x = static_cast<const TI*>(a.x) + last * a.ldx + p.c0 + t.col * V;
    TO* out = static_cast<TO*>(a.out) + last * a.ldo + p.c0 + t.col * V;
    RowStream<TI, V> rows;
    // the first rows are on their way before the sums kernel has ended (x is not its output)
    if (mine > 0 && t.col < vpr) rows.begin(x, -x_step, mine, ring);
    cudaGridDependencySynchronize();
    const int64_t g0 = p.inst * a.slices * G + p.c0 / a.width;
    join_groups(
        0, G, a.parts, 1,
        [&](int g, int k, int) {
            const float2 v = a.partial[(g0 + g) * a.parts + k];
            return make_float3((float)part_rows(a, k) * a.width, v.x, v.y);
        },
        [&](int g, float3 j) { stat[g] = make_float2(j.y, 1.f / sqrtf(not_negative(j.z / j.x) + a.eps)); });
    __syncthreads();
    for (int cb = 0; cb < vpr; cb += t.cols, x += t.cols * V, out += t.cols * V)
    {
        const int col = cb + t.col;
        if (mine == 0 || col >= vpr) continue;
        if (cb > 0) rows.begin(x, -x_step, mine, ring);
        Scale<TO, V> sc;
        sc.load(a, stat, p.c0, col);
        with_act(a.act, [&](auto act) {
            TO* o = out;
            rows.run([&](const Raw<TI, V>& raw) {
                float2 f[kPairs<V>];
                unpack<TI, V>(raw, f);
                sc.template row<decltype(act)::value>(f, o);
                o -= o_step;
            });
        });
    }
}

// ---------------------------------------------------------------- host
int gcd(int a, int b)
{
    while (b)
    {
        const int t = a % b;
        a = b;
        b = t;
    }
    return a;
}

// The widest slice of at most `most` channels made of whole units that divides C (one unit at least).
int widest_slice(int C, int unit, int most)
{
    const int units = C / unit;
    for (int d = std::min(units, std::max(1, most / unit)); d > 1; d--)
        if (units % d == 0) return unit * d;
    return unit;
}

struct Cut
{
    int held; // rows a thread of the slab kernel holds, 0: sums and apply
    int slice, parts;
};

// How a problem is cut for vectors of V channels (16 or 8 bytes, or 1 where
// groups, strides or bases do not admit them).
//   Slab kernel: slices of 64 bytes (more CTAs; 256 x 512 bf16 with SiLU 5.0 us,
//   against 5.4 in slices of 128 bytes and 5.7 with clusters of 8), 8 rows a
//   thread, clusters as small as hold the rows, and only where all of it is
//   resident at once: two CTAs a SM for clusters of up to 8 (8 x 512 x 512 takes
//   5.8 us so and 8.1 in two kernels, 2,048 x 512 7.2 and 7.7, 4,096 x 512 8.7 and
//   8.5), fewer for larger ones, which find less room (6,000 x 512: 9.2 us in
//   clusters of 12, 192 CTAs, 14.2 in clusters of 16; 7,000 x 512 15.1 in clusters
//   of 14, 224 CTAs).  What does not fit so gets up to 12 rows a thread with the
//   same bound (7,000 x 512 10.6 us and 9,000 x 512 11.1, against 11.5 and 13.3 in
//   two kernels; 4 x 4,400 x 256 10.4 and 14.2; 3 x 3,555 x 320 fp32, 288 CTAs,
//   would take 17.6 against 11.0).
//   Sums and apply: slices of at most 128 channels, one wave of CTAs (6 x
//   14,400 x 512 bf16: 51.5 us at 444 parts, 61 at 296, 56 at 888).
constexpr int kSlabCtas = kSlabBlocks * 148, kLongCtas = 192;
constexpr int kPartCtas = kBlocks * 148;
// Values a CTA at least: with fewer its set-up costs more than it saves (6 x
// 4,282 x 128 in two kernels 18.0 us at 8,192, 15.7 at 16,384 and 12.5 at 32,768; 1
// x 53,217 x 33 20.3, 22.0 and 26.1).
constexpr int kPartMin = 16384;

Cut cut(int64_t instances, int64_t rows, int C, int width, int V)
{
    Cut c = {};
    c.slice = widest_slice(C, width / gcd(width, V) * V, V > 1 ? 4 * V : 32);
    if (c.slice / V <= kThreads)
    {
        const int64_t slots = kThreads / (c.slice / V), slabs = instances * (C / c.slice);
        int64_t p = 1, fewest = (rows + slots * kHeld - 1) / (slots * kHeld);
        while (p < fewest && p < 8) p *= 2;
        p = std::max(p, fewest);
        if (p <= kMaxCluster && slabs * p <= (p > 8 ? kLongCtas : kSlabCtas)) c.held = kHeld;
        if (!c.held)
        {
            p = (rows + slots * kHeldMost - 1) / (slots * kHeldMost);
            if (p <= kMaxCluster && slabs * p <= kLongCtas) c.held = kHeldMost;
        }
        c.parts = (int)p; // of the slab kernel
    }
    if (!c.held)
    {
        // the same slices for every V that vectors_fit() admits: multiples of 8
        // channels where these fit the row, else of 4, else single groups
        const int u8 = width / gcd(width, 8) * 8, u4 = width / gcd(width, 4) * 4;
        c.slice = widest_slice(C, C % u8 == 0 ? u8 : (C % u4 == 0 ? u4 : width), 128);
        const int64_t runs = instances * (C / c.slice);
        c.parts = (int)std::max<int64_t>(1, std::min<int64_t>(kPartCtas / runs, rows * c.slice / kPartMin));
    }
    return c;
}

template <class K>
int launch_kernel(Context& ctx, K kernel, std::atomic<uint64_t>& configured, int64_t grid, int cluster, size_t smem,
                  bool after, const GroupNormArgs& a)
{
    if (grid > 0x7fffffff || smem > 200 * 1024) return S2_ERR_INVALID;
    if (set_up_current_device(configured, [&] {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
            return e != cudaSuccess ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        }) != cudaSuccess)
        return S2_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1)
    {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    if (after)
    {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx.stream;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess)
    {
        (void)cudaGetLastError();
        return S2_ERR_CUDA;
    }
    ctx.launches++;
    return S2_OK;
}

template <typename TI, typename TO, int V>
int launch(Context& ctx, GroupNormArgs a, int instances, int C, void* workspace)
{
    a.sub = gcd(a.width, V);
    const Cut c = cut(instances, a.rows, C, a.width, V);
    a.slice = c.slice;
    a.slices = C / c.slice;
    a.groups = c.slice / a.width;
    a.parts = c.parts;
    const int cols = std::min(kThreads, a.slice / V);
    a.slots = kThreads / cols;
    a.red_bytes = (int)red_bytes(cols, V / a.sub);
    a.by_cols = (uint32_t)(((1ull << 32) + cols - 1) / cols);
    a.part_rows = a.rows / c.parts;
    a.longer = a.rows - a.part_rows * c.parts;
    a.by_width = (uint32_t)(((1ull << 32) + a.width - 1) / a.width);
    const int64_t grid = (int64_t)instances * a.slices * a.parts;
    ProfileScope prof(ctx, K_NORM, 0.0, (double)instances * a.rows * C * (sizeof(TI) + sizeof(TO)));
    if (c.held)
    {
        static std::atomic<uint64_t> seen{0}, seen_long{0};
        const size_t smem = slab_smem(a.parts, a.groups, cols, V / a.sub);
        if (c.held == kHeld)
            return launch_kernel(ctx, group_norm_slab_kernel<TI, TO, V, kHeld>, seen, grid, a.parts, smem, false, a);
        return launch_kernel(ctx, group_norm_slab_kernel<TI, TO, V, kHeldMost>, seen_long, grid, a.parts, smem, false, a);
    }
    a.partial = static_cast<float2*>(workspace);
    static std::atomic<uint64_t> seen_sums{0}, seen_apply{0};
    const int r = launch_kernel(ctx, group_norm_sums_kernel<TI, V>, seen_sums, grid, 1,
                                (size_t)a.groups * 16 + red_bytes(cols, V / a.sub) + kRingBytes<TI, V>, false, a);
    if (r != S2_OK) return r;
    return launch_kernel(ctx, group_norm_apply_kernel<TI, TO, V>, seen_apply, grid, 1,
                         ((size_t)a.groups * 8 + 15) / 16 * 16 + kRingBytes<TI, V>, true, a);
}

// Vectors of V channels: whole ones in a row's groups, at aligned addresses.
template <typename TI, typename TO, int V>
bool vectors_fit(const GroupNormArgs& a, int C)
{
    const int unit = a.width / gcd(a.width, V) * V;
    const size_t in = V * sizeof(TI), out = std::min<size_t>(16, V * sizeof(TO));
    return C % unit == 0 && (a.ldx * sizeof(TI)) % in == 0 && (a.ldo * sizeof(TO)) % out == 0 &&
           reinterpret_cast<uintptr_t>(a.x) % in == 0 && reinterpret_cast<uintptr_t>(a.out) % out == 0;
}

template <typename TI, typename TO>
int launch_types(Context& ctx, const GroupNormArgs& a, int instances, int C, void* ws)
{
    if constexpr (sizeof(TI) == 2)
        if (vectors_fit<TI, TO, 8>(a, C)) return launch<TI, TO, 8>(ctx, a, instances, C, ws);
    if (vectors_fit<TI, TO, 4>(a, C)) return launch<TI, TO, 4>(ctx, a, instances, C, ws);
    return launch<TI, TO, 1>(ctx, a, instances, C, ws);
}

} // namespace

} // namespace s2

extern "C" {

size_t s2_group_norm_workspace(int instances, int64_t rows, int channels, int groups)
{
    if (instances <= 0 || rows <= 0 || channels <= 0 || groups <= 0 || channels % groups) return 0;
    size_t need = 0;
    for (int V : {8, 4, 1}) // whatever the type and alignment turn out to be
    {
        const s2::Cut c = s2::cut(instances, rows, channels, channels / groups, V);
        if (!c.held) need = std::max(need, (size_t)instances * groups * c.parts * sizeof(float2));
    }
    return need;
}

int s2_group_norm(s2_context* ctx, int instances, int64_t rows, int channels, int groups, int in_dtype, const void* x,
                  int64_t ldx, const float* gamma, const float* beta, float eps, int act, int out_dtype, void* out,
                  int64_t ldo, void* workspace, size_t workspace_bytes)
{
    if (!ctx || instances < 0 || rows < 0 || rows > (1 << 30) || channels <= 0 || channels > 65536 || groups <= 0 ||
        channels % groups != 0 || ldx < channels || ldo < channels || !(eps >= 0.f) || act < S2_ACT_NONE ||
        act > S2_ACT_GELU_ERF || (in_dtype != S2_DTYPE_F32 && in_dtype != S2_DTYPE_BF16) ||
        (out_dtype != S2_DTYPE_F32 && out_dtype != S2_DTYPE_BF16))
        return S2_ERR_INVALID;
    if (instances == 0 || rows == 0) return S2_OK;
    const uintptr_t in_mask = in_dtype == S2_DTYPE_F32 ? 3 : 1, out_mask = out_dtype == S2_DTYPE_F32 ? 3 : 1;
    if (!x || !out || (reinterpret_cast<uintptr_t>(x) & in_mask) || (reinterpret_cast<uintptr_t>(out) & out_mask) ||
        ((reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(beta)) & 3))
        return S2_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(workspace) & 7) return S2_ERR_INVALID;
    // in place only element for element
    if (x == out && (in_dtype != out_dtype || ldx != ldo)) return S2_ERR_INVALID;
    const size_t need = s2_group_norm_workspace(instances, rows, channels, groups);
    if (need > 0 && (!workspace || workspace_bytes < need)) return S2_ERR_INVALID;
    if (cudaSetDevice(ctx->c.device) != cudaSuccess) return S2_ERR_CUDA;
    s2::GroupNormArgs a = {};
    a.x = x;
    a.out = out;
    a.gamma = gamma;
    a.beta = beta;
    a.ldx = ldx;
    a.ldo = ldo;
    a.rows = (int)rows;
    a.width = channels / groups;
    a.eps = eps;
    a.act = act;
    if (in_dtype == S2_DTYPE_F32)
        return out_dtype == S2_DTYPE_F32
                   ? s2::launch_types<float, float>(ctx->c, a, instances, channels, workspace)
                   : s2::launch_types<float, __nv_bfloat16>(ctx->c, a, instances, channels, workspace);
    return out_dtype == S2_DTYPE_F32
               ? s2::launch_types<__nv_bfloat16, float>(ctx->c, a, instances, channels, workspace)
               : s2::launch_types<__nv_bfloat16, __nv_bfloat16>(ctx->c, a, instances, channels, workspace);
}

} // extern "C"
