// Group norm with an activation, channels last, on sm_100a:
//   y[i][r][c] = act((x - mean(i, g)) * rstd(i, g) * gamma[c] + beta[c]),
// g = c / (C / groups), statistics over the instance's rows and the group's
// channels, rstd = 1 / sqrt(var + eps) with the biased variance.
//
// HBM-bound: x is read once and y written once at best.  A slab (one
// instance, a slice of whole groups) belongs to one thread-block cluster, so
// its statistics need neither a workspace nor a second launch: each CTA takes
// a contiguous run of the slab's rows, keeps as many of them as fit in its
// shared memory while it sums, pushes its groups' (count, mean, M2) into every
// CTA of the cluster, and after one cluster barrier normalises -- the kept
// rows from shared memory, the others from L2 or HBM, last read first.
//
// Statistics: each thread sums d = x - p and d^2 per channel in fp32 around
// its own first value p (no cancellation for channels far from zero), turns
// them into (mean, M2), and these are joined by
//   mean = sum n_k mean_k / n,  M2 = sum M2_k + n_k (mean_k - mean)^2,
// in a fixed order: results do not depend on the run.
#include "activation.cuh"
#include "s2_common.cuh"
#include "s2_internal.h"
#include "s2_objects.h"

namespace s2 {

namespace {

constexpr int kThreads = 512;
constexpr int kMaxCluster = 16;
constexpr int kMaxSliceChannels = 128; // unless one group (or vector unit) is wider

struct GroupNormArgs
{
    const void* x;
    void* out;
    const float* gamma;
    const float* beta;
    int64_t ldx, ldo, rows;
    int width;       // channels per group
    int slice;       // channels per slab (whole groups)
    int slices;      // slabs per instance
    int cluster;     // CTAs per slab
    int stash_rows;  // rows of its run a CTA keeps in shared memory
    int groups_slab; // groups per slab
    float eps;
    int act;
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
struct Raw<float, 8>
{
    float4 lo, hi;
};

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&f)[V])
{
    if constexpr (V == 8 && sizeof(T) == 2)
    {
        const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
        for (int j = 0; j < 4; j++)
        {
            const float2 p = unpack_bf16x2(w[j]);
            f[2 * j] = p.x;
            f[2 * j + 1] = p.y;
        }
    }
    else if constexpr (V == 8)
    {
        f[0] = r.lo.x, f[1] = r.lo.y, f[2] = r.lo.z, f[3] = r.lo.w;
        f[4] = r.hi.x, f[5] = r.hi.y, f[6] = r.hi.z, f[7] = r.hi.w;
    }
    else
        f[0] = static_cast<float>(r.v[0]);
}

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p, bool last)
{
    Raw<T, V> r;
    if constexpr (V == 8 && sizeof(T) == 2)
        r.q = last ? __ldcs(reinterpret_cast<const uint4*>(p)) : *reinterpret_cast<const uint4*>(p);
    else if constexpr (V == 8)
    {
        const float4* q = reinterpret_cast<const float4*>(p);
        r.lo = last ? __ldcs(q) : q[0];
        r.hi = last ? __ldcs(q + 1) : q[1];
    }
    else
        r.v[0] = *p;
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_out(T* p, const float (&f)[V])
{
    if constexpr (V == 8 && sizeof(T) == 2)
        __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                                       pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])));
    else if constexpr (V == 8)
    {
        __stcs(reinterpret_cast<float4*>(p), make_float4(f[0], f[1], f[2], f[3]));
        __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(f[4], f[5], f[6], f[7]));
    }
    else if constexpr (sizeof(T) == 2)
        *p = __float2bfloat16_rn(f[0]);
    else
        *p = f[0];
}

__device__ __forceinline__ float warp_add(float v)
{
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, float4 v)
{
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}

// max(v, 0), NaN kept
__device__ __forceinline__ float not_negative(float v)
{
    return v < 0.f ? 0.f : v;
}

// Joins (n, mean, M2) triples k = 0 .. count-1 in order.
template <class Get>
__device__ __forceinline__ float3 join(int count, Get get)
{
    float n = 0.f, s = 0.f;
    for (int k = 0; k < count; k++)
    {
        const float4 t = get(k);
        n += t.x;
        s += t.x * t.y;
    }
    const float mean = n > 0.f ? s / n : 0.f;
    float m2 = 0.f;
    for (int k = 0; k < count; k++)
    {
        const float4 t = get(k);
        const float d = t.y - mean;
        m2 += t.z + t.x * d * d;
    }
    return make_float3(n, mean, m2);
}

// Shared memory: group table [cluster][groups] float4 | own groups float4 |
// (mean, rstd) float2 per group | reduction [kThreads * V] float2 | kept rows.
__host__ __device__ inline size_t table_bytes(int cluster, int groups)
{
    return ((size_t)(cluster + 1) * groups * 16 + (size_t)groups * 8 + 15) & ~size_t(15);
}

template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(kThreads, 1) group_norm_kernel(const GroupNormArgs a)
{
    constexpr int U = 8; // rows in flight per thread
    extern __shared__ __align__(16) uint8_t smem[];
    const int G = a.groups_slab;
    float4* table = reinterpret_cast<float4*>(smem);
    float4* own = table + a.cluster * G;
    float2* stat = reinterpret_cast<float2*>(own + G);
    float2* red = reinterpret_cast<float2*>(smem + table_bytes(a.cluster, G));
    Raw<TI, V>* stash = reinterpret_cast<Raw<TI, V>*>(red + kThreads * V);

    const int rank = a.cluster > 1 ? (int)cluster_ctarank() : 0;
    const int64_t slab = blockIdx.x / a.cluster;
    const int64_t inst = slab / a.slices;
    const int c_first = (int)(slab - inst * a.slices) * a.slice;
    const int64_t per = (a.rows + a.cluster - 1) / a.cluster;
    const int64_t r0 = rank * per;
    const int64_t left = a.rows - r0;
    const int nrows = left <= 0 ? 0 : (int)(left < per ? left : per);
    const int64_t row_base = inst * a.rows + r0;
    const TI* x = static_cast<const TI*>(a.x) + row_base * a.ldx + c_first;
    TO* out = static_cast<TO*>(a.out) + row_base * a.ldo + c_first;

    const int vpr = a.slice / V; // vectors per row
    const int cbw = vpr < kThreads ? vpr : kThreads;
    const int slots = kThreads / cbw;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int slot = tid / cbw, tcol = tid - slot * cbw;
    const int stash_rows = a.stash_rows < nrows ? a.stash_rows : nrows;

    for (int j = tid; j < G; j += kThreads) own[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    // every CTA of the cluster runs before any writes into its shared memory
    if (a.cluster > 1) cluster_sync();

    // ---- statistics, one block of cbw vector columns at a time
    for (int cb = 0; cb < vpr; cb += cbw)
    {
        const int col = cb + tcol;
        const bool live = slot < slots && col < vpr && slot < nrows;
        if (live)
        {
            float p[V], s1[V], s2[V];
            const TI* px = x + (int64_t)slot * a.ldx + (int64_t)col * V;
            unpack<TI, V>(load_raw<TI, V>(px, false), p);
#pragma unroll
            for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.f;
            const int64_t step = (int64_t)slots * a.ldx;
            int r = slot;
            for (; r + (U - 1) * slots < nrows; r += U * slots, px += U * step)
            {
                Raw<TI, V> raw[U];
#pragma unroll
                for (int u = 0; u < U; u++) raw[u] = load_raw<TI, V>(px + u * step, false);
#pragma unroll
                for (int u = 0; u < U; u++)
                {
                    const int rr = r + u * slots;
                    if (rr < stash_rows) stash[rr * vpr + col] = raw[u];
                    float f[V];
                    unpack<TI, V>(raw[u], f);
#pragma unroll
                    for (int j = 0; j < V; j++)
                    {
                        const float d = f[j] - p[j];
                        s1[j] += d;
                        s2[j] = fmaf(d, d, s2[j]);
                    }
                }
            }
            for (; r < nrows; r += slots, px += step)
            {
                const Raw<TI, V> raw = load_raw<TI, V>(px, false);
                if (r < stash_rows) stash[r * vpr + col] = raw;
                float f[V];
                unpack<TI, V>(raw, f);
#pragma unroll
                for (int j = 0; j < V; j++)
                {
                    const float d = f[j] - p[j];
                    s1[j] += d;
                    s2[j] = fmaf(d, d, s2[j]);
                }
            }
            const float inv_n = 1.f / (float)((nrows - slot + slots - 1) / slots);
#pragma unroll
            for (int j = 0; j < V; j++)
            {
                const float m = s1[j] * inv_n;
                red[(slot * cbw + tcol) * V + j] = make_float2(p[j] + m, not_negative(s2[j] - s1[j] * m));
            }
        }
        __syncthreads();
        // one warp per group with channels in this block
        const int ch0 = cb * V, ch1 = min(vpr, cb + cbw) * V;
        const int slots_live = slots < nrows ? slots : nrows;
        for (int g = ch0 / a.width + warp; g * a.width < ch1; g += kThreads / 32)
        {
            const int lo = max(g * a.width, ch0) - ch0, w = min((g + 1) * a.width, ch1) - ch0 - lo;
            const int entries = slots_live * w;
            float n = 0.f, s = 0.f;
            for (int e = lane; e < entries; e += 32)
            {
                const int sl = e / w;
                const float k = (float)((nrows - sl + slots - 1) / slots);
                n += k;
                s += k * red[sl * cbw * V + lo + (e - sl * w)].x;
            }
            n = warp_add(n);
            s = warp_add(s);
            const float mean = n > 0.f ? s / n : 0.f;
            float m2 = 0.f;
            for (int e = lane; e < entries; e += 32)
            {
                const int sl = e / w;
                const float k = (float)((nrows - sl + slots - 1) / slots);
                const float2 t = red[sl * cbw * V + lo + (e - sl * w)];
                const float d = t.x - mean;
                m2 += t.y + k * d * d;
            }
            m2 = warp_add(m2);
            if (lane == 0)
            {
                const float4 was = own[g];
                const float4 now = make_float4(n, mean, m2, 0.f);
                const float3 both = join(2, [&](int k) { return k ? now : was; });
                own[g] = make_float4(both.x, both.y, both.z, 0.f);
            }
        }
        __syncthreads();
    }

    // ---- exchange over the cluster
    for (int e = tid; e < G * a.cluster; e += kThreads)
    {
        const int to = e / G, g = e - to * G;
        if (a.cluster > 1)
            st_cluster_v4(mapa_shared(table + rank * G + g, to), own[g]);
        else
            table[g] = own[g];
    }
    if (a.cluster > 1)
        cluster_sync();
    else
        __syncthreads();
    for (int g = tid; g < G; g += kThreads)
    {
        const float3 t = join(a.cluster, [&](int k) { return table[k * G + g]; });
        stat[g] = make_float2(t.y, 1.f / sqrtf(not_negative(t.z / t.x) + a.eps));
    }
    __syncthreads();

    // ---- normalise: rows not kept first, last read first, then the kept ones
    for (int cb = 0; cb < vpr; cb += cbw)
    {
        const int col = cb + tcol;
        if (slot >= slots || col >= vpr || slot >= nrows) continue;
        float mean[V], mul[V], add[V];
#pragma unroll
        for (int j = 0; j < V; j++)
        {
            const int c = col * V + j;
            const float2 t = stat[c / a.width];
            mean[j] = t.x;
            mul[j] = t.y * (a.gamma ? __ldg(a.gamma + c_first + c) : 1.f);
            add[j] = a.beta ? __ldg(a.beta + c_first + c) : 0.f;
        }
        auto emit = [&](const Raw<TI, V>& raw, int r) {
            float f[V];
            unpack<TI, V>(raw, f);
#pragma unroll
            for (int j = 0; j < V; j++) f[j] = fmaf(f[j] - mean[j], mul[j], add[j]);
            activate<V>(f, a.act);
            store_out<TO, V>(out + (int64_t)r * a.ldo + (int64_t)col * V, f);
        };
        constexpr int W = 4;
        // this thread's rows are slot + k * slots; the first kept_k of them are in shared memory
        const int total_k = (nrows - slot + slots - 1) / slots;
        const int kept_k = stash_rows > slot ? (stash_rows - slot + slots - 1) / slots : 0;
        int k = total_k;
        for (; k - W >= kept_k; k -= W)
        {
            Raw<TI, V> raw[W];
#pragma unroll
            for (int u = 0; u < W; u++)
                raw[u] = load_raw<TI, V>(x + (int64_t)(slot + (k - 1 - u) * slots) * a.ldx + (int64_t)col * V, true);
#pragma unroll
            for (int u = 0; u < W; u++) emit(raw[u], slot + (k - 1 - u) * slots);
        }
        for (; k > kept_k; k--)
        {
            const int r = slot + (k - 1) * slots;
            emit(load_raw<TI, V>(x + (int64_t)r * a.ldx + (int64_t)col * V, true), r);
        }
        for (k = 0; k < kept_k; k++)
        {
            const int r = slot + k * slots;
            emit(stash[r * vpr + col], r);
        }
    }
}

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

template <typename TI, typename TO, int V>
int launch(Context& ctx, GroupNormArgs a, int instances, int C, int unit)
{
    // Slice: whole groups in whole vectors, a divisor of C.  Wide slices keep
    // rows contiguous; narrower ones (down to 64 bytes) make more slabs, taken
    // until eight clusters of 16 CTAs can work.
    const int units = C / unit;
    int slice = unit;
    for (int d = units; d >= 1; d--)
    {
        if (units % d) continue;
        slice = unit * d;
        if (d == 1) break;
        if (slice > kMaxSliceChannels) continue;
        if ((int64_t)instances * (C / slice) >= 8) break;
        int narrower = 0; // the next narrower slice of at least 64 bytes
        for (int e = d - 1; e >= 1 && !narrower; e--)
            if (units % e == 0) narrower = e;
        if (unit * narrower * (int)sizeof(TI) < 64) break;
    }
    a.slice = slice;
    a.slices = C / slice;
    a.groups_slab = slice / a.width;
    const int64_t slabs = (int64_t)instances * a.slices;
    const size_t row_bytes = (size_t)slice * sizeof(TI);
    const size_t fixed = (size_t)kThreads * V * sizeof(float2);
    const size_t limit = 227 * 1024;
    auto keep_bytes = [&](int cs) { return limit - fixed - table_bytes(cs, a.groups_slab); };
    int cs = 1;
    while (cs < kMaxCluster)
    {
        const int64_t bytes = ((a.rows + cs - 1) / cs) * (int64_t)row_bytes;
        const bool idle = slabs * cs < ctx.num_sms && bytes > 16384;
        const bool spills = bytes > (int64_t)keep_bytes(cs);
        if (!idle && !spills) break;
        cs *= 2;
    }
    if (slabs * cs > 0x7fffffff || table_bytes(cs, a.groups_slab) + fixed > limit) return S2_ERR_INVALID;
    a.cluster = cs;
    const int64_t run = (a.rows + cs - 1) / cs;
    const int64_t fit = (int64_t)(keep_bytes(cs) / row_bytes);
    a.stash_rows = slice / V <= kThreads ? (int)(run < fit ? run : fit) : 0;
    const size_t smem = table_bytes(cs, a.groups_slab) + fixed + (size_t)a.stash_rows * row_bytes;

    static std::atomic<uint64_t> configured{0};
    auto kernel = group_norm_kernel<TI, TO, V>;
    if (first_on_device(configured))
    {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)limit) != cudaSuccess ||
            cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return S2_ERR_CUDA;
    }
    const double n = (double)instances * a.rows * C;
    ProfileScope prof(ctx, K_NORM, 0.0, n * (sizeof(TI) + sizeof(TO)));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(slabs * cs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx.stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess)
    {
        (void)cudaGetLastError();
        return S2_ERR_CUDA;
    }
    ctx.launches++;
    return S2_OK;
}

template <typename TI, typename TO>
int launch_types(Context& ctx, const GroupNormArgs& a, int instances, int C)
{
    // 8 channels a thread where rows and groups allow 16-byte accesses
    const int unit = a.width / gcd(a.width, 8) * 8;
    const bool vec = C % unit == 0 && (a.ldx * (int64_t)sizeof(TI)) % 16 == 0 && (a.ldo * (int64_t)sizeof(TO)) % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
    return vec ? launch<TI, TO, 8>(ctx, a, instances, C, unit) : launch<TI, TO, 1>(ctx, a, instances, C, a.width);
}

} // namespace

} // namespace s2

extern "C" {

int s2_group_norm(s2_context* ctx, int instances, int64_t rows, int channels, int groups, int in_dtype, const void* x,
                  int64_t ldx, const float* gamma, const float* beta, float eps, int act, int out_dtype, void* out,
                  int64_t ldo)
{
    if (!ctx || instances < 0 || rows < 0 || rows > (1 << 30) || channels <= 0 || groups <= 0 ||
        channels % groups != 0 || ldx < channels || ldo < channels || !(eps >= 0.f) || act < S2_ACT_NONE ||
        act > S2_ACT_GELU_ERF || (in_dtype != S2_DTYPE_F32 && in_dtype != S2_DTYPE_BF16) ||
        (out_dtype != S2_DTYPE_F32 && out_dtype != S2_DTYPE_BF16))
        return S2_ERR_INVALID;
    if (instances == 0 || rows == 0) return S2_OK;
    const uintptr_t in_mask = in_dtype == S2_DTYPE_F32 ? 3 : 1, out_mask = out_dtype == S2_DTYPE_F32 ? 3 : 1;
    if (!x || !out || (reinterpret_cast<uintptr_t>(x) & in_mask) || (reinterpret_cast<uintptr_t>(out) & out_mask) ||
        ((reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(beta)) & 3))
        return S2_ERR_INVALID;
    // in place only element for element
    if (x == out && (in_dtype != out_dtype || ldx != ldo)) return S2_ERR_INVALID;
    if (cudaSetDevice(ctx->c.device) != cudaSuccess) return S2_ERR_CUDA;
    s2::GroupNormArgs a = {};
    a.x = x;
    a.out = out;
    a.gamma = gamma;
    a.beta = beta;
    a.ldx = ldx;
    a.ldo = ldo;
    a.rows = rows;
    a.width = channels / groups;
    a.eps = eps;
    a.act = act;
    if (in_dtype == S2_DTYPE_F32)
        return out_dtype == S2_DTYPE_F32 ? s2::launch_types<float, float>(ctx->c, a, instances, channels)
                                         : s2::launch_types<float, __nv_bfloat16>(ctx->c, a, instances, channels);
    return out_dtype == S2_DTYPE_F32 ? s2::launch_types<__nv_bfloat16, float>(ctx->c, a, instances, channels)
                                     : s2::launch_types<__nv_bfloat16, __nv_bfloat16>(ctx->c, a, instances, channels);
}

} // extern "C"
