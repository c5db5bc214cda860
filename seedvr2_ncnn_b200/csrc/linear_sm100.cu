// Linear and grouped linear on sm_100a:
//   out[r] = residual[r] + gate[g] * act(A[r] W[g]^T + bias[g]),  offsets[g] <= r < offsets[g + 1]
// (s2_linear is the one-group form).  Two kernels:
//   * linear_tile_kernel: output tiles of 128 rows a CTA (or 256 rows a CTA
//     pair), persistent, for many rows;
//   * linear_rows_kernel: 128 output features a CTA against a few rows, K
//     split over a thread-block cluster, for few rows a group.
#include <algorithm>

#include "activation.cuh"
#include "s2_common.cuh"
#include "s2_internal.h"
#include "s2_objects.h"

namespace s2 {

namespace {

constexpr int BM = 128;
constexpr int BK = 64; // one 128-byte swizzle row of bf16
constexpr int A_BYTES = BM * BK * 2;
constexpr int kMaxGroups = 1024;
constexpr size_t kSmemLimit = 232448;

struct LinearArgs
{
    int rows, N, K, groups, num_kb, nblk;
    const int* offsets; // device [groups + 1], or null: one group of all rows
    int act;
    const float* bias;
    const float* gate;
    const void* residual;
    int64_t residual_ld;
    void* out;
    int64_t out_ld;
    int out_f32;
    int tma_out; // out through its tensor map
    int tma_res; // residual through its tensor map
    int stages;
    int group_m; // M blocks per raster group
    int cluster; // linear_rows_kernel: K parts
    int* status;
};

__device__ __forceinline__ void add_bias32(const LinearArgs& a, const float* bias, int n, float (&x)[32])
{
    if (n + 32 <= a.N && (reinterpret_cast<uintptr_t>(bias + n) & 15) == 0)
    {
#pragma unroll
        for (int j = 0; j < 32; j += 4)
        {
            const float4 b = __ldg(reinterpret_cast<const float4*>(bias + n + j));
            x[j] += b.x;
            x[j + 1] += b.y;
            x[j + 2] += b.z;
            x[j + 3] += b.w;
        }
    }
    else
    {
#pragma unroll
        for (int j = 0; j < 32; j++) x[j] += n + j < a.N ? __ldg(bias + n + j) : 0.f;
    }
}

__device__ __forceinline__ void mul_gate32(const LinearArgs& a, const float* gate, int n, float (&x)[32])
{
    if (n + 32 <= a.N && (reinterpret_cast<uintptr_t>(gate + n) & 15) == 0)
    {
#pragma unroll
        for (int j = 0; j < 32; j += 4)
        {
            const float4 g = __ldg(reinterpret_cast<const float4*>(gate + n + j));
            x[j] *= g.x;
            x[j + 1] *= g.y;
            x[j + 2] *= g.z;
            x[j + 3] *= g.w;
        }
    }
    else
    {
#pragma unroll
        for (int j = 0; j < 32; j++) x[j] *= n + j < a.N ? __ldg(gate + n + j) : 0.f;
    }
}

// Group rows and unit numbers of a launch, built once per CTA in shared
// memory by one warp: off[j] (j <= groups) is the offset clamped to [0, rows]
// and to its predecessors, so no offset array can lead a row outside the
// buffers (a changed one records a bad index); first[j] the first unit of
// group j, first[groups] their number.
__device__ __forceinline__ void build_groups(const LinearArgs& a, int rows_per_unit, int* off, int* first)
{
    const int lane = threadIdx.x & 31;
    if (!a.offsets)
    {
        if (lane == 0)
        {
            off[0] = 0;
            off[1] = a.rows;
            first[0] = 0;
            first[1] = (a.rows + rows_per_unit - 1) / rows_per_unit * a.nblk;
        }
        return;
    }
    int carry = 0;
    bool bad = false;
    for (int base = 0; base <= a.groups; base += 32)
    {
        const int j = base + lane;
        const int raw = j <= a.groups ? __ldg(a.offsets + j) : 0;
        int v = max(0, min(raw, a.rows));
#pragma unroll
        for (int m = 1; m < 32; m <<= 1)
        {
            const int o = __shfl_up_sync(0xffffffffu, v, m);
            if (lane >= m) v = max(v, o);
        }
        v = max(v, carry);
        if (j <= a.groups)
        {
            off[j] = v;
            bad |= v != raw;
        }
        carry = __shfl_sync(0xffffffffu, v, 31);
    }
    if (bad) record_status(a.status, kStatusBadIndex);
    __syncwarp();
    carry = 0;
    for (int base = 0; base < a.groups; base += 32)
    {
        const int j = base + lane;
        const int own = j < a.groups ? (off[j + 1] - off[j] + rows_per_unit - 1) / rows_per_unit * a.nblk : 0;
        int v = own;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1)
        {
            const int o = __shfl_up_sync(0xffffffffu, v, m);
            if (lane >= m) v += o;
        }
        if (j < a.groups) first[j] = carry + v - own;
        carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) first[a.groups] = carry;
}

// One role's walk over the CTA's units (increasing, so the group cursor only
// moves forward).
struct Unit
{
    int group, m0, end, n0; // first row of the unit, end of the group's rows, first column
};
template <int BMT, int BN>
struct UnitWalk
{
    const int* off;
    const int* first;
    int g = 0;
    __device__ Unit decode(const LinearArgs& a, int u)
    {
        while (u >= first[g + 1]) g++;
        const int t = u - first[g];
        const int mt = (off[g + 1] - off[g] + BMT - 1) / BMT;
        const int per = a.group_m * a.nblk;
        const int q = t / per;
        const int gm = min(a.group_m, mt - q * a.group_m);
        const int r = t - q * per;
        Unit v;
        v.group = g;
        v.m0 = off[g] + (q * a.group_m + r % gm) * BMT;
        v.end = off[g + 1];
        v.n0 = r / gm * BN;
        return v;
    }
};

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity)
{
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(bar, parity))
        if (global_timer_ns() - t0 > kWaitLimitNs) break;
}

// ---------------------------------------------------------------- many rows
constexpr int kEpiWarps = 8; // two per TMEM lane quarter, half the columns each
constexpr int kTileThreads = 64 + 32 * kEpiWarps;
constexpr int kBox = 4096; // 32 rows x 128 bytes

// CTAS = 2: a pair of CTAs (cluster of 2) computes 256 rows x BN columns with
// M = 256 MMAs, each holding its 128 rows of A and BN / 2 rows of W.
template <int CTAS, int BN, int R>
struct TileShape
{
    static constexpr int W_BYTES = BN / CTAS * BK * 2;
    static constexpr int STAGE_BYTES = A_BYTES + W_BYTES;
    static constexpr int EPI_BYTES = kEpiWarps * R * kBox;
    static constexpr int TMEM_COLS = 2 * BN;
    static constexpr uint32_t IDESC = umma_idesc_bf16(CTAS * BM, BN, 0, 0);
    static constexpr int MAX_STAGES = 8;
    static size_t fixed_bytes(int groups) { return 1024 + EPI_BYTES + 512 + 8 * (size_t)(groups + 1); }
    static int stages(int groups)
    {
        const int s = (int)((kSmemLimit - fixed_bytes(groups)) / STAGE_BYTES);
        return s < MAX_STAGES ? s : MAX_STAGES;
    }
};

// Byte of (row r, byte b) in a 128-byte-swizzled box.
__device__ __forceinline__ int box_at(int r, int b)
{
    return r * 128 + ((((b >> 4) ^ r) & 7) << 4) + (b & 15);
}

// Rows and columns that a tensor map cannot take (group ends inside a box,
// strides or bases off 16 bytes): the warp copies element by element.
template <typename T>
__device__ __forceinline__ void box_to_global(const uint8_t* box, T* out, int64_t ld, int rows, int cols, int lane)
{
    constexpr int W = 128 / sizeof(T);
    for (int r = 0; r < rows; r++)
#pragma unroll
        for (int c = lane; c < W; c += 32)
            if (c < cols) out[r * ld + c] = *reinterpret_cast<const T*>(box + box_at(r, c * (int)sizeof(T)));
}
template <typename T>
__device__ __forceinline__ void global_to_box(uint8_t* box, const T* in, int64_t ld, int rows, int cols, int lane)
{
    constexpr int W = 128 / sizeof(T);
    for (int r = 0; r < rows; r++)
#pragma unroll
        for (int c = lane; c < W; c += 32)
            if (c < cols) *reinterpret_cast<T*>(box + box_at(r, c * (int)sizeof(T))) = in[r * ld + c];
}

// Epilogue of one warp over all of the CTA's units.  Boxes (32 rows x 128
// bytes of output) run in a fixed sequence; each is combined in one of the
// warp's R shared-memory boxes and written by one TMA store.  A residual box is
// TMA-loaded R - 1 boxes ahead into the slot its result will leave from.
template <int CTAS, int BN, int R>
__device__ __forceinline__ void tile_epilogue(const LinearArgs& a, const CUtensorMap* tmap_out,
                                              const CUtensorMap* tmap_res, UnitWalk<CTAS * BM, BN> walk,
                                              UnitWalk<CTAS * BM, BN> ahead, int first_unit, int step, int units,
                                              int rank, uint8_t* stg, uint64_t* rfull, uint64_t* tfull,
                                              uint64_t* tempty, uint32_t tmem_base, int quarter, int half, int lane,
                                              volatile int* abort_flag)
{
    const int esz = a.out_f32 ? 4 : 2;
    const int box_cols = 128 / esz;
    const int row_in = rank * BM + quarter * 32; // of the unit, this warp's first
    const int c_lo = half * (BN / 2), c_hi = c_lo + BN / 2;
    const int sw = lane & 7;
    // loader cursor (lane 0)
    int lu = first_unit, lc = c_lo, lq = 0;
    Unit lun{};
    bool have = false;
    auto issue_load = [&]() {
        for (;;)
        {
            if (lu >= units) return;
            if (!have)
            {
                lun = ahead.decode(a, lu);
                have = true;
                lc = c_lo;
            }
            if (lc < c_hi && lun.n0 + lc < a.N && lun.m0 + row_in < lun.end) break;
            lu += step;
            have = false;
        }
        const int slot = lq % R;
        mbar_arrive_expect_tx(&rfull[slot], kBox);
        tma_load_2d(stg + slot * kBox, tmap_res, &rfull[slot], lun.n0 + lc, lun.m0 + row_in);
        lq++;
        lc += box_cols;
    };
    if (a.tma_res && lane == 0)
        for (int i = 0; i < R - 1; i++) issue_load();

    int q = 0, acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int u = first_unit; u < units && ok; u += step)
    {
        int w = 0;
        if (lane == 0) w = mbar_wait<true>(&tfull[acc], acc_phase, abort_flag, a.status) ? 1 : 0;
        w = __shfl_sync(0xffffffffu, w, 0);
        if (!w) break;
        __syncwarp();
        tc_fence_after();
        const Unit un = walk.decode(a, u);
        const int row0 = un.m0 + row_in;
        const int live_rows = min(32, un.end - row0);
        const float* bias = a.bias ? a.bias + (int64_t)un.group * a.N : nullptr;
        const float* gate = a.gate ? a.gate + (int64_t)un.group * a.N : nullptr;
        const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN;
#pragma unroll 1
        for (int c = c_lo; c < c_hi && un.n0 + c < a.N && live_rows > 0; c += box_cols, q++)
        {
            const int slot = q % R;
            uint8_t* box = stg + slot * kBox;
            const int n = un.n0 + c;
            const int live_cols = min(box_cols, a.N - n);
            if (a.tma_res)
            {
                int r = 0;
                if (lane == 0) r = mbar_wait<true>(&rfull[slot], (uint32_t)(q / R) & 1u, abort_flag, a.status) ? 1 : 0;
                r = __shfl_sync(0xffffffffu, r, 0);
                if (!r)
                {
                    ok = false;
                    break;
                }
            }
            else
            {
                if (lane == 0) bulk_wait_read<R - 1>(); // this slot's previous store has read it
                __syncwarp();
                if (a.residual)
                {
                    const int64_t at = (int64_t)row0 * a.residual_ld + n;
                    if (a.out_f32)
                        global_to_box(box, static_cast<const float*>(a.residual) + at, a.residual_ld, live_rows,
                                      live_cols, lane);
                    else
                        global_to_box(box, static_cast<const uint16_t*>(a.residual) + at, a.residual_ld, live_rows,
                                      live_cols, lane);
                    __syncwarp();
                }
            }
            uint8_t* srow = box + lane * 128;
#pragma unroll 1
            for (int k = 0; k < box_cols / 32; k++)
            {
                uint32_t v[32];
                tmem_ld32(t_row + c + 32 * k, v);
                tmem_ld_wait();
                float x[32];
#pragma unroll
                for (int j = 0; j < 32; j++) x[j] = __uint_as_float(v[j]);
                if (bias) add_bias32(a, bias, n + 32 * k, x);
                activate<32>(x, a.act);
                if (gate) mul_gate32(a, gate, n + 32 * k, x);
                if (a.out_f32)
                {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                    {
                        float4* p = reinterpret_cast<float4*>(srow + ((j ^ sw) << 4));
                        float4 o = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
                        if (a.residual)
                        {
                            const float4 r = *p;
                            o.x += r.x;
                            o.y += r.y;
                            o.z += r.z;
                            o.w += r.w;
                        }
                        *p = o;
                    }
                }
                else
                {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                    {
                        uint4* p = reinterpret_cast<uint4*>(srow + (((4 * k + j) ^ sw) << 4));
                        if (a.residual)
                        {
                            const uint4 r = *p;
                            const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                            for (int e = 0; e < 4; e++)
                            {
                                const float2 f = unpack_bf16x2(rw[e]);
                                x[8 * j + 2 * e] += f.x;
                                x[8 * j + 2 * e + 1] += f.y;
                            }
                        }
                        *p = make_uint4(pack_bf16x2(x[8 * j], x[8 * j + 1]), pack_bf16x2(x[8 * j + 2], x[8 * j + 3]),
                                        pack_bf16x2(x[8 * j + 4], x[8 * j + 5]),
                                        pack_bf16x2(x[8 * j + 6], x[8 * j + 7]));
                    }
                }
            }
            const bool whole = a.tma_out && live_rows == 32;
            fence_proxy_async_smem();
            __syncwarp();
            if (!whole)
            {
                const int64_t at = (int64_t)row0 * a.out_ld + n;
                if (a.out_f32)
                    box_to_global(box, static_cast<float*>(a.out) + at, a.out_ld, live_rows, live_cols, lane);
                else
                    box_to_global(box, static_cast<uint16_t*>(a.out) + at, a.out_ld, live_rows, live_cols, lane);
                fence_proxy_async_smem(); // before a TMA load reuses the box
                __syncwarp();
            }
            if (lane == 0)
            {
                if (whole) tma_store_2d(tmap_out, box, n, row0);
                bulk_commit();
                if (a.tma_res)
                {
                    bulk_wait_read<1>(); // the store of box q-1 has read box (q-1) % R
                    issue_load();        // box q+R-1 into it
                }
            }
        }
        if (!ok) break;
        tc_fence_before();
        __syncwarp();
        if (lane == 0)
        {
            if (CTAS == 2)
                mbar_arrive_cluster(mapa_shared(&tempty[acc], 0));
            else
                mbar_arrive(&tempty[acc]);
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
    }
    if (lane == 0)
    {
        // no TMA load may land after the CTA exits
        if (a.tma_res)
            for (int i = q; i < lq; i++) drain_wait(&rfull[i % R], (uint32_t)(i / R) & 1u);
        bulk_wait<0>();
    }
    __syncwarp();
}

template <int CTAS, int BN, int R>
__global__ void __launch_bounds__(kTileThreads, 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                       const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ CUtensorMap tmap_res,
                       const LinearArgs args)
{
    using TL = TileShape<CTAS, BN, R>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int stages = args.stages;
    uint8_t* epi_stage = smem + stages * TL::STAGE_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(epi_stage + TL::EPI_BYTES);
    uint64_t* empty = full + TL::MAX_STAGES;
    uint64_t* tfull = empty + TL::MAX_STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint64_t* rfull = drain + 1; // [kEpiWarps][R]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rfull + kEpiWarps * R);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((2 * TL::MAX_STAGES + 5 + kEpiWarps * R) * 8 + 8 <= 512, "barriers");
    int* off = reinterpret_cast<int*>(epi_stage + TL::EPI_BYTES + 512);
    int* first = off + args.groups + 1;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = CTAS == 2 ? (int)cluster_ctarank() : 0;
    const bool leader = rank == 0;
    const int unit0 = blockIdx.x / CTAS, step = gridDim.x / CTAS;

    if (threadIdx.x == 0)
    {
        for (int s = 0; s < stages; s++)
        {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++)
        {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], CTAS * kEpiWarps);
        }
        mbar_init(drain, 1);
        for (int i = 0; i < kEpiWarps * R; i++) mbar_init(&rfull[i], 1);
        *abort_flag = 0;
        *tmem_slot = 0;
        fence_mbarrier_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_w);
        if (args.tma_out) tma_prefetch_desc(&tmap_out);
        if (args.tma_res) tma_prefetch_desc(&tmap_res);
    }
    if (warp == 2) build_groups(args, CTAS * BM, off, first);
    __syncthreads();
    if (warp == 1)
    {
        if (CTAS == 2)
            tmem_alloc_pair(tmem_slot, TL::TMEM_COLS);
        else
            tmem_alloc(tmem_slot, TL::TMEM_COLS);
    }
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync(); // both CTAs' barriers exist before any remote arrival
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int units = first[args.groups];
    UnitWalk<CTAS * BM, BN> walk{off, first};

    if (warp == 0)
    {
        if (lane == 0)
        {
            // ---------------- TMA producer (a pair completes on the leader's barriers)
            int stage = 0;
            uint32_t phase = 0, issued = 0, last_phase = 0; // one bit per stage
            for (int u = unit0; u < units && !*abort_flag; u += step)
            {
                const Unit un = walk.decode(args, u);
                const int ay = un.m0 + rank * BM;
                const int wy = un.group * args.N + un.n0 + rank * (BN / CTAS);
                for (int kb = 0; kb < args.num_kb; kb++)
                {
                    if (!mbar_wait<true>(&empty[stage], phase ^ 1, abort_flag, args.status)) break;
                    uint8_t* sa = smem + stage * TL::STAGE_BYTES;
                    uint8_t* sb = sa + A_BYTES;
                    if (CTAS == 2)
                    {
                        if (leader) mbar_arrive_expect_tx(&full[stage], 2 * TL::STAGE_BYTES);
                        const uint32_t fb = mapa_shared(&full[stage], 0);
                        tma_load_2d_pair(sa, &tmap_a, fb, kb * BK, ay);
                        tma_load_2d_pair(sb, &tmap_w, fb, kb * BK, wy);
                    }
                    else
                    {
                        mbar_arrive_expect_tx(&full[stage], TL::STAGE_BYTES);
                        tma_load_2d(sa, &tmap_a, &full[stage], kb * BK, ay);
                        tma_load_2d(sb, &tmap_w, &full[stage], kb * BK, wy);
                    }
                    issued |= 1u << stage;
                    last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == stages)
                    {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // No TMA write may land after the CTAs exit (the peer's loads
            // complete on the leader's barriers too).
            if (*abort_flag && leader)
                for (int s = 0; s < stages; s++)
                    if ((issued >> s) & 1) drain_wait(&full[s], (last_phase >> s) & 1);
        }
    }
    else if (warp == 1)
    {
        if (lane == 0 && leader)
        {
            // ---------------- MMA issuer
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            for (int u = unit0; u < units && !*abort_flag; u += step)
            {
                if (!mbar_wait<true>(&tempty[acc], acc_phase ^ 1, abort_flag, args.status)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * BN;
                bool ok = true;
                for (int kb = 0; kb < args.num_kb; kb++)
                {
                    if (!mbar_wait<true>(&full[stage], phase, abort_flag, args.status))
                    {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(smem + stage * TL::STAGE_BYTES);
                    const uint32_t b_addr = a_addr + A_BYTES;
#pragma unroll
                    for (int k = 0; k < BK / 16; k++)
                    {
                        const uint64_t ad = umma_desc_sw128(a_addr + k * 32, 16, 1024);
                        const uint64_t bd = umma_desc_sw128(b_addr + k * 32, 16, 1024);
                        if (CTAS == 2)
                            umma_bf16_pair(d_tmem, ad, bd, TL::IDESC, (kb | k) != 0);
                        else
                            umma_bf16(d_tmem, ad, bd, TL::IDESC, (kb | k) != 0);
                    }
                    if (CTAS == 2)
                        umma_commit_pair(&empty[stage], 0x3);
                    else
                        umma_commit(&empty[stage]);
                    if (++stage == stages)
                    {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                if (CTAS == 2)
                    umma_commit_pair(&tfull[acc], 0x3);
                else
                    umma_commit(&tfull[acc]);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
            // every MMA completes (in both CTAs) before TMEM is released
            if (CTAS == 2)
                umma_commit_pair(drain, 0x3);
            else
                umma_commit(drain);
        }
        if (lane == 0) drain_wait(drain, 0);
    }
    else
    {
        const int e = warp - 2;
        tile_epilogue<CTAS, BN, R>(args, &tmap_out, &tmap_res, walk, walk, unit0, step, units, rank,
                                   epi_stage + e * R * kBox, rfull + e * R, tfull, tempty, tmem_base, warp & 3, e >> 2,
                                   lane, abort_flag);
    }

    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync(); // no remote arrival or MMA operand read outlives either CTA
    tc_fence_after();
    if (warp == 1)
    {
        if (CTAS == 2)
            tmem_dealloc_pair(tmem_base, TL::TMEM_COLS);
        else
            tmem_dealloc(tmem_base, TL::TMEM_COLS);
    }
}

// ---------------------------------------------------------------- few rows
// The product transposed: 128 features of W are the MMA's rows, TN rows of A
// its columns, so few rows cost few tensor core cycles and the kernel is
// bound by reading W.  A cluster of S CTAs splits K; each leaves its fp32
// partial sums in its shared memory, and after a cluster barrier CTA r adds
// the S parts of rows r, r + S, ... in rank order (the result does not depend
// on the run), applies the epilogue and stores.
constexpr int kRowsThreads = 192;

template <int TN>
struct RowsShape
{
    static constexpr int W_BYTES = 128 * BK * 2;
    static constexpr int X_BYTES = TN * BK * 2;
    static constexpr int STAGE_BYTES = W_BYTES + X_BYTES;
    static constexpr int PART_BYTES = TN * 128 * 4;
    // two CTAs a SM
    static constexpr int STAGES = (112 * 1024 - PART_BYTES - 1024 - 256) / STAGE_BYTES;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + PART_BYTES + 1024 + 256;
    static constexpr uint32_t IDESC = umma_idesc_bf16(128, TN, 0, 0);
    static constexpr int TMEM_COLS = TN < 32 ? 32 : TN;
    static_assert((2 * STAGES + 3) * 8 + 8 <= 256, "barriers");
};

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

template <int TN>
__global__ void __launch_bounds__(kRowsThreads, 2)
    linear_rows_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                       const LinearArgs args)
{
    using RS = RowsShape<TN>;
    constexpr int STAGES = RS::STAGES;
    const int S = args.cluster;
    const int rank = S > 1 ? (int)cluster_ctarank() : 0;
    const int unit = blockIdx.x / S;
    const int group = unit / args.nblk;
    const int n0 = (unit - group * args.nblk) * 128;
    int lo = 0, hi = args.rows;
    if (args.offsets)
    {
        const int a = __ldg(args.offsets + group), b = __ldg(args.offsets + group + 1);
        lo = max(0, min(a, args.rows));
        hi = max(0, min(b, args.rows));
        if ((a != lo || b != hi || hi < lo) && threadIdx.x == 0) record_status(args.status, kStatusBadIndex);
    }
    if (hi <= lo) return; // the whole cluster: no rows in this group

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* part = reinterpret_cast<float*>(smem + STAGES * RS::STAGE_BYTES); // [TN][128]
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * RS::STAGE_BYTES + RS::PART_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + 1;
    uint64_t* drain = tempty + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0)
    {
        for (int s = 0; s < STAGES; s++)
        {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(tfull, 1);
        mbar_init(tempty, 4);
        mbar_init(drain, 1);
        *abort_flag = 0;
        *tmem_slot = 0;
        fence_mbarrier_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_w);
    }
    __syncthreads();
    if (warp == 1) tmem_alloc(tmem_slot, RS::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int kb0 = (int)((int64_t)args.num_kb * rank / S);
    const int kb1 = (int)((int64_t)args.num_kb * (rank + 1) / S);
    const int tiles = (hi - lo + TN - 1) / TN; // the same in every CTA of the cluster
    int stage = 0;
    uint32_t phase = 0, issued = 0, last_phase = 0;
    for (int t = 0; t < tiles; t++)
    {
        const int row0 = lo + t * TN;
        const int live = min(TN, hi - row0);
        if (warp == 0)
        {
            if (lane == 0)
            {
                for (int kb = kb0; kb < kb1; kb++)
                {
                    if (!mbar_wait<true>(&empty[stage], phase ^ 1, abort_flag, args.status)) break;
                    uint8_t* sw = smem + stage * RS::STAGE_BYTES;
                    mbar_arrive_expect_tx(&full[stage], RS::STAGE_BYTES);
                    tma_load_2d(sw, &tmap_w, &full[stage], kb * BK, group * args.N + n0);
                    tma_load_2d(sw + RS::W_BYTES, &tmap_a, &full[stage], kb * BK, row0);
                    issued |= 1u << stage;
                    last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == STAGES)
                    {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            __syncwarp();
        }
        else if (warp == 1)
        {
            if (lane == 0 && mbar_wait<true>(tempty, (t & 1) ^ 1, abort_flag, args.status))
            {
                tc_fence_after();
                bool ok = true;
                for (int kb = kb0; kb < kb1 && ok; kb++)
                {
                    ok = mbar_wait<true>(&full[stage], phase, abort_flag, args.status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t w_addr = smem_u32(smem + stage * RS::STAGE_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / 16; k++)
                        umma_bf16(tmem_base, umma_desc_sw128(w_addr + k * 32, 16, 1024),
                                  umma_desc_sw128(w_addr + RS::W_BYTES + k * 32, 16, 1024), RS::IDESC,
                                  kb > kb0 || k > 0);
                    umma_commit(&empty[stage]);
                    if (++stage == STAGES)
                    {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (ok) umma_commit(tfull);
            }
            __syncwarp();
        }
        else
        {
            int ok = 0;
            if (lane == 0) ok = mbar_wait<true>(tfull, t & 1, abort_flag, args.status) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (ok)
            {
                __syncwarp();
                tc_fence_after();
                const int f = (warp & 3) * 32 + lane;
                const uint32_t t_row = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
                for (int c = 0; c < live; c += 32)
                {
                    uint32_t v[32];
                    tmem_ld32(t_row + c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (c + j < live) part[(c + j) * 128 + f] = __uint_as_float(v[j]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty);
            }
        }
        __syncwarp();
        if (S > 1)
            cluster_sync();
        if (warp >= 2 && !*abort_flag)
        {
            const int f = (warp & 3) * 32 + lane;
            const int n = n0 + f;
            if (n < args.N)
            {
                const float b = args.bias ? __ldg(args.bias + (int64_t)group * args.N + n) : 0.f;
                const float gt = args.gate ? __ldg(args.gate + (int64_t)group * args.N + n) : 1.f;
                for (int r = rank; r < live; r += S)
                {
                    float x[1] = {0.f};
                    if (S > 1)
                    {
                        for (int k = 0; k < S; k++) x[0] += ld_cluster_f32(mapa_shared(part + r * 128 + f, k));
                    }
                    else
                        x[0] = part[r * 128 + f]; // this thread's own
                    x[0] += b;
                    activate<1>(x, args.act);
                    x[0] *= gt;
                    const int64_t row = row0 + r;
                    if (args.out_f32)
                    {
                        if (args.residual)
                            x[0] += static_cast<const float*>(args.residual)[row * args.residual_ld + n];
                        static_cast<float*>(args.out)[row * args.out_ld + n] = x[0];
                    }
                    else
                    {
                        if (args.residual)
                            x[0] += __bfloat162float(
                                static_cast<const __nv_bfloat16*>(args.residual)[row * args.residual_ld + n]);
                        static_cast<__nv_bfloat16*>(args.out)[row * args.out_ld + n] = __float2bfloat16_rn(x[0]);
                    }
                }
            }
        }
        __syncwarp();
        if (S > 1) cluster_sync(); // the parts are read before the next rows' overwrite them, or the CTA exits
    }
    if (warp == 0 && lane == 0 && *abort_flag)
        for (int s = 0; s < STAGES; s++)
            if ((issued >> s) & 1) drain_wait(&full[s], (last_phase >> s) & 1);
    if (warp == 1 && lane == 0)
    {
        umma_commit(drain);
        drain_wait(drain, 0);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem_base, RS::TMEM_COLS);
}

// ---------------------------------------------------------------- host
cudaLaunchConfig_t cluster_config(cudaLaunchAttribute* attr, int cluster, unsigned grid, int threads, size_t smem,
                                  cudaStream_t stream)
{
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

struct Operands
{
    const void* A;
    int64_t lda;
    const void* W;
    int64_t ldw;
};

template <int CTAS, int BN, int R>
int launch_tiles(Context& ctx, const Operands& o, LinearArgs a)
{
    using TL = TileShape<CTAS, BN, R>;
    auto kernel = linear_tile_kernel<CTAS, BN, R>;
    CUtensorMap ta, tw, to, tr;
    int r = make_tmap_bf16_2d(&ta, o.A, a.K, a.rows, (uint64_t)o.lda * 2, BK, BM);
    if (r == S2_OK)
        r = make_tmap_bf16_2d(&tw, o.W, a.K, (uint64_t)a.groups * a.N, (uint64_t)o.ldw * 2, BK, BN / CTAS);
    if (r != S2_OK) return r;
    const int esz = a.out_f32 ? 4 : 2;
    a.tma_out = make_tmap_2d(&to, a.out, a.out_f32, a.N, a.rows, (uint64_t)a.out_ld * esz, 128 / esz, 32) == S2_OK;
    if (!a.tma_out) to = ta;
    a.tma_res = a.residual && make_tmap_2d(&tr, a.residual, a.out_f32, a.N, a.rows, (uint64_t)a.residual_ld * esz,
                                           128 / esz, 32) == S2_OK;
    if (!a.tma_res) tr = ta;
    a.nblk = (a.N + BN - 1) / BN;
    a.stages = TL::stages(a.groups);
    a.group_m = a.K >= 8192 ? 1 : (a.N <= 4096 ? 8 : 16);
    const int64_t units = ((int64_t)a.rows / (CTAS * BM) + a.groups) * a.nblk; // at most
    if (units > 0x7fffffff) return S2_ERR_INVALID;
    const size_t smem = TL::fixed_bytes(a.groups) + (size_t)a.stages * TL::STAGE_BYTES;

    static std::atomic<uint64_t> configured{0}; // per instantiation and device
    static std::atomic<int> resident{0};        // CTAs or pairs at once, the same on every B200
    if (first_on_device(configured))
    {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit) != cudaSuccess)
            return S2_ERR_CUDA;
    }
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = cluster_config(attr, CTAS, CTAS, kTileThreads, smem, ctx.stream);
    int most = CTAS == 1 ? ctx.num_sms : resident.load();
    if (most == 0)
    {
        if (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess || most <= 0)
        {
            (void)cudaGetLastError();
            return S2_ERR_CUDA;
        }
        resident.store(most);
    }
    cfg.gridDim = dim3((unsigned)(CTAS * std::min<int64_t>(units, most)));
    if (cudaLaunchKernelEx(&cfg, kernel, ta, tw, to, tr, a) != cudaSuccess)
    {
        (void)cudaGetLastError();
        return S2_ERR_CUDA;
    }
    ctx.launches++;
    return S2_OK;
}

template <int TN>
int launch_rows(Context& ctx, const Operands& o, LinearArgs a)
{
    using RS = RowsShape<TN>;
    auto kernel = linear_rows_kernel<TN>;
    CUtensorMap ta, tw;
    int r = make_tmap_bf16_2d(&ta, o.A, a.K, a.rows, (uint64_t)o.lda * 2, BK, TN);
    if (r == S2_OK)
        r = make_tmap_bf16_2d(&tw, o.W, a.K, (uint64_t)a.groups * a.N, (uint64_t)o.ldw * 2, BK, 128);
    if (r != S2_OK) return r;
    a.nblk = (a.N + 127) / 128;
    const int64_t units = (int64_t)a.groups * a.nblk;
    // K parts: as many as the two CTAs a SM leave room for
    int s = 1;
    while (s < 8 && 2 * s <= a.num_kb && units * 2 * s <= 2 * ctx.num_sms) s *= 2;
    if (units * s > 0x7fffffff) return S2_ERR_INVALID;
    a.cluster = s;
    static std::atomic<uint64_t> configured{0};
    if (first_on_device(configured))
    {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RS::SMEM_BYTES) != cudaSuccess)
            return S2_ERR_CUDA;
    }
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg =
        cluster_config(attr, s, (unsigned)(units * s), kRowsThreads, RS::SMEM_BYTES, ctx.stream);
    if (cudaLaunchKernelEx(&cfg, kernel, ta, tw, a) != cudaSuccess)
    {
        (void)cudaGetLastError();
        return S2_ERR_CUDA;
    }
    ctx.launches++;
    return S2_OK;
}

int run_linear(s2_context* ctx, int rows, int groups, const int* offsets, int N, int K, const void* A, int64_t lda,
               const void* W, int64_t ldw, const s2_linear_epilogue* epi, int out_dtype, void* out, int64_t ldo)
{
    static const s2_linear_epilogue kNone = {S2_ACT_NONE, nullptr, nullptr, nullptr, 0};
    if (!epi) epi = &kNone;
    if (!ctx || rows < 0 || groups <= 0 || groups > kMaxGroups || N <= 0 || K <= 0 || K > (1 << 30) ||
        (int64_t)groups * N > 0x7fffffff - 256 || rows > 0x7fffffff - 256 || lda < K || ldw < K || ldo < N ||
        lda % 8 || ldw % 8 || (out_dtype != S2_DTYPE_F32 && out_dtype != S2_DTYPE_BF16) || epi->act < S2_ACT_NONE ||
        epi->act > S2_ACT_GELU_ERF || (epi->residual && epi->residual_ld < N))
        return S2_ERR_INVALID;
    if (rows == 0) return S2_OK;
    const uintptr_t mask = out_dtype == S2_DTYPE_F32 ? 3 : 1;
    if (!A || !W || !out || ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(W)) & 15) ||
        ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(epi->residual)) & mask) ||
        ((reinterpret_cast<uintptr_t>(epi->bias) | reinterpret_cast<uintptr_t>(epi->gate) |
          reinterpret_cast<uintptr_t>(offsets)) & 3))
        return S2_ERR_INVALID;
    // a residual in place is read element by element before its result is written
    if (epi->residual == out && epi->residual_ld != ldo) return S2_ERR_INVALID;
    Context& c = ctx->c;
    if (cudaSetDevice(c.device) != cudaSuccess) return S2_ERR_CUDA;
    LinearArgs a = {};
    a.rows = rows;
    a.N = N;
    a.K = K;
    a.groups = groups;
    a.num_kb = (K + BK - 1) / BK;
    a.offsets = offsets;
    a.act = epi->act;
    a.bias = epi->bias;
    a.gate = epi->gate;
    a.residual = epi->residual;
    a.residual_ld = epi->residual_ld;
    a.out = out;
    a.out_ld = ldo;
    a.out_f32 = out_dtype == S2_DTYPE_F32;
    a.status = c.status;
    const Operands o = {A, lda, W, ldw};
    const double osz = (a.out_f32 ? 4.0 : 2.0) * (a.residual ? 2 : 1);
    ProfileScope prof(c, K_GEMM, 2.0 * rows * N * K,
                      ((double)rows * K + (double)groups * N * K) * 2.0 + (double)rows * N * osz);
    const int mean_rows = (rows + groups - 1) / groups;
    if (mean_rows <= 16) return launch_rows<16>(c, o, a);
    if (mean_rows <= 32) return launch_rows<32>(c, o, a);
    if (mean_rows <= 64) return launch_rows<64>(c, o, a);
    const int64_t pair_tiles = ((int64_t)rows / 256 + 1) * ((N + 255) / 256);
    if (N > 128 && pair_tiles >= c.num_sms / 2) return launch_tiles<2, 256, 2>(c, o, a);
    return launch_tiles<1, 128, 3>(c, o, a);
}

} // namespace

} // namespace s2

extern "C" {

int s2_linear(s2_context* ctx, int M, int N, int K, const void* A, int64_t lda, const void* W, int64_t ldw,
              const s2_linear_epilogue* epilogue, int out_dtype, void* out, int64_t ldo)
{
    return s2::run_linear(ctx, M, 1, nullptr, N, K, A, lda, W, ldw, epilogue, out_dtype, out, ldo);
}

int s2_grouped_linear(s2_context* ctx, int rows, int groups, const int* offsets, int N, int K, const void* A,
                      int64_t lda, const void* W, int64_t ldw, const s2_linear_epilogue* epilogue, int out_dtype,
                      void* out, int64_t ldo)
{
    if (!offsets) return S2_ERR_INVALID;
    return s2::run_linear(ctx, rows, groups, offsets, N, K, A, lda, W, ldw, epilogue, out_dtype, out, ldo);
}

} // extern "C"
