// Linear and grouped linear on sm_100a:
//   out[r] = residual[r] + gate[g] * act(A[r] W[g]^T + bias[g]),  offsets[g] <= r < offsets[g + 1]
// (s2_linear is the one-group form).  Two kernels:
//   * linear_tile_kernel: output tiles of 128 rows a CTA (or 256 rows a CTA
//     pair), persistent, for many rows;
//   * linear_rows_kernel: 128 output features a CTA against a few rows, K
//     split over a thread-block cluster, for few rows a group.
#include <algorithm>
#include <cmath>
#include <type_traits>

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

// The tensor core adds into its fp32 accumulator without rounding to nearest:
// an fp32 result is off by 6.2e-8 of itself for each K block in one sum (1.1e-5
// over K = 10,240).  Where the result is fp32, sums of at most kChunk blocks
// (8.7e-7, so that an activation's slope keeps it below 1e-6) are therefore
// added up in fp32 registers (or shared memory), each while the tensor core
// works on the next one: 21,658 x 2,560 x 10,240 with an fp32 residual takes 854
// us so (820 at 24 blocks, 867 at 12) and 782 in one sum.  The price is highest
// where K just passes one sum: x 1,024 203 us against 143.  A bf16 result rounds
// at 2^-9 and keeps one sum.
constexpr int kChunk = 14;

// Blocks of one sum: equal ones.
constexpr int chunk_blocks(int num_kb, bool out_f32)
{
    const int chunks = out_f32 ? (num_kb + kChunk - 1) / kChunk : 1;
    return (num_kb + chunks - 1) / chunks;
}

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
    int chunk_kb; // K blocks summed by the tensor core before the sum is taken over (see kChunk)
    int vec_out, vec_res; // linear_rows_kernel: four outputs / residuals at once
    int* status;
};

// v[j] = vec[n + j], 0 past N
template <int W>
__device__ __forceinline__ void load_columns(const float* vec, int n, int N, float (&v)[W])
{
    if (n + W <= N && (reinterpret_cast<uintptr_t>(vec + n) & 15) == 0)
    {
#pragma unroll
        for (int j = 0; j < W; j += 4)
        {
            const float4 b = __ldg(reinterpret_cast<const float4*>(vec + n + j));
            v[j] = b.x;
            v[j + 1] = b.y;
            v[j + 2] = b.z;
            v[j + 3] = b.w;
        }
    }
    else
    {
#pragma unroll
        for (int j = 0; j < W; j++) v[j] = n + j < N ? __ldg(vec + n + j) : 0.f;
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
// Bound by the tensor core: 21,658 x 7,680 x 2,560 in two groups takes 559 us =
// 1,523 TFLOP/s of the 1,701 that a library product reaches at full clock (682 us
// where power holds the clock down).  Short K is bound by memory and by the
// epilogue that shares it: 288,000 x 256 x 512 with a residual 111 us = 5.3 TB/s
// of 6.45.
// Warps: TMA, MMA, then EW for the epilogue, in equal parts over the four TMEM
// lane quarters, each with its share of the columns.  Eight do where boxes
// leave by TMA; sixteen where the warps copy them, a chain of latencies that
// only more warps hide (21,247 x 409 x 303 in 56 groups, bf16 with a residual:
// 44 us against 85; but 117 against 110 where TMA does it: 288,000 x 256 x 512).
// Where a warp holds sums of the accumulator in registers (SUM) the eight begin
// at warp 4, so that setmaxnreg can give them what the first four do not need:
// 104 + 2 x 200 = 3 x 168 registers per thread and warpgroup, the 168 a thread
// that 384 threads are launched with.
constexpr int kSumRegs = 200, kOtherRegs = 104, kLaunchRegs = 168;
static_assert(kOtherRegs + 2 * kSumRegs == 3 * kLaunchRegs, "register split");
constexpr int first_epilogue_warp(bool sum)
{
    return sum ? 4 : 2;
}
constexpr int tile_threads(int EW, bool sum)
{
    return 32 * (first_epilogue_warp(sum) + EW);
}
template <int N>
__device__ __forceinline__ void regs_increase()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_decrease()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
constexpr int kBox = 4096; // 32 rows x 128 bytes

// CTAS = 2: a pair of CTAs (cluster of 2) computes 256 rows x BN columns with
// M = 256 MMAs, each holding its 128 rows of A and BN / 2 rows of W.
// R: boxes per epilogue warp.
template <int CTAS, int BN, int R, int EW>
struct TileShape
{
    static constexpr int W_BYTES = BN / CTAS * BK * 2;
    static constexpr int STAGE_BYTES = A_BYTES + W_BYTES;
    static constexpr int EPI_BYTES = EW * R * kBox;
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

// 32 lanes x 16 consecutive 32-bit columns -> 16 registers per thread.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// Byte of (row r, byte b) in a 128-byte-swizzled box.
__device__ __forceinline__ int box_at(int r, int b)
{
    return r * 128 + ((((b >> 4) ^ r) & 7) << 4) + (b & 15);
}

// Rows and columns that a tensor map cannot take (group ends inside a box,
// strides or bases off 16 bytes): the warp copies row by row, a 32-bit word a
// lane.  A bf16 row that begins off a word is shifted by one element between
// the lanes, and its first and last elements go by themselves.
__device__ __forceinline__ uint32_t box_word(const uint8_t* box, int r, int lane)
{
    return *reinterpret_cast<const uint32_t*>(box + box_at(r, lane * 4));
}
// Predicated accesses: written as branches, the three a bf16 row needs took
// 6,000 cycles a box instead of some 1,500.
__device__ __forceinline__ void st32_if(bool p, void* to, uint32_t v)
{
    asm volatile("{.reg .pred p; setp.ne.b32 p, %2, 0; @p st.global.b32 [%0], %1;}" ::"l"(to), "r"(v), "r"((int)p)
                 : "memory");
}
__device__ __forceinline__ void st16_if(bool p, void* to, uint32_t v)
{
    asm volatile("{.reg .pred p; setp.ne.b32 p, %2, 0; @p st.global.b16 [%0], %1;}" ::"l"(to), "h"((uint16_t)v),
                 "r"((int)p)
                 : "memory");
}
// 0 where p is false
__device__ __forceinline__ uint32_t ld32_if(bool p, const void* from)
{
    uint32_t v;
    asm volatile("{.reg .pred p; setp.ne.b32 p, %2, 0; mov.b32 %0, 0; @p ld.global.b32 %0, [%1];}"
                 : "=r"(v)
                 : "l"(from), "r"((int)p)
                 : "memory");
    return v;
}
__device__ __forceinline__ uint32_t ld16_if(bool p, const void* from)
{
    uint16_t v;
    asm volatile("{.reg .pred p; setp.ne.b32 p, %2, 0; mov.b16 %0, 0; @p ld.global.b16 %0, [%1];}"
                 : "=h"(v)
                 : "l"(from), "r"((int)p)
                 : "memory");
    return v;
}

__device__ __forceinline__ void box_to_global(const uint8_t* box, float* out, int64_t ld, int rows, int cols, int lane)
{
    constexpr int B = 8;
    out += lane;
    for (int r0 = 0; r0 < rows; r0 += B)
    {
        uint32_t w[B];
#pragma unroll
        for (int i = 0; i < B; i++) w[i] = box_word(box, r0 + i, lane);
#pragma unroll
        for (int i = 0; i < B; i++, out += ld) st32_if(lane < cols && r0 + i < rows, out, w[i]);
    }
}
__device__ __forceinline__ void box_to_global(const uint8_t* box, uint16_t* out, int64_t ld, int rows, int cols, int lane)
{
    constexpr int B = 8;
    cols = min(cols, 64);
    for (int r0 = 0; r0 < rows; r0 += B)
    {
        uint32_t w[B];
#pragma unroll
        for (int i = 0; i < B; i++) w[i] = box_word(box, r0 + i, lane);
#pragma unroll
        for (int i = 0; i < B; i++, out += ld)
        {
            const uint32_t next = __shfl_down_sync(0xffffffffu, w[i], 1);
            const int off = (reinterpret_cast<uintptr_t>(out) >> 1) & 1;
            const uint32_t v = __byte_perm(w[i], next, off ? 0x5432 : 0x3210);
            const int e = 2 * lane + off; // the word's first element
            const bool in = r0 + i < rows;
            st32_if(in && e + 1 < cols, out + e, v);
            st16_if(in && e + 1 == cols, out + e, v);
            st16_if(in && off && lane == 0, out, w[i]);
        }
    }
}

// Residual rows -> the box.
__device__ __forceinline__ void global_to_box(uint8_t* box, const float* in, int64_t ld, int rows, int cols, int lane)
{
    constexpr int B = 16;
    in += lane;
    for (int r0 = 0; r0 < rows; r0 += B)
    {
        uint32_t w[B];
#pragma unroll
        for (int i = 0; i < B; i++, in += ld) w[i] = ld32_if(lane < cols && r0 + i < rows, in);
#pragma unroll
        for (int i = 0; i < B; i++) *reinterpret_cast<uint32_t*>(box + box_at(r0 + i, lane * 4)) = w[i];
    }
}
__device__ __forceinline__ void global_to_box(uint8_t* box, const uint16_t* in, int64_t ld, int rows, int cols, int lane)
{
    constexpr int B = 8;
    cols = min(cols, 64);
    for (int r0 = 0; r0 < rows; r0 += B)
    {
        uint32_t w[B], one[B]; // one: a last odd element, or (lane 0) the first of a row off a word
        const uint16_t* row = in;
#pragma unroll
        for (int i = 0; i < B; i++, row += ld)
        {
            const int off = (reinterpret_cast<uintptr_t>(row) >> 1) & 1;
            const int e = 2 * lane + off;
            const bool live = r0 + i < rows;
            w[i] = ld32_if(live && e + 1 < cols, row + e);
            w[i] |= ld16_if(live && e + 1 == cols, row + e);
            one[i] = ld16_if(live && off && lane == 0, row);
        }
#pragma unroll
        for (int i = 0; i < B; i++, in += ld)
        {
            const uint32_t before = __shfl_up_sync(0xffffffffu, w[i], 1);
            const int off = (reinterpret_cast<uintptr_t>(in) >> 1) & 1;
            const uint32_t shifted = (lane == 0 ? one[i] : before >> 16) | w[i] << 16;
            *reinterpret_cast<uint32_t*>(box + box_at(r0 + i, lane * 4)) = off ? shifted : w[i];
        }
    }
}
__device__ __forceinline__ void prefetch_row(const void* from, const void* to)
{
    for (uintptr_t p = reinterpret_cast<uintptr_t>(from) & ~uintptr_t(127); p < reinterpret_cast<uintptr_t>(to); p += 128)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// W accumulator columns of this lane's row -> the result, in the box (srow: the
// lane's row of it; col: the first column's place in the box).
template <int W>
__device__ __forceinline__ void finish(const LinearArgs& a, const float* x0, const float* bias, const float* gate, int n,
                                       uint8_t* srow, int sw, int col)
{
    float x[W], v[W];
#pragma unroll
    for (int j = 0; j < W; j++) x[j] = x0[j];
    if (bias)
    {
        load_columns<W>(bias, n, a.N, v);
#pragma unroll
        for (int j = 0; j < W; j++) x[j] += v[j];
    }
    activate<W>(x, a.act);
    if (gate)
    {
        load_columns<W>(gate, n, a.N, v);
#pragma unroll
        for (int j = 0; j < W; j++) x[j] *= v[j];
    }
    if (a.out_f32)
    {
#pragma unroll
        for (int j = 0; j < W; j += 4)
        {
            float4* p = reinterpret_cast<float4*>(srow + ((((col + j) >> 2) ^ sw) << 4));
            float4 o = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
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
        for (int j = 0; j < W; j += 8)
        {
            uint4* p = reinterpret_cast<uint4*>(srow + ((((col + j) >> 3) ^ sw) << 4));
            if (a.residual)
            {
                const uint4 r = *p;
                const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int e = 0; e < 4; e++)
                {
                    const float2 f = unpack_bf16x2(rw[e]);
                    x[j + 2 * e] += f.x;
                    x[j + 2 * e + 1] += f.y;
                }
            }
            *p = make_uint4(pack_bf16x2(x[j], x[j + 1]), pack_bf16x2(x[j + 2], x[j + 3]),
                            pack_bf16x2(x[j + 4], x[j + 5]), pack_bf16x2(x[j + 6], x[j + 7]));
        }
    }
}

// x = the i-th sixteen of N * 16 sums in registers
template <int N>
__device__ __forceinline__ void take_piece(const float (&sum)[N / 2][32], int i, float (&x)[16])
{
    auto take = [&](auto k) {
        constexpr int K = decltype(k)::value;
        if constexpr (K < N)
        {
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = sum[K / 2][16 * (K % 2) + j];
        }
    };
    switch (i)
    {
    case 0: take(std::integral_constant<int, 0>()); break;
    case 1: take(std::integral_constant<int, 1>()); break;
    case 2: take(std::integral_constant<int, 2>()); break;
    case 3: take(std::integral_constant<int, 3>()); break;
    case 4: take(std::integral_constant<int, 4>()); break;
    case 5: take(std::integral_constant<int, 5>()); break;
    case 6: take(std::integral_constant<int, 6>()); break;
    default: take(std::integral_constant<int, N - 1>()); break;
    }
}

// Epilogue of one warp over all of the CTA's units.  Boxes (32 rows x 128
// bytes of output) run in a fixed sequence; each is combined in one of the
// warp's R shared-memory boxes and written by one TMA store.  A residual box is
// TMA-loaded R - 1 boxes ahead (R = 1: as soon as the box before has left) into
// the slot its result will leave from; where
// TMA cannot take it the warp copies it.  Either way a unit's residual is asked
// for in L2 a unit ahead.  SUM (fp32 results,
// long K): the accumulator's chunks are added up in registers first.
template <int CTAS, int BN, int R, int EW, bool SUM>
__device__ __forceinline__ void tile_epilogue(const LinearArgs& a, const CUtensorMap* tmap_out,
                                              const CUtensorMap* tmap_res, UnitWalk<CTAS * BM, BN> walk,
                                              UnitWalk<CTAS * BM, BN> ahead, int first_unit, int step, int units,
                                              int rank, uint8_t* stg, uint64_t* rfull, uint64_t* tfull,
                                              uint64_t* tempty, uint32_t tmem_base, int quarter, int part, int lane,
                                              volatile int* abort_flag)
{
    constexpr int COLS = BN * 4 / EW; // of a unit, per warp
    constexpr int PIECE = EW > 8 ? 16 : 32; // columns at a time: by the registers there are
    const int esz = SUM || a.out_f32 ? 4 : 2;
    const int box_cols = 128 / esz;
    const int row_in = rank * BM + quarter * 32; // of the unit, this warp's first
    const int c_lo = part * COLS, c_hi = c_lo + COLS;
    const int sw = lane & 7;
    const bool copied = a.residual && !a.tma_res;
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
    // a unit's residual goes to L2 a unit ahead
    UnitWalk<CTAS * BM, BN> far = ahead;
    auto prefetch_unit = [&](int u) {
        if (!a.residual || u >= units) return;
        const Unit p = far.decode(a, u);
        const int row = p.m0 + row_in;
        if (a.tma_res)
        {
            if (lane == 0 && row < p.end)
                for (int c = c_lo; c < c_hi && p.n0 + c < a.N; c += box_cols) tma_prefetch_l2_2d(tmap_res, p.n0 + c, row);
        }
        else if (row + lane < p.end && p.n0 + c_lo < a.N)
        {
            const uint8_t* line = static_cast<const uint8_t*>(a.residual) + (int64_t)(row + lane) * a.residual_ld * esz;
            prefetch_row(line + (int64_t)(p.n0 + c_lo) * esz, line + (int64_t)min(p.n0 + c_hi, a.N) * esz);
        }
    };
    prefetch_unit(first_unit);
    if (a.tma_res && lane == 0)
        for (int i = 0; i < (R > 1 ? R - 1 : 1); i++) issue_load();

    int q = 0, acc = 0;
    uint32_t acc_phase = 0;
    auto wait_acc = [&]() {
        const bool w = mbar_wait_warp<true>(&tfull[acc], acc_phase, abort_flag, a.status);
        tc_fence_after();
        return w;
    };
    auto release_acc = [&]() {
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
    };
    bool ok = true;
    for (int u = first_unit; u < units && ok; u += step)
    {
        const Unit un = walk.decode(a, u);
        const int row0 = un.m0 + row_in;
        const int live_rows = min(32, un.end - row0);
        const float* bias = a.bias ? a.bias + (int64_t)un.group * a.N : nullptr;
        const float* gate = a.gate ? a.gate + (int64_t)un.group * a.N : nullptr;
        const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
        prefetch_unit(u + step);

        // box q of the warp, columns [c, c + box_cols) of the unit: from its
        // slot's release to its store
        auto open_box = [&](int c) {
            const int slot = q % R;
            uint8_t* box = stg + slot * kBox;
            if (a.tma_res) return mbar_wait_warp<true>(&rfull[slot], (uint32_t)(q / R) & 1u, abort_flag, a.status);
            if (lane == 0) bulk_wait_read<R - 1>(); // this slot's previous store has read it
            __syncwarp();
            if (copied)
            {
                const int64_t at = (int64_t)row0 * a.residual_ld + un.n0 + c;
                const int cols = a.N - un.n0 - c;
                if (esz == 4)
                    global_to_box(box, static_cast<const float*>(a.residual) + at, a.residual_ld, live_rows, cols, lane);
                else
                    global_to_box(box, static_cast<const uint16_t*>(a.residual) + at, a.residual_ld, live_rows, cols, lane);
                __syncwarp();
            }
            return true;
        };
        auto close_box = [&](int c) {
            uint8_t* box = stg + (q % R) * kBox;
            const int n = un.n0 + c;
            const int live_cols = min(box_cols, a.N - n);
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
                    // the store of box q-1 (of q itself if there is but one) has
                    // read its slot, which takes the next load
                    bulk_wait_read<(R > 1 ? 1 : 0)>();
                    issue_load();
                }
            }
            q++;
        };

        if constexpr (SUM)
        {
            float sum[COLS / 32][32];
#pragma unroll
            for (int i = 0; i < COLS / 32; i++)
#pragma unroll
                for (int j = 0; j < 32; j++) sum[i][j] = 0.f;
            for (int kb = 0; kb < a.num_kb; kb += a.chunk_kb)
            {
                ok = wait_acc();
                if (!ok) break;
                const uint32_t t_row = t_lane + acc * BN + c_lo;
#pragma unroll
                for (int i = 0; i < COLS / 16; i++)
                {
                    uint32_t v[16];
                    tmem_ld16(t_row + 16 * i, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; j++) sum[i / 2][16 * (i % 2) + j] += __uint_as_float(v[j]);
                }
                release_acc();
            }
            if (!ok) break;
            // one body for all pieces, which fits the instruction cache with its
            // activations (unrolled, 21,658 x 2,560 x 2,560 with an fp32 residual
            // takes 290 us instead of 265, with erf GELU 431 instead of 297; the four
            // of a 128-wide tile, 5,000 x 2,560 x 1,024 in 64 groups, 98 instead of 95,
            // without the residual 77 and 79): `sum` stays in registers, a jump takes
            // out a piece
#pragma unroll 1
            for (int i = 0; i < COLS / 16; i++)
            {
                const int c = c_lo + 16 * i;
                if (i % 2 == 0)
                {
                    if (un.n0 + c >= a.N || live_rows <= 0) break;
                    ok = open_box(c);
                    if (!ok) break;
                }
                float x[16];
                take_piece<COLS / 16>(sum, i, x);
                finish<16>(a, x, bias, gate, un.n0 + c, stg + (q % R) * kBox + lane * 128, sw, 16 * (i % 2));
                if (i % 2 == 1) close_box(c - 16);
            }
        }
        else
        {
            ok = wait_acc();
            if (!ok) break;
            const uint32_t t_row = t_lane + acc * BN;
#pragma unroll 1
            for (int c = c_lo; c < c_hi && un.n0 + c < a.N && live_rows > 0; c += box_cols)
            {
                ok = open_box(c);
                if (!ok) break;
#pragma unroll 1
                for (int k = 0; k < box_cols; k += PIECE)
                {
                    uint32_t v[PIECE];
                    if constexpr (PIECE == 32)
                        tmem_ld32(t_row + c + k, v);
                    else
                        tmem_ld16(t_row + c + k, v);
                    tmem_ld_wait();
                    float x[PIECE];
#pragma unroll
                    for (int j = 0; j < PIECE; j++) x[j] = __uint_as_float(v[j]);
                    finish<PIECE>(a, x, bias, gate, un.n0 + c + k, stg + (q % R) * kBox + lane * 128, sw, k);
                }
                close_box(c);
            }
            if (!ok) break;
            release_acc();
        }
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

template <int CTAS, int BN, int R, int EW, bool SUM>
__global__ void __launch_bounds__(tile_threads(EW, SUM), 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                       const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ CUtensorMap tmap_res,
                       const LinearArgs args)
{
    using TL = TileShape<CTAS, BN, R, EW>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int stages = args.stages;
    uint8_t* epi_stage = smem + stages * TL::STAGE_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(epi_stage + TL::EPI_BYTES);
    uint64_t* empty = full + TL::MAX_STAGES;
    uint64_t* tfull = empty + TL::MAX_STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint64_t* rfull = drain + 1; // [EW][R]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rfull + EW * R);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((2 * TL::MAX_STAGES + 5 + EW * R) * 8 + 8 <= 512, "barriers");
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
            mbar_init(&tempty[b], CTAS * EW);
        }
        mbar_init(drain, 1);
        for (int i = 0; i < EW * R; i++) mbar_init(&rfull[i], 1);
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

    // each role's code follows its own setmaxnreg, so that the compiler gives
    // it that many registers
    if (warp >= first_epilogue_warp(SUM))
    {
        if constexpr (SUM) regs_increase<kSumRegs>();
        const int e = warp - first_epilogue_warp(SUM);
        tile_epilogue<CTAS, BN, R, EW, SUM>(args, &tmap_out, &tmap_res, walk, walk, unit0, step, units, rank,
                                        epi_stage + e * R * kBox, rfull + e * R, tfull, tempty, tmem_base, warp & 3,
                                        e >> 2, lane, abort_flag);
    }
    else
    {
    if constexpr (SUM) regs_decrease<kOtherRegs>();
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
                bool ok = true;
                for (int kb0 = 0; kb0 < args.num_kb && ok; kb0 += args.chunk_kb)
                {
                    ok = mbar_wait<true>(&tempty[acc], acc_phase ^ 1, abort_flag, args.status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d_tmem = tmem_base + acc * BN;
                    const int kb1 = min(args.num_kb, kb0 + args.chunk_kb);
                    for (int kb = kb0; kb < kb1; kb++)
                    {
                        ok = mbar_wait<true>(&full[stage], phase, abort_flag, args.status);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t a_addr = smem_u32(smem + stage * TL::STAGE_BYTES);
                        const uint32_t b_addr = a_addr + A_BYTES;
#pragma unroll
                        for (int k = 0; k < BK / 16; k++)
                        {
                            const uint64_t ad = umma_desc_sw128(a_addr + k * 32, 16, 1024);
                            const uint64_t bd = umma_desc_sw128(b_addr + k * 32, 16, 1024);
                            if (CTAS == 2)
                                umma_bf16_pair(d_tmem, ad, bd, TL::IDESC, kb > kb0 || k > 0);
                            else
                                umma_bf16(d_tmem, ad, bd, TL::IDESC, kb > kb0 || k > 0);
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
                if (!ok) break;
            }
            // every MMA completes (in both CTAs) before TMEM is released
            if (CTAS == 2)
                umma_commit_pair(drain, 0x3);
            else
                umma_commit(drain);
        }
        if (lane == 0) drain_wait(drain, 0);
    }
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
// on the run), applies the epilogue and stores: a warp takes one row's 128
// features, four a lane.  1 x 2,560 x 2,560 takes 7.0 us (2.0 at the memory's
// rate: the set-up, one trip to memory and two cluster barriers are the rest), 58 x
// 10,240 x 2,560 16.0 (8.4), 64 groups of 2,048 x 1,024 at 2 rows each 53 = 5.1
// TB/s.
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
    static constexpr int ACC_COLS = TN < 32 ? 32 : TN;
    static constexpr int TMEM_COLS = 2 * ACC_COLS; // two accumulators
    static_assert((2 * STAGES + 5) * 8 + 8 <= 256, "barriers");
};

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// Four residuals of a row from column n on, as they lie in memory.
struct Res4
{
    float v[4];
    __device__ void load(const LinearArgs& a, int64_t row, int n, bool four)
    {
        if (a.out_f32)
        {
            const float* p = static_cast<const float*>(a.residual) + row * a.residual_ld + n;
            if (four && a.vec_res)
            {
                const float4 q = *reinterpret_cast<const float4*>(p);
                v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
            }
            else
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = __uint_as_float(ld32_if(n + e < a.N, p + e));
        }
        else
        {
            const uint16_t* p = static_cast<const uint16_t*>(a.residual) + row * a.residual_ld + n;
            if (four && a.vec_res)
            {
                const uint2 q = *reinterpret_cast<const uint2*>(p);
                const float2 lo = unpack_bf16x2(q.x), hi = unpack_bf16x2(q.y);
                v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
            }
            else
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = __uint_as_float(ld16_if(n + e < a.N, p + e) << 16);
        }
    }
};

__device__ __forceinline__ void store4(const LinearArgs& a, int64_t row, int n, bool four, const float (&y)[4])
{
    if (a.out_f32)
    {
        float* o = static_cast<float*>(a.out) + row * a.out_ld + n;
        if (four && a.vec_out)
            *reinterpret_cast<float4*>(o) = make_float4(y[0], y[1], y[2], y[3]);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) st32_if(n + e < a.N, o + e, __float_as_uint(y[e]));
    }
    else
    {
        uint16_t* o = static_cast<uint16_t*>(a.out) + row * a.out_ld + n;
        const uint32_t lo = pack_bf16x2(y[0], y[1]), hi = pack_bf16x2(y[2], y[3]);
        if (four && a.vec_out)
            *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) st16_if(n + e < a.N, o + e, (e < 2 ? lo : hi) >> 16 * (e & 1));
    }
}

// Rows rank, rank + S, ... of the unit: the S parts added, the epilogue, the
// store.  Several rows at once, their loads first, so that these are in flight
// together.
template <int S>
__device__ __forceinline__ void rows_finish(const LinearArgs& a, const float* part, int rank, int warp, int lane,
                                            int group, int64_t row0, int live, int n0)
{
    constexpr int B = S > 4 ? 2 : 4; // rows at once
    const int n = n0 + lane * 4;
    if (n >= a.N) return;
    const bool four = n + 4 <= a.N;
    float b[4], g[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
    {
        b[e] = a.bias && n + e < a.N ? __ldg(a.bias + (int64_t)group * a.N + n + e) : 0.f;
        g[e] = a.gate && n + e < a.N ? __ldg(a.gate + (int64_t)group * a.N + n + e) : 1.f;
    }
    uint32_t at[S];
#pragma unroll
    for (int k = 0; k < S; k++) at[k] = S > 1 ? mapa_shared(part + lane * 4, k) : smem_u32(part + lane * 4);
    for (int r = rank + S * warp; r < live; r += 4 * S * B)
    {
        Res4 res[B];
        float x[B][4] = {};
        if (a.residual)
#pragma unroll
            for (int i = 0; i < B; i++)
                if (r + 4 * S * i < live) res[i].load(a, row0 + r + 4 * S * i, n, four);
#pragma unroll
        for (int i = 0; i < B; i++)
        {
            const int rr = min(r + 4 * S * i, live - 1); // a row past the end is read again and not used
            float4 v[S];
#pragma unroll
            for (int k = 0; k < S; k++) v[k] = ld_cluster_v4(at[k] + rr * 512);
#pragma unroll
            for (int k = 0; k < S; k++)
            {
                x[i][0] += v[k].x;
                x[i][1] += v[k].y;
                x[i][2] += v[k].z;
                x[i][3] += v[k].w;
            }
        }
#pragma unroll
        for (int i = 0; i < B; i++)
        {
            if (r + 4 * S * i >= live) break;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = x[i][e] + b[e];
            activate<4>(y, a.act);
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = a.residual ? fmaf(y[e], g[e], res[i].v[e]) : y[e] * g[e];
            store4(a, row0 + r + 4 * S * i, n, four, y);
        }
    }
}

// Row tile j of those behind the first of their groups, in the groups' order:
// its group and its number there (0 if there are fewer).  Each warp looks by
// itself, a lane over a run of groups.
template <int TN>
__device__ __forceinline__ int find_row_tile(const LinearArgs& a, int j, int& group)
{
    const int lane = threadIdx.x & 31;
    const int run = (a.groups + 31) / 32, first = lane * run;
    auto at = [&](int g) { return max(0, min(__ldg(a.offsets + min(g, a.groups)), a.rows)); };
    int own = 0;
    for (int i = 0, lo = at(first); i < run; i++)
    {
        const int hi = at(first + i + 1);
        own += max(0, hi - lo - 1) / TN;
        lo = hi;
    }
    int upto = own;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1)
    {
        const int o = __shfl_up_sync(0xffffffffu, upto, m);
        if (lane >= m) upto += o;
    }
    const unsigned past = __ballot_sync(0xffffffffu, j < upto);
    if (!past) return 0;
    const int owner = __ffs(past) - 1;
    int g = first, left = j - (upto - own);
    if (lane == owner)
        for (int i = 0, lo = at(g); i < run; i++, g++)
        {
            const int hi = at(g + 1), more = max(0, hi - lo - 1) / TN;
            if (left < more) break;
            left -= more;
            lo = hi;
        }
    group = __shfl_sync(0xffffffffu, g, owner);
    return 1 + __shfl_sync(0xffffffffu, left, owner);
}

template <int TN, int S>
__global__ void __launch_bounds__(kRowsThreads, 2)
    linear_rows_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                       const LinearArgs args)
{
    using RS = RowsShape<TN>;
    constexpr int STAGES = RS::STAGES;
    const int rank = S > 1 ? (int)cluster_ctarank() : 0;
    // Units: row tiles, each over the blocks of 128 features.  With offsets: each
    // group's first row tile, then some CTAs (or clusters) that share the others,
    // whose number the host does not know, in turn.  What they find is the same in
    // every CTA of a cluster; without rows they return at once.
    const int unit = blockIdx.x / S;
    const int entry = unit / args.nblk;
    const int n0 = (unit - entry * args.nblk) * 128;
    const int sharing = args.offsets ? (int)(gridDim.x / S) / args.nblk - args.groups : 0;
    int other = args.offsets ? entry - args.groups : -1;
    int group = 0, row0 = 0, live = 0;
    auto locate = [&]() {
        int tile = entry, end = args.rows;
        row0 = 0;
        if (args.offsets)
        {
            group = entry;
            tile = 0;
            if (other >= 0)
            {
                tile = find_row_tile<TN>(args, other, group);
                if (tile == 0) return false;
            }
            const int a = __ldg(args.offsets + group), b = __ldg(args.offsets + group + 1);
            row0 = max(0, min(a, args.rows));
            end = max(0, min(b, args.rows));
            if ((a != row0 || b != end || end < row0) && threadIdx.x == 0) record_status(args.status, kStatusBadIndex);
        }
        row0 += tile * TN;
        live = min(TN, end - row0);
        return live > 0;
    };
    if (!locate()) return;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* part = reinterpret_cast<float*>(smem + STAGES * RS::STAGE_BYTES); // [TN][128]
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * RS::STAGE_BYTES + RS::PART_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int kb0 = (int)((int64_t)args.num_kb * rank / S);
    const int kb1 = (int)((int64_t)args.num_kb * (rank + 1) / S);

    int stage = 0;
    uint32_t phase = 0, issued = 0, last_phase = 0;
    auto load = [&](int kb) {
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
    };
    int early = 0; // K blocks already sent for
    if (threadIdx.x == 0)
    {
        for (int s = 0; s < STAGES; s++)
        {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++)
        {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], 4);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        *tmem_slot = 0;
        fence_mbarrier_init();
        fence_proxy_async_smem();
        // the ring's first fill does not wait for the set-up below
        for (; early < STAGES && kb0 + early < kb1; early++) load(kb0 + early);
    }
    __syncthreads();
    if (warp == 1) tmem_alloc(tmem_slot, RS::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    int acc = 0;
    uint32_t acc_phase = 0;
    for (;;)
    {
        if (warp == 0)
        {
            if (lane == 0)
            {
                for (int kb = kb0 + early; kb < kb1; kb++)
                {
                    if (!mbar_wait<true>(&empty[stage], phase ^ 1, abort_flag, args.status)) break;
                    load(kb);
                }
                early = 0;
            }
            __syncwarp();
        }
        else if (warp == 1)
        {
            if (lane == 0)
            {
                bool ok = true;
                for (int c0 = kb0; c0 < kb1 && ok; c0 += args.chunk_kb)
                {
                    ok = mbar_wait<true>(&tempty[acc], acc_phase ^ 1, abort_flag, args.status);
                    if (!ok) break;
                    tc_fence_after();
                    const int c1 = min(kb1, c0 + args.chunk_kb);
                    for (int kb = c0; kb < c1; kb++)
                    {
                        ok = mbar_wait<true>(&full[stage], phase, abort_flag, args.status);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t w_addr = smem_u32(smem + stage * RS::STAGE_BYTES);
#pragma unroll
                        for (int k = 0; k < BK / 16; k++)
                            umma_bf16(tmem_base + acc * RS::ACC_COLS, umma_desc_sw128(w_addr + k * 32, 16, 1024),
                                      umma_desc_sw128(w_addr + RS::W_BYTES + k * 32, 16, 1024), RS::IDESC,
                                      kb > c0 || k > 0);
                        umma_commit(&empty[stage]);
                        if (++stage == STAGES)
                        {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                    if (!ok) break;
                    umma_commit(&tfull[acc]);
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1;
                }
            }
            __syncwarp();
        }
        else
        {
            const int f = (warp & 3) * 32 + lane;
            for (int c0 = kb0; c0 < kb1; c0 += args.chunk_kb)
            {
                if (!mbar_wait_warp<true>(&tfull[acc], acc_phase, abort_flag, args.status)) break;
                tc_fence_after();
                const uint32_t t_row = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + acc * RS::ACC_COLS;
#pragma unroll 1
                for (int c = 0; c < live; c += 32)
                {
                    uint32_t v[32];
                    tmem_ld32(t_row + c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < (TN < 32 ? TN : 32); j++)
                    {
                        float* p = part + (c + j) * 128 + f; // this thread's own until the cluster meets
                        *p = c0 > kb0 ? *p + __uint_as_float(v[j]) : __uint_as_float(v[j]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&tempty[acc]);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
        }
        __syncwarp();
        if (S > 1)
            cluster_sync();
        else
            __syncthreads();
        if (warp >= 2 && !*abort_flag) rows_finish<S>(args, part, rank, warp - 2, lane, group, row0, live, n0);
        __syncwarp();
        // the parts are read before the next rows' overwrite them, or the CTA exits
        if (S > 1)
            cluster_sync();
        else
            __syncthreads();
        if (other < 0) break;
        other += sharing;
        if (!locate()) break;
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

// Output and residual maps, where TMA can take them.
struct BoxMaps
{
    CUtensorMap out, res;
};

template <int CTAS, int BN, int R, int EW, bool SUM>
int launch_tiles(Context& ctx, const Operands& o, const BoxMaps& m, LinearArgs a)
{
    using TL = TileShape<CTAS, BN, R, EW>;
    auto kernel = linear_tile_kernel<CTAS, BN, R, EW, SUM>;
    CUtensorMap ta, tw;
    int r = make_tmap_bf16_2d(&ta, o.A, a.K, a.rows, (uint64_t)o.lda * 2, BK, BM);
    if (r == S2_OK)
        r = make_tmap_bf16_2d(&tw, o.W, a.K, (uint64_t)a.groups * a.N, (uint64_t)o.ldw * 2, BK, BN / CTAS);
    if (r != S2_OK) return r;
    a.nblk = (a.N + BN - 1) / BN;
    a.stages = TL::stages(a.groups);
    // M blocks that share a pass over W: sixteen where W is wide (16,384 x 8,192 x
    // 4,096: 684 us, against 737 for one; 8,000 x 10,240 x 8,192: 907 and 996), one
    // where a row of units is about a round of them anyway (21,658 x 2,560 x 10,240
    // with an fp32 residual: 848 us, against 867 for sixteen; x 2,560: 273 and 284;
    // 16,384 x 4,096 x 4,096: 341 and 345).
    a.group_m = a.N <= 4096 ? 1 : 16;
    a.chunk_kb = chunk_blocks(a.num_kb, SUM);
    const int64_t units = ((int64_t)a.rows / (CTAS * BM) + a.groups) * a.nblk; // at most
    if (units > 0x7fffffff) return S2_ERR_INVALID;
    const size_t smem = TL::fixed_bytes(a.groups) + (size_t)a.stages * TL::STAGE_BYTES;

    static std::atomic<uint64_t> configured{0}; // per instantiation and device
    static std::atomic<int> resident{0};        // CTAs or pairs at once, the same on every B200
    const int set = set_up_current_device(configured, [&] {
        cudaFuncAttributes f;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit) != cudaSuccess ||
            cudaFuncGetAttributes(&f, kernel) != cudaSuccess)
            return (int)S2_ERR_CUDA;
        // launched with fewer registers, setmaxnreg.inc would wait for good
        return SUM && f.numRegs != kLaunchRegs ? (int)S2_ERR_CUDA : (int)S2_OK;
    });
    if (set != S2_OK) return set;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = cluster_config(attr, CTAS, CTAS, tile_threads(EW, SUM), smem, ctx.stream);
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
    if (cudaLaunchKernelEx(&cfg, kernel, ta, tw, a.tma_out ? m.out : ta, a.tma_res ? m.res : ta, a) != cudaSuccess)
    {
        (void)cudaGetLastError();
        return S2_ERR_CUDA;
    }
    ctx.launches++;
    return S2_OK;
}

template <int TN, int S>
int launch_rows_as(Context& ctx, const Operands& o, const LinearArgs& a, int64_t units)
{
    using RS = RowsShape<TN>;
    auto kernel = linear_rows_kernel<TN, S>;
    CUtensorMap ta, tw;
    int r = make_tmap_bf16_2d(&ta, o.A, a.K, a.rows, (uint64_t)o.lda * 2, BK, TN);
    if (r == S2_OK)
        r = make_tmap_bf16_2d(&tw, o.W, a.K, (uint64_t)a.groups * a.N, (uint64_t)o.ldw * 2, BK, 128);
    if (r != S2_OK) return r;
    static std::atomic<uint64_t> configured{0};
    if (set_up_current_device(configured, [&] {
            return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RS::SMEM_BYTES);
        }) != cudaSuccess)
        return S2_ERR_CUDA;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = cluster_config(attr, S, (unsigned)(units * S), kRowsThreads, RS::SMEM_BYTES, ctx.stream);
    if (cudaLaunchKernelEx(&cfg, kernel, ta, tw, a) != cudaSuccess)
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
    a.nblk = (a.N + 127) / 128;
    // K parts: as many as the resident CTAs leave room for, by the row tiles that
    // equal groups would have
    const int mean_rows = (a.rows + a.groups - 1) / a.groups;
    const int64_t usual = (int64_t)a.groups * ((mean_rows + TN - 1) / TN) * a.nblk;
    int s = 1;
    for (int p : {2, 3, 4, 6, 8})
        if (p <= a.num_kb && usual * p <= 2 * ctx.num_sms) s = p;
    // A CTA (or cluster) for each row tile of one group; of several, for each
    // group's first, and for the others, of which there can be (rows - 1) / TN, as
    // many as are resident at once.  8,192 rows in 1,024 groups, 512 x 512: all in
    // one group 137 us (1,886 where a group's CTAs took its tiles in turn, 90 with a
    // CTA for each tile that there can be), 8 rows in each 113 (105 and 160).
    const int64_t others = (a.rows - 1) / TN;
    const int64_t resident = std::max<int64_t>(1, 2 * ctx.num_sms / ((int64_t)a.nblk * s));
    const int64_t units = (a.groups + (a.offsets ? std::min(others, resident) : others)) * a.nblk;
    if (units * s > 0x7fffffff) return S2_ERR_INVALID;
    a.chunk_kb = chunk_blocks((a.num_kb + s - 1) / s, a.out_f32);
    const int esz = a.out_f32 ? 4 : 2;
    a.vec_out = reinterpret_cast<uintptr_t>(a.out) % (4 * esz) == 0 && a.out_ld % 4 == 0;
    a.vec_res = reinterpret_cast<uintptr_t>(a.residual) % (4 * esz) == 0 && a.residual_ld % 4 == 0;
    switch (s)
    {
    case 1: return launch_rows_as<TN, 1>(ctx, o, a, units);
    case 2: return launch_rows_as<TN, 2>(ctx, o, a, units);
    case 3: return launch_rows_as<TN, 3>(ctx, o, a, units);
    case 4: return launch_rows_as<TN, 4>(ctx, o, a, units);
    case 6: return launch_rows_as<TN, 6>(ctx, o, a, units);
    default: return launch_rows_as<TN, 8>(ctx, o, a, units);
    }
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
    // Tiles of m x n; the sizes of several groups are not known here: each ends
    // in half a tile on average.
    auto tiles = [&](int m, int n) {
        const double row_tiles = groups == 1 ? (rows + m - 1) / m : groups * ((double)rows / groups / m + 0.5);
        return row_tiles * ((N + n - 1) / n);
    };
    // The transposed product, whose K is split over clusters: up to 16 rows a
    // group (64 groups of 2,048 x 1,024: 2 rows 53 us, against 58 in tiles; 16 rows
    // 58 and 59, 24 rows 61 and 60; 16 x 51,200 x 2,560 55 and 82), up to 64 where
    // there are fewer than two tiles a SM (16 groups of 2,048 x 2,048, 256 tiles, at
    // 64 rows 35 against 37; 32 of 2,560 x 2,560, 480 tiles, at 32 rows 87.3 and
    // 86.8; 64 x 51,200 x 2,560, 400 tiles, 63 and 59), and more rows of one group
    // while half the SMs would have no tile (2,560 x 2,560: 300 rows, 60 tiles, 19
    // us against 21; 512 rows, 80 tiles, 24 and 20).
    const double few = tiles(128, 128);
    if (mean_rows <= 16 || (mean_rows <= 64 && few < 2 * c.num_sms) || (groups == 1 && few < 0.5 * c.num_sms))
    {
        // groups somewhat above the mean still fit one row tile
        const int most = groups == 1 ? rows : mean_rows + mean_rows / 2;
        if (most <= 16) return launch_rows<16>(c, o, a);
        if (most <= 32) return launch_rows<32>(c, o, a);
        return launch_rows<64>(c, o, a);
    }
    // A round of 256 x 256 tiles on CTA pairs takes 1.45 times one of 128 x 128
    // tiles for four times the work on twice the SMs, and wins unless its last
    // round is mostly empty (2,560 x 2,560, 512 rows: 23.9 against 19.9 us;
    // 1,000 rows: 25.8 against 31.7).
    auto rounds = [&](double t, int slots) { return groups == 1 ? std::ceil(t / slots) : t / slots + 0.5; };
    const bool pair = N > 128 && 1.45 * rounds(tiles(256, 256), c.num_sms / 2) <= rounds(tiles(128, 128), c.num_sms);
    BoxMaps m;
    const int esz = a.out_f32 ? 4 : 2;
    a.tma_out = make_tmap_2d(&m.out, out, a.out_f32, N, rows, (uint64_t)ldo * esz, 128 / esz, 32) == S2_OK;
    a.tma_res = a.residual && make_tmap_2d(&m.res, a.residual, a.out_f32, N, rows, (uint64_t)a.residual_ld * esz,
                                           128 / esz, 32) == S2_OK;
    // Boxes per epilogue warp: a third one costs an operand stage and pays
    // where the epilogue moves much beside the operands (of 128 x 256 outputs a
    // CTA): from a quarter of their bytes on (288,000 x 256 x 512 with a bf16
    // residual 124 against 134 us; 21,658 x 2,560 x 1,280: 131 against 124),
    // for sums from a fifth (21,658 x 2,560 x 2,560 with an fp32 residual 293
    // against 317 us; x 10,240: 896 against 857).
    const double moved = 128.0 * 256 * osz, fed = (double)a.num_kb * 32768;
    if (a.out_f32 && a.num_kb > kChunk)
    {
        if (!pair) return launch_tiles<1, 128, 2, 8, true>(c, o, m, a);
        return moved >= 0.2 * fed ? launch_tiles<2, 256, 3, 8, true>(c, o, m, a)
                                  : launch_tiles<2, 256, 2, 8, true>(c, o, m, a);
    }
    if (!pair) return launch_tiles<1, 128, 2, 8, false>(c, o, m, a);
    if (!a.tma_out || (a.residual && !a.tma_res)) return launch_tiles<2, 256, 1, 16, false>(c, o, m, a);
    return moved >= 0.25 * fed ? launch_tiles<2, 256, 3, 8, false>(c, o, m, a)
                               : launch_tiles<2, 256, 2, 8, false>(c, o, m, a);
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
