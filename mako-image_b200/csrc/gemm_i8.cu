// The 8-bit integer projection (see gemm_i8.cuh): three kernels for three ranges of rows.
//   k_i8_rows    one or two rows: the weights stream through the CUDA cores once (dp4a); HBM is the bound.
//   k_i8_few     few rows: 128 rows of W are the MMA's M and the tokens its N (16 to 64), so that a stage is mostly weights
//                and the outputs' columns lie along the lanes; K is cut over a cluster whose CTAs add their integer sums
//                through distributed shared memory. Bound by HBM for wide W, else by latency.
//   k_i8_pair    the rest: persistent 256 x BN tiles on CTA pairs (cta_group::2), the tensor pipe is the bound.
// The sums are exact integers, so a row's result is the same bits whichever kernel and split computes it.
#include "gemm_i8.cuh"
#include "common.cuh"
#include "gemm.cuh"
#include "launch.cuh"
#include "sm100.cuh"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cudaTypedefs.h>
#include <algorithm>
#include <mutex>
#include <type_traits>

namespace mkb {

namespace {

constexpr int kBK = 128;  // bytes of K a stage: one 128-byte swizzle row

// ------------------------------------------------------------------------------------------------ epilogue arithmetic

// v / (1 + 2^e).
__device__ __forceinline__ float over_one_and_power(float v, float e)
{
    float p, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(e));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + p));
    return v * r;
}

// Activations to a few fp32 roundings of their value (the erf form's are of v). The GELU's (1 + tanh(u)) / 2 is
// 1 / (1 + e^-2u): 1 + tanh(u) cancels where v is negative, and with tanh.approx the result was off by a fifth of itself at -3.
// The second SFU operation costs where tiles wait for their epilogue: 8192 x 12288 x 3072 to bf16 205 -> 207 us,
// 3679 x 10240 x 1216 57 -> 63, 700 x 8192 x 1024 14.1 -> 15.1; nothing for few rows.
__device__ __forceinline__ float act1(float v, int act)
{
    constexpr float kLog2e = 1.4426950408889634f;
    if (act == kActGeluTanh) {
        constexpr float c = -2.0f * 0.7978845608028654f * kLog2e;
        return over_one_and_power(v, v * fmaf(c * 0.044715f, v * v, c));
    }
    if (act == kActSilu)
        return over_one_and_power(v, -kLog2e * v);
    if (act == kActQuickGelu)
        return over_one_and_power(v, -1.702f * kLog2e * v);
    if (act == kActGeluErf)
        return 0.5f * v * (1.0f + erff(v * 0.7071067811865476f));
    return v;
}

// The switch outside the loop, so that the columns' chains interleave.
template <int N>
__device__ __forceinline__ void act_out(float (&v)[N], int act)
{
    switch (act) {
    case kActGeluTanh:
#pragma unroll
        for (int j = 0; j < N; ++j)
            v[j] = act1(v[j], kActGeluTanh);
        break;
    case kActSilu:
#pragma unroll
        for (int j = 0; j < N; ++j)
            v[j] = act1(v[j], kActSilu);
        break;
    case kActQuickGelu:
#pragma unroll
        for (int j = 0; j < N; ++j)
            v[j] = act1(v[j], kActQuickGelu);
        break;
    case kActGeluErf:
#pragma unroll
        for (int j = 0; j < N; ++j)
            v[j] = act1(v[j], kActGeluErf);
        break;
    }
}

// ------------------------------------------------------------------------------------------------ few rows

constexpr int kRowsMax = 2;

// MR rows of x against R rows of W a warp (WK = 1), or against R rows of W a block whose 8 warps share the K axis (WK =
// 8, for matrices with too few rows of W to fill the GPU otherwise). Lanes take 16 bytes of K each.
template <int MR, int R, int WK>
__global__ void __launch_bounds__(256) k_i8_rows(const GemmI8Args a)
{
    __shared__ int part[WK > 1 ? 8 * MR * R : 1];
    grid_dep_wait();
    grid_dep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = WK == 1 ? (blockIdx.x * 8 + warp) * R : blockIdx.x * R;
    int acc[MR][R] = {};
    if (WK > 1 || n0 < a.N) {
        const int8_t* w[R];
#pragma unroll
        for (int r = 0; r < R; ++r)
            w[r] = a.w + long(min(n0 + r, a.N - 1)) * a.ldw;
        const int whole = a.K >> 4;
#pragma unroll 2
        for (int c = (WK == 1 ? 0 : warp * 32) + lane; c < whole; c += 32 * WK) {
            int4 wv[R];
#pragma unroll
            for (int r = 0; r < R; ++r)
                wv[r] = __ldg(reinterpret_cast<const int4*>(w[r]) + c);
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                if (m < a.M) {
                    const int4 xv = __ldg(reinterpret_cast<const int4*>(a.x + m * a.ldx) + c);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        int s = __dp4a(xv.x, wv[r].x, acc[m][r]);
                        s = __dp4a(xv.y, wv[r].y, s);
                        s = __dp4a(xv.z, wv[r].z, s);
                        acc[m][r] = __dp4a(xv.w, wv[r].w, s);
                    }
                }
            }
        }
        // The last K % 16 values one by one: a row's memory may end with them.
        const int k = (whole << 4) + lane;
        if (k < a.K && (WK == 1 || warp == 0))
#pragma unroll
            for (int m = 0; m < MR; ++m)
                if (m < a.M)
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        acc[m][r] += int(a.x[m * a.ldx + k]) * int(w[r][k]);
    }
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int r = 0; r < R; ++r)
            acc[m][r] = __reduce_add_sync(0xffffffffu, acc[m][r]);
    if constexpr (WK > 1) {
        if (lane == 0)
#pragma unroll
            for (int m = 0; m < MR; ++m)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    part[(warp * MR + m) * R + r] = acc[m][r];
        __syncthreads();
        if (warp)
            return;
    }
    // Lane m * R + r finishes output (m, r).
    const int m = lane / R, r = lane % R, n = n0 + r;
    int s = 0;
    if constexpr (WK > 1) {
        if (m < MR)
            for (int i = 0; i < 8; ++i)
                s += part[(i * MR + m) * R + r];
    } else {
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (m == i && r == j)
                    s = acc[i][j];
    }
    if (m >= a.M || m >= MR || n >= a.N)
        return;
    float v[1] = {fmaf(float(s) * a.x_scale[m], a.w_scale[n], a.bias ? a.bias[n] : 0.0f)};
    act_out(v, a.act);
    if (a.out_f32)
        static_cast<float*>(a.y)[m * a.ldy + n] = v[0];
    else
        static_cast<__nv_bfloat16*>(a.y)[m * a.ldy + n] = __float2bfloat16(v[0]);
}

// ------------------------------------------------------------------------------------------------ tensor-core kernels

struct I8Params {
    CUtensorMap tx, tw, ty;
    GemmI8Args a;
    int splits;   // k_i8_few: CTAs of a cluster, each a part of K
    int boxes;    // k_i8_pair: outputs leave as TMA boxes
};

template <int BN>
struct FewCfg {
    static constexpr int kWBytes = 128 * kBK, kXBytes = BN * kBK, kStageBytes = kWBytes + kXBytes;
    static constexpr int kStages = (200 * 1024) / kStageBytes;
    static constexpr int kTmemCols = BN < 32 ? 32 : BN;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + BN * 4 + 256;
    static_assert(kSmem <= 227 * 1024);
    static_assert(kStages * kStageBytes >= 128 * BN * 4, "the partial sums reuse the stages");
};

// Two (or eight) consecutive columns of this warp's lanes.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[2])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(taddr) : "memory");
}

__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// One tile of 128 output columns x BN tokens a cluster (blockIdx.x = tile * splits + part), K cut into `splits` runs of whole
// stages. Accumulator lane n holds output column n, its columns the tokens. After the main loop CTA p holds the sums of its
// run; it hands the tokens [o * BN / splits, ...) to CTA o's shared memory for every other o, and finishes its own tokens with
// what the others brought. The epilogue is written small: a launch runs it once or twice, and long straight code costs more
// in instruction misses (7 us for 32 unrolled columns) than it saves.
template <int BN>
__global__ void __launch_bounds__(192, 1) k_i8_few(const __grid_constant__ I8Params P)
{
    using C = FewCfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* sx = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);  // [BN] the tokens' scales
    uint64_t* full = reinterpret_cast<uint64_t*>(sx + BN);
    uint64_t* empty = full + C::kStages;
    uint64_t* acc_full = empty + C::kStages;
    uint64_t* drain = acc_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const GemmI8Args& a = P.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int S = P.splits, part = S > 1 ? int(cluster_ctarank()) : 0, tile = blockIdx.x / S;
    const int num_m = (a.M + BN - 1) / BN, mb = tile % num_m, nb = tile / num_m;
    const int num_k = (a.K + kBK - 1) / kBK, k_lo = int(long(num_k) * part / S), k_hi = int(long(num_k) * (part + 1) / S);

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&P.tx);
        prefetch_tmap(&P.tw);
    }
    grid_dep_wait();  // before TMEM allocation and the first global access
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_launch();
    const uint32_t tmem = *tmem_slot;
    const int n = nb * 128 + (warp & 3) * 32 + lane;  // this epilogue thread's output column
    float sw = 0.0f, bias = 0.0f;
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            for (int kb = k_lo; kb < k_hi; ++kb, ++it) {
                const int s = it % C::kStages;
                if (!mbar_wait(&empty[s], ((it / C::kStages) & 1) ^ 1, a.status, kErrWaitEmpty, abort_flag)) {
                    ok = false;
                    break;
                }
                uint8_t* st = smem + s * C::kStageBytes;
                mbar_arrive_expect_tx(&full[s], C::kStageBytes);
                tma_load_2d(st, &P.tw, &full[s], kb * kBK, nb * 128);
                tma_load_2d(st + C::kWBytes, &P.tx, &full[s], kb * kBK, mb * BN);
            }
            if (!ok)  // let the loads already issued land before the CTA can exit
                for (int j = std::max(0, it - C::kStages); j < it; ++j)
                    mbar_wait(&full[j % C::kStages], (j / C::kStages) & 1, a.status, kErrWaitDrain, nullptr);
        }
    } else if (warp == 1) {
        // The whole warp walks and waits, so that descriptors stay in uniform registers; one lane issues.
        constexpr uint32_t idesc = idesc_i8_s32(128, BN);
        int it = 0;
        for (int kb = k_lo; kb < k_hi; ++kb, ++it) {
            const int s = it % C::kStages;
            if (!__all_sync(0xffffffffu,
                            mbar_wait(&full[s], (it / C::kStages) & 1, a.status, kErrWaitFull, abort_flag))) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint64_t dw = desc_kmajor_sw128(smem_u32(smem + s * C::kStageBytes)),
                           dx = desc_kmajor_sw128(smem_u32(smem + s * C::kStageBytes + C::kWBytes));
            if (elect_one_sync()) {
#pragma unroll
                for (int k = 0; k < kBK / 32; ++k)  // 32 bytes are 2 units of a descriptor's address
                    mma_i8_ss(tmem, dw + 2 * k, dx + 2 * k, idesc, (it | k) != 0);
                mma_commit(&empty[s]);
            }
            __syncwarp();
        }
        if (elect_one_sync()) {
            if (ok)
                mma_commit(acc_full);
            mma_commit(drain);
        }
        __syncwarp();
        mbar_wait(drain, 0, a.status, kErrWaitDrain, nullptr);
    } else {
        // While the main loop runs: the tokens' scales, this thread's column's scale and bias.
        for (int i = int(threadIdx.x) - 64; i < BN; i += 128)
            sx[i] = mb * BN + i < a.M ? __ldg(a.x_scale + mb * BN + i) : 0.0f;
        if (n < a.N) {
            sw = __ldg(a.w_scale + n);
            bias = a.bias ? __ldg(a.bias + n) : 0.0f;
        }
        named_barrier_sync<1, 128>();
        ok = mbar_wait(acc_full, 0, a.status, kErrWaitAccFull, abort_flag);
        tc_fence_after();
    }
    __syncwarp();
    const int r = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem + (uint32_t((warp & 3) * 32) << 16);
    const int mine = BN / S;  // tokens of this CTA, two at least
    int* sums = reinterpret_cast<int*>(smem);  // [splits - 1][mine][128]
    if (S > 1) {
        __syncthreads();  // the producer and the MMA warp are past their last use of the stages
        cluster_sync_all();
        if (warp >= 2 && ok)
#pragma unroll 1
            for (int o = 0; o < S; ++o) {
                if (o == part)
                    continue;
                const uint32_t dst = map_to_cta(smem_u32(sums) + ((part < o ? part : part - 1) * mine * 128 + r) * 4, o);
                const auto send = [&](auto width, int c) {
                    constexpr int W = decltype(width)::value;
                    uint32_t v[W];
                    tmem_ld(t_lane + o * mine + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        st_cluster(dst + (c + j) * 512, v[j]);
                };
                const int want = min(mine, a.M - mb * BN - o * mine);  // tokens that exist
                if (mine >= 8) {
#pragma unroll 1
                    for (int c = 0; c < want; c += 8)
                        send(std::integral_constant<int, 8>{}, c);
                } else {
#pragma unroll 1
                    for (int c = 0; c < want; c += 2)
                        send(std::integral_constant<int, 2>{}, c);
                }
            }
        cluster_sync_all();
    }
    if (warp >= 2 && ok) {
        const int m0 = mb * BN + part * mine;
        const auto finish = [&](auto width, int c) {
            constexpr int W = decltype(width)::value;
            uint32_t s[W];
            tmem_ld(t_lane + part * mine + c, s);
            tmem_wait_ld();
#pragma unroll 1
            for (int o = 0; o < S - 1; ++o)
#pragma unroll
                for (int j = 0; j < W; ++j)
                    s[j] += uint32_t(sums[(o * mine + c + j) * 128 + r]);
            float v[W];
#pragma unroll
            for (int j = 0; j < W; ++j)
                v[j] = fmaf(float(int(s[j])) * sx[part * mine + c + j], sw, bias);
            act_out(v, a.act);
            if (n < a.N)
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (m0 + c + j < a.M) {
                        if (a.out_f32)
                            static_cast<float*>(a.y)[long(m0 + c + j) * a.ldy + n] = v[j];
                        else
                            static_cast<__nv_bfloat16*>(a.y)[long(m0 + c + j) * a.ldy + n] = __float2bfloat16(v[j]);
                    }
        };
        if (mine >= 8) {
#pragma unroll 1
            for (int c = 0; c < mine && m0 + c < a.M; c += 8)
                finish(std::integral_constant<int, 8>{}, c);
        } else {
#pragma unroll 1
            for (int c = 0; c < mine && m0 + c < a.M; c += 2)
                finish(std::integral_constant<int, 2>{}, c);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
}

constexpr int kEpiWarps = 8;
constexpr int kPairThreads = 32 * (2 + kEpiWarps);

template <int BN, bool F32>
struct PairCfg {
    static constexpr int kABytes = 128 * kBK, kBBytes = BN / 2 * kBK, kStageBytes = kABytes + kBBytes;
    // A warp's boxes of 32 rows of 64 bytes: one for bf16, two for fp32, whose 32 columns are two of them (3679 x 10240 x 1216
    // with GELU, as it was then, 81 -> 74 us, 68 now; the stage that they cost 256 columns: 8192 x 3072 x 3072 60.0 -> 61.5).
    static constexpr int kBox = 32 * 64, kBoxes = F32 ? 2 : 1;
    static constexpr int kStages = BN == 256 ? 6 - F32 : BN == 192 ? 7 - F32 : BN == 160 ? 7 : 8 - F32;
    static constexpr int kVec = 2 * 2 * BN * 4;  // w_scale and bias of two tiles
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kEpiWarps * kBoxes * kBox + kVec + 256;
    static constexpr int kTmemCols = BN > 128 ? 512 : 256;  // two accumulators, a power of two
    static_assert(kStageBytes % 1024 == 0 && kSmem <= 227 * 1024);
};

// Tiles in groups of 8 along M, so that concurrent tiles share panels of x and W in L2.
__device__ __forceinline__ void tile_of(int tile, int num_m, int num_n, int& mb, int& nb)
{
    const int per_group = 8 * num_n, group = tile / per_group, first = group * 8;
    const int gsize = min(num_m - first, 8), t = tile - group * per_group;
    mb = first + t % gsize;
    nb = t / gsize;
}

// A warp's box, 32 rows of 64 bytes in pieces of 16 that are exchanged by the row (as TMA's 64-byte swizzle has them), to rows
// of any alignment: a lane a column, a row or two at a time. The values come back 16 at a time ahead of their stores: the
// compiler keeps a load behind a store that might be to the same place (one at a time 22.5 us at 2300 x 2100 x 2048 to bf16).
__device__ __forceinline__ int box_piece(int row, int piece) { return row * 64 + ((piece ^ ((row >> 1) & 3)) << 4); }

template <typename T>
__device__ __forceinline__ void store_box(T* p, long ldy, const uint8_t* box, int rows, int cols, int lane)
{
    constexpr int kCols = 64 / sizeof(T), kRows = 32 / kCols, kPiece = 16 / sizeof(T);
    const int col = lane % kCols, row = lane / kCols;
    p += row * ldy + col;
#pragma unroll 1
    for (int i = 0; i < 32; i += 16 * kRows, p += 16 * kRows * ldy) {
        T x[16];
#pragma unroll
        for (int k = 0; k < 16; ++k)
            x[k] = *reinterpret_cast<const T*>(box + box_piece(i + k * kRows + row, col / kPiece) + col % kPiece * sizeof(T));
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (i + k * kRows + row < rows && col < cols)
                p[k * kRows * ldy] = x[k];
    }
}

// Persistent CTA pairs. Warp 0 of each CTA loads its 128 rows of x and its half of the W tile by TMA, the leader's warp 1
// issues 256 x BN x 32 MMAs into one of two accumulators, warps 2-9 of both CTAs drain the other: a thread a row, 32 columns at
// a time and every second 32 each, through a 2 KB box a warp that leaves as TMA stores. With four such warps and boxes of 4 KB
// the epilogue was what the tensor pipe waited for (8192 x 12288 x 3072 with a GELU by tanh.approx 218 us, with eight 205).
template <int BN, bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1) k_i8_pair(const __grid_constant__ I8Params P)
{
    using C = PairCfg<BN, F32>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* boxes = smem + C::kStages * C::kStageBytes;
    float* vec = reinterpret_cast<float*>(boxes + kEpiWarps * C::kBoxes * C::kBox);  // [2][w_scale, bias][BN]
    uint64_t* full = reinterpret_cast<uint64_t*>(boxes + kEpiWarps * C::kBoxes * C::kBox + C::kVec);
    uint64_t* empty = full + C::kStages;
    uint64_t* acc_full = empty + C::kStages;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* drain = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile uint32_t* gave_up = tmem_slot + 2;  // either CTA's roles
    volatile uint32_t* loaded = tmem_slot + 3;   // the leader's: stages that each CTA had loaded when it gave up
    const GemmI8Args& a = P.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int pair = blockIdx.x / 2, npairs = gridDim.x / 2;
    const int num_m = int((a.M + 255L) / 256), num_n = int((a.N + BN - 1L) / BN), num_k = (a.K + kBK - 1) / kBK;
    const int num_tiles = num_m * num_n;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 2 * 32 * kEpiWarps);  // the epilogue threads of both CTAs (leader's barrier)
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        *gave_up = 0;
        loaded[0] = loaded[1] = ~0u;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&P.tx);
        prefetch_tmap(&P.tw);
    }
    grid_dep_wait();  // before TMEM allocation and the first global access
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, C::kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers exist before either signals the other's
    tc_fence_after();
    grid_dep_launch();
    const uint32_t tmem = *tmem_slot;
    uint32_t it = 0;  // warp 0: stages loaded; warp 1: stages multiplied

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (int tile = pair; tile < num_tiles && ok; tile += npairs) {
                int mb, nb;
                tile_of(tile, num_m, num_n, mb, nb);
                for (int kb = 0; kb < num_k; ++kb, ++it) {
                    const int s = it % C::kStages;
                    if (!mbar_wait(&empty[s], ((it / C::kStages) & 1) ^ 1, a.status, kErrWaitEmpty, abort_flag)) {
                        ok = false;
                        break;
                    }
                    uint8_t* sa = smem + s * C::kStageBytes;
                    if (leader)
                        mbar_arrive_expect_tx(&full[s], 2 * C::kStageBytes);  // both CTAs' loads land on it
                    if (a.test_stall && it == 0 && blockIdx.x == 0)
                        continue;  // half of the stage's bytes never arrive: full[0] cannot complete (failure-path test)
                    tma_load_2d_pair(sa, &P.tx, &full[s], kb * kBK, mb * 256 + int(rank) * 128);
                    tma_load_2d_pair(sa + C::kABytes, &P.tw, &full[s], kb * kBK, nb * BN + int(rank) * (BN / 2));
                }
            }
        }
    } else if (warp == 1) {
        // The leader's whole warp walks and waits, so that descriptors stay in uniform registers; one lane issues.
        if (leader) {
            constexpr uint32_t idesc = idesc_i8_s32(256, BN);
            uint32_t lt = 0;
            bool ok = true;
            for (int tile = pair; tile < num_tiles && ok; tile += npairs, ++lt) {
                const uint32_t acc = lt & 1, acc_ph = (lt >> 1) & 1;
                if (!__all_sync(0xffffffffu,
                                mbar_wait(&acc_empty[acc], acc_ph ^ 1, a.status, kErrWaitAccEmpty, abort_flag)))
                    break;
                tc_fence_after();
                for (int kb = 0; kb < num_k; ++kb, ++it) {
                    const int s = it % C::kStages;
                    if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (it / C::kStages) & 1, a.status, kErrWaitFull,
                                                           abort_flag))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t da = desc_kmajor_sw128(smem_u32(smem + s * C::kStageBytes)),
                                   db = desc_kmajor_sw128(smem_u32(smem + s * C::kStageBytes + C::kABytes));
                    if (elect_one_sync()) {
#pragma unroll
                        for (int k = 0; k < kBK / 32; ++k)  // 32 bytes are 2 units of a descriptor's address
                            mma_i8_ss_pair(tmem + acc * BN, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
                        mma_commit_pair(&empty[s]);
                    }
                    __syncwarp();
                }
                if (ok && elect_one_sync())
                    mma_commit_pair(&acc_full[acc]);
                __syncwarp();
            }
            if (elect_one_sync())
                mma_commit_pair(drain);
            __syncwarp();
            mbar_wait(drain, 0, a.status, kErrWaitDrain, nullptr);
        }
    } else {
        const int q = warp & 3, et = int(threadIdx.x) - 64;
        const uint32_t acc_empty0 = map_to_cta(smem_u32(&acc_empty[0]), 0);
        uint8_t* const own = boxes + (warp - 2) * C::kBoxes * C::kBox;
        uint32_t lt = 0, turn = 0;
        for (int tile = pair; tile < num_tiles; tile += npairs, ++lt) {
            int mb, nb;
            tile_of(tile, num_m, num_n, mb, nb);
            const uint32_t acc = lt & 1, acc_ph = (lt >> 1) & 1;
            const int n0 = nb * BN, row0 = mb * 256 + int(rank) * 128 + q * 32, row = row0 + lane;
            // The tile's column vectors, into the copy that the tile before last read.
            float* sw = vec + acc * 2 * BN;
            for (int i = et; i < BN; i += 32 * kEpiWarps) {
                const bool in = n0 + i < a.N;
                sw[i] = in ? __ldg(a.w_scale + n0 + i) : 0.0f;
                sw[BN + i] = in && a.bias ? __ldg(a.bias + n0 + i) : 0.0f;
            }
            const float sx = row < a.M ? __ldg(a.x_scale + row) : 0.0f;
            const bool got = mbar_wait(&acc_full[acc], acc_ph, a.status, kErrWaitAccFull, abort_flag);
            __syncwarp();  // a wait that ran out may have left the lanes apart
            // Also publishes the vectors; the warps leave together or not at all.
            if (named_barrier_or<1, 32 * kEpiWarps>(!got))
                break;
            tc_fence_after();
            const uint32_t t_row = tmem + (uint32_t(q * 32) << 16) + acc * BN;
#pragma unroll 1
            for (int c = 32 * ((warp - 2) >> 2); c < BN; c += 64) {
                if (n0 + c >= a.N)
                    break;
                uint32_t t[32];
                tmem_ld32(t_row + c, t);
                tmem_wait_ld();
                float v[32];
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 s = *reinterpret_cast<const float4*>(sw + c + j);
                    const float4 b = *reinterpret_cast<const float4*>(sw + BN + c + j);
                    v[j] = fmaf(float(int(t[j])) * sx, s.x, b.x);
                    v[j + 1] = fmaf(float(int(t[j + 1])) * sx, s.y, b.y);
                    v[j + 2] = fmaf(float(int(t[j + 2])) * sx, s.z, b.z);
                    v[j + 3] = fmaf(float(int(t[j + 3])) * sx, s.w, b.w);
                }
                act_out(v, a.act);
                // Through the box to columns from `col`: as a TMA store, or along rows that TMA cannot address (a thread storing
                // its own row: 45 against 16 us at 2300 x 2100 x 2048 to bf16, 81 against 19 at 8000 x 777 x 1000) and the last
                // columns (a cut box would write zeros as far as a piece of 16 bytes goes).
                const auto send = [&](const uint4 (&w)[4], int col, auto* y) {
                    uint8_t* box = own + turn++ % C::kBoxes * C::kBox;
                    if (lane == 0)
                        bulk_wait_read<C::kBoxes - 1>();  // the last store from this box has read it
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<uint4*>(box + box_piece(lane, j)) = w[j];
                    if (!P.boxes || col + int(64 / sizeof(*y)) > a.N) {
                        __syncwarp();
                        store_box(y + row0 * a.ldy + col, a.ldy, box, a.M - row0, a.N - col, lane);
                        if (lane == 0)
                            bulk_commit();  // a group a box, empty here: the waits count them
                        return;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (row0 < a.M)
                            tma_store_2d(&P.ty, box, col, row0);
                        bulk_commit();
                    }
                };
                if constexpr (F32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint4 w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float* f = v + 16 * h + 4 * j;
                            w[j] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                              __float_as_uint(f[3]));
                        }
                        send(w, n0 + c + 16 * h, static_cast<float*>(a.y));
                    }
                } else {
                    uint4 w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        w[j] = make_uint4(pack_bf16x2(v[8 * j], v[8 * j + 1]), pack_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                                          pack_bf16x2(v[8 * j + 4], v[8 * j + 5]), pack_bf16x2(v[8 * j + 6], v[8 * j + 7]));
                    send(w, n0 + c, static_cast<__nv_bfloat16*>(a.y));
                }
            }
            tc_fence_before();
            if (leader)
                mbar_arrive(&acc_empty[acc]);
            else
                mbar_arrive_cluster(acc_empty0 + acc * 8);
        }
        if (lane == 0)
            bulk_wait_all();  // the last boxes are written before the CTA and its shared memory go
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) {
        st_cluster(map_to_cta(smem_u32(const_cast<uint32_t*>(loaded) + rank), 0), it);
        for (uint32_t c = 0; c < 2; ++c)
            st_cluster(map_to_cta(smem_u32(const_cast<uint32_t*>(gave_up)), c), 1);
    }
    __syncwarp();
    cluster_sync_all();  // the leader's MMAs read this CTA's shared memory until here
    if (*gave_up) {
        // Let the loads already issued land before either CTA can exit. They complete on the leader's barriers, which it alone
        // can wait on; a stage that only the other CTA has loaded expects that CTA's bytes, one that only this CTA has (the
        // other gave up first) does not complete, and its wait runs out: the rest have had as long.
        if (threadIdx.x == 0 && leader) {
            const uint32_t whole = uint32_t((num_tiles - pair + npairs - 1) / npairs) * num_k;  // where a CTA did not give up
            const uint32_t mine = min(loaded[0], whole), all = max(mine, min(loaded[1], whole));
            for (uint32_t j = all > C::kStages ? all - C::kStages : 0; j < all; ++j) {
                if (j >= mine)
                    mbar_arrive_expect_tx(&full[j % C::kStages], C::kStageBytes);
                if (!mbar_wait(&full[j % C::kStages], (j / C::kStages) & 1, a.status, kErrWaitDrain, nullptr))
                    break;
            }
        }
        __syncwarp();
        cluster_sync_all();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, C::kTmemCols);
    }
}

// ------------------------------------------------------------------------------------------------ host

PFN_cuTensorMapEncodeTiled_v12000 encode_fn()
{
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

bool encode_2d(CUtensorMap* m, CUtensorMapDataType type, const void* p, long inner, long outer, long row_bytes,
               int box_inner, int box_outer, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B)
{
    auto fn = encode_fn();
    const cuuint64_t dims[2] = {cuuint64_t(inner), cuuint64_t(outer)};
    const cuuint64_t strides[1] = {cuuint64_t(row_bytes)};
    const cuuint32_t box[2] = {cuuint32_t(box_inner), cuuint32_t(box_outer)};
    const cuuint32_t es[2] = {1, 1};
    return fn && fn(m, type, 2, const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MR>
cudaError_t launch_rows(const GemmI8Args& a, cudaStream_t st)
{
    // Few rows of W and a long K: a block a pair of rows, its warps along K. Otherwise a warp takes 4 rows of W where that
    // still gives every SM eight warps, else one.
    const int warps = 8 * num_sms();
    if (a.N < 4 * warps && a.K >= 4096)
        return launch_k(k_i8_rows<MR, 2, 8>, dim3((a.N + 1) / 2), 256, 0, st, a);
    if (a.N >= 4 * warps)
        return launch_k(k_i8_rows<MR, 4, 1>, dim3((a.N + 31) / 32), 256, 0, st, a);
    return launch_k(k_i8_rows<MR, 1, 1>, dim3((a.N + 7) / 8), 256, 0, st, a);
}

// How k_i8_few would run: tokens a tile, parts of K, and about how long in steps of kBK of K (0.2 us each). Beside its steps
// a tile takes 8, its epilogue 0.42 a token that a CTA finishes, and a cut of K 6.5 and 0.17 a token that is sent. Many parts
// pay for long K (132 x 1056 x 6784: 16 tokens, whole 14.1 us, 64 tokens in four parts 8.8), small tiles for short K (77 x 1280
// x 1280: 16 tokens in two parts 4.7, 64 in four 6.0).
struct FewPlan {
    int bn, splits;
    float steps;
};

// Clusters of `size` (2, 4, 8) k_i8_few CTAs, one an SM, that the current device runs at once: they have to fit its GPCs (36
// clusters of four are two waves: 192 x 288 x 9600 15.4 us, 18 of them 8.4). Kept for devices 0..63 once asked.
int clusters_at_once(int size)
{
    static std::atomic<int> known[64][9];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess)
        return 0;
    const bool keep = dev >= 0 && dev < 64;
    if (keep && known[dev][size].load(std::memory_order_relaxed))
        return known[dev][size].load(std::memory_order_relaxed);
    static std::atomic<uint64_t> devs{0};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = FewCfg<16>::kSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = size;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (smem_limit_once(devs, k_i8_few<16>, FewCfg<16>::kSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, k_i8_few<16>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (keep)
        known[dev][size].store(n, std::memory_order_relaxed);
    return n;
}

FewPlan plan_few(long M, long N, int K)
{
    FewPlan best{0, 0, 0.0f};
    const int num_k = (K + kBK - 1) / kBK;
    for (int bn = 16; bn <= 64; bn *= 2) {
        const long tiles = (M + bn - 1) / bn * ((N + 127) / 128);
        // Parts that all run at once, two steps each or more.
        for (int s = 1; s <= 8 && (s == 1 || (num_k >= 2 * s && tiles * s <= num_sms() && tiles <= clusters_at_once(s))); s *= 2) {
            const float sent = s > 1 ? 6.5f + 0.17f * bn * (s - 1) / s : 0.0f;
            const float steps = float((tiles + num_sms() - 1) / num_sms()) * ((num_k + s - 1) / s + 8.0f + 0.42f * bn / s + sent);
            if (!best.bn || steps < best.steps)
                best = FewPlan{bn, s, steps};
        }
    }
    return best;
}

template <int BN>
cudaError_t launch_few(I8Params& P, cudaStream_t st)
{
    static std::atomic<uint64_t> devs{0};
    const cudaError_t e = smem_limit_once(devs, k_i8_few<BN>, FewCfg<BN>::kSmem);
    if (e != cudaSuccess)
        return e;
    const int tiles = (P.a.M + BN - 1) / BN * ((P.a.N + 127) / 128);
    return launch_k_cluster(k_i8_few<BN>, dim3(unsigned(tiles) * P.splits), P.splits, 192, FewCfg<BN>::kSmem, st, P);
}

template <int BN, bool F32>
cudaError_t launch_pair_of(I8Params& P, const char** err, cudaStream_t st)
{
    const GemmI8Args& a = P.a;
    const int size = F32 ? 4 : 2;
    P.boxes = (reinterpret_cast<uintptr_t>(a.y) & 15) == 0 && (a.ldy * size) % 16 == 0;
    if (P.boxes && !encode_2d(&P.ty, F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.y, a.N,
                              a.M, a.ldy * size, 64 / size, 32, CU_TENSOR_MAP_SWIZZLE_64B)) {
        *err = "proj_i8: tensor map encoding failed";
        return cudaErrorInvalidValue;
    }
    const int tiles = int((a.M + 255L) / 256 * ((a.N + BN - 1L) / BN));
    static std::atomic<uint64_t> devs{0};
    const cudaError_t e = smem_limit_once(devs, k_i8_pair<BN, F32>, PairCfg<BN, F32>::kSmem);
    if (e != cudaSuccess)
        return e;
    const int pairs = std::min(tiles, num_sms() / 2);
    return launch_k(k_i8_pair<BN, F32>, dim3(2 * pairs), kPairThreads, PairCfg<BN, F32>::kSmem, st, P);
}

template <int BN>
cudaError_t launch_pair(I8Params& P, const char** err, cudaStream_t st)
{
    return P.a.out_f32 ? launch_pair_of<BN, true>(P, err, st) : launch_pair_of<BN, false>(P, err, st);
}

}  // namespace

cudaError_t gemm_i8(const GemmI8Args& a, const char** err, cudaStream_t st)
{
    cudaError_t e;
    if (a.M <= kRowsMax && !a.test_stall) {
        e = a.M == 1   ? launch_rows<1>(a, st)
                       : launch_rows<2>(a, st);
    } else {
        I8Params P{};
        P.a = a;
        // Pair tiles of 256, 192, 160 or 128 columns: a round of tiles takes about as long as its columns and 128 more (its rows
        // of x, the way in and out), so the width whose rounds take least, the widest among equals. In us, 256, 192, 160, 128
        // columns: 4097 x 1280 x 5120 31.1, 26.6, 25.5, 32.8; 700 x 8192 x 1024 13.0, 11.7, 14.5, 13.9; 512 x 9216 x 3072
        // 14.4, 17.8, 17.3, 16.7; 1000 x 1536 x 1536 9.6, 8.4, 8.2, 7.8.
        const long slots = num_sms() / 2;
        const auto cost = [&](int bn) {
            return (((a.M + 255L) / 256) * ((a.N + bn - 1L) / bn) + slots - 1) / slots * (bn + 128);
        };
        int bn = 256;
        for (const int width : {192, 160, 128})
            if (cost(width) < cost(bn))
                bn = width;
        // Against k_i8_few in its steps: a round of 128 columns takes one for each of K, and a launch 24 beside them (256 x 3072 x
        // 3072 10.3 us here, 12.6 there; 200 x 1280 x 1280 6.8 and 5.3, 500 x 512 x 8192 18.0 and 9.4).
        const FewPlan plan = plan_few(a.M, a.N, a.K);
        const bool few = !a.test_stall && plan.steps <= float(cost(bn)) / 256.0f * ((a.K + kBK - 1) / kBK) + 24.0f;
        P.splits = plan.splits;
        const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
        if (!encode_2d(&P.tx, u8, a.x, a.K, a.M, a.ldx, kBK, few ? plan.bn : 128) ||
            !encode_2d(&P.tw, u8, a.w, a.K, a.N, a.ldw, kBK, few ? 128 : bn / 2)) {
            *err = "proj_i8: tensor map encoding failed";
            return cudaErrorInvalidValue;
        }
        if (few) {
            e = plan.bn == 16   ? launch_few<16>(P, st)
                : plan.bn == 32 ? launch_few<32>(P, st)
                                : launch_few<64>(P, st);
        } else {
            e = bn == 256   ? launch_pair<256>(P, err, st)
                : bn == 192 ? launch_pair<192>(P, err, st)
                : bn == 160 ? launch_pair<160>(P, err, st)
                            : launch_pair<128>(P, err, st);
        }
    }
    if (e != cudaSuccess)
        return e;
    count_launch();
    return cudaGetLastError();
}

}  // namespace mkb
