// Attention to another stream's keys (see cross_attention.cuh): k_cross on tcgen05, and for a handful of query rows
// k_cross_few on the CUDA cores.
//
// k_cross: keys are few and queries many, so the work is a stream of query tiles past small sets of keys: persistent CTAs walk
// items of (sample, head, 256 query rows) as two 128-row tiles A and B, and every stage runs ahead into the next item, so
// that one item's loads, another's products and a third's stores overlap. Twelve warps:
//   warp 0     TMA: Q tiles in one ring, K and V tiles of 128 keys in another
//   warp 1     MMA: S = Q K^T, then O += P V with P in tensor memory, for A and B in turn (a warp for each of A and B, whose
//              products then mix on the tensor pipe, was slower: 603 against 455 us at 2 x 24 x 4096 x 4096 x 128)
//   warp 2     with a mask: a bound for each key's score, -inf for a hidden one, ahead of the softmax
//   warps 4-7  softmax of tile A, 8-11 of tile B: a thread a row, the running maximum and sum of one pass; where a step has
//              hidden keys each thread also clears its row of V if that is one (0 * NaN would spread); each warp stages its
//              output rows in 4 KB of its own, 64 columns at a time, and sends them off as TMA stores (a thread storing its
//              row directly touches 32 lines an instruction)
// Where the items leave most of the GPU idle and the keys are many, SPLIT runs one item a cluster, whose CTAs take a run of
// the key steps each and put the parts together through distributed shared memory: no workspace, no second launch. An item of a
// single query tile gives it to both softmax groups there, who take the steps in turn as two parts.
// Only ceil(visible / 16) * 16 keys of the last tile are multiplied and exponentiated (77 keys cost 80, not 128).
// Scores, maxima, sums and O are fp32. The weights alone are rounded, to bf16, as the second product takes P in V's type: each is
// off by up to 2^-8 of itself, which leaves results a relative error of 2.0 to 2.1e-3 where their own rounding to bf16 makes
// 1.7e-3. The sum l adds them before that rounding. k_cross_few keeps fp32 weights (1.7e-3).
// TMEM columns: S_A [0, 128), S_B [128, 256), O_A [256, 384), O_B [384, 512); P takes the first half of its S.
#include "cross_attention.cuh"
#include "common.cuh"
#include "gemm.cuh"
#include "launch.cuh"
#include "sm100.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <algorithm>
#include <mutex>
#include <type_traits>

namespace mkb {

namespace {

constexpr int kThreads = 384;
// The launch gives every thread 168 registers; the control warpgroup drops to kRegsCtl and the softmax warpgroups rise to
// kRegsSoftmax, enough for a row's 128 scores.
constexpr int kLaunchRegs = (65536 / kThreads) / 8 * 8;
constexpr int kRegsCtl = 88, kRegsSoftmax = 208;
static_assert(128 * kRegsCtl + 256 * kRegsSoftmax <= kThreads * kLaunchRegs, "register split exceeds the CTA pool");
constexpr int kTile = 128;              // query rows a tile, keys a tile
constexpr int kPanel = kTile * 64 * 2;  // 64 bf16 columns of 128 rows
constexpr int kSteps = 5;               // full barriers of K and of V: no more key steps than that are ever in flight
constexpr int kHideSteps = 2;           // key steps whose hidden keys are kept ready
constexpr float kRescaleThreshold = 8.0f;  // log2 units: O is rescaled only when a row's maximum grows by more

template <int D, bool SPLIT>
struct Cfg {
    static constexpr int kTileBytes = (D / 64) * kPanel;
    // Q tiles (two at work and, unless the item is the only one, the next on their way), K and V tiles, the output stage.
    static constexpr int kQ = SPLIT ? 2 : D == 64 ? 5 : 3;
    static constexpr int kSlots = SPLIT ? (D == 64 ? 10 : 5) : (D == 64 ? 7 : 3);
    static constexpr int kStage = SPLIT ? 0 : 2 * kPanel;
    static constexpr int kSmem = 1024 + (kQ + kSlots) * kTileBytes + kStage + 512 + kHideSteps * (kTile * 4 + 16);
    static_assert(kSmem <= 227 * 1024);
    static_assert((kSlots + 1) / 2 <= kSteps);
    // SPLIT: two tiles' parts and (m, l) pairs for up to 8 CTAs (S * ceil(128 / S) <= 133 rows for S <= 8) fit the stages.
    static_assert(2 * 133 * D * 4 + 2 * 8 * kTile * 8 <= (kQ + kSlots) * kTileBytes);
};

struct CrossParams {
    CUtensorMap tq, tk, tv, to;
    CrossArgs a;
    // 0 where a dimension is shared (stride 0): its coordinate stays 0.
    int q_head, q_sample, kv_head_k, kv_sample_k, kv_head_v, kv_sample_v, o_head, o_sample;
    int items, blocks;  // work items, query blocks of 256 rows
    int splits;         // SPLIT: CTAs of a cluster
    int in_step;        // every item gives both softmax groups work
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A CTA's items, gridDim.x apart: (sample, head, query block) and its keys. The digits of the item number are advanced by
// the digits of the stride (a division for each item would sit in every role's way).
template <bool SPLIT>
struct Items {
    int item, b, h, blk, db, dh, dblk;
    // n: keys up to the last that may be visible; lo, hi: this CTA's steps of 128 of them; tiles: 1 or 2 query tiles
    int n, lo, hi, tiles;
    __device__ __forceinline__ void keys(const CrossArgs& a)
    {
        n = a.key_len ? min(max(__ldg(a.key_len + min(b, a.B - 1)), 0), a.Lk) : a.Lk;
    }
    __device__ __forceinline__ void sizes(const CrossParams& P)
    {
        lo = 0;
        hi = (n + kTile - 1) / kTile;
        if constexpr (SPLIT) {
            const int part = int(cluster_ctarank()), steps = hi;
            lo = int(long(steps) * part / P.splits);
            hi = int(long(steps) * (part + 1) / P.splits);
        }
        tiles = blk * 2 * kTile + kTile < P.a.Lq ? 2 : 1;
    }
    __device__ __forceinline__ void first(const CrossParams& P)
    {
        item = SPLIT ? int(blockIdx.x) / P.splits : int(blockIdx.x);
        const int bh = item / P.blocks, dbh = int(gridDim.x) / P.blocks;
        blk = item - bh * P.blocks;
        b = bh / P.a.H;
        h = bh - b * P.a.H;
        dblk = int(gridDim.x) - dbh * P.blocks;
        db = dbh / P.a.H;
        dh = dbh - db * P.a.H;
        keys(P.a);
        sizes(P);
    }
    __device__ __forceinline__ void next(const CrossParams& P)
    {
        if constexpr (SPLIT) {
            item = P.items;
            return;
        }
        const int was = b;
        item += gridDim.x;
        blk += dblk;
        h += dh;
        b += db;
        if (blk >= P.blocks) {
            blk -= P.blocks;
            ++h;
        }
        if (h >= P.a.H) {
            h -= P.a.H;
            ++b;
        }
        if (b != was)
            keys(P.a);
        sizes(P);
    }
    __device__ __forceinline__ bool more(const CrossParams& P) const { return item < P.items; }
    __device__ __forceinline__ int q0() const { return blk * 2 * kTile; }
};

// The walk over all key steps of a CTA's items that have keys.
template <bool SPLIT>
struct Walk {
    Items<SPLIT> it;
    int j;
    __device__ __forceinline__ void settle(const CrossParams& P)  // on to an item with keys
    {
        while (it.more(P) && it.lo == it.hi)
            it.next(P);
        j = it.lo;
    }
    __device__ __forceinline__ void first(const CrossParams& P)
    {
        it.first(P);
        settle(P);
    }
    __device__ __forceinline__ void next(const CrossParams& P)
    {
        if (++j == it.hi) {
            it.next(P);
            settle(P);
        }
    }
    __device__ __forceinline__ bool more(const CrossParams& P) const { return it.more(P); }
    __device__ __forceinline__ bool start() const { return j == it.lo; }
    __device__ __forceinline__ bool last() const { return j + 1 == it.hi; }
    // Keys of the step that are multiplied: those up to n, in sixteens.
    __device__ __forceinline__ int width() const { return min(kTile, (it.n - j * kTile + 15) & ~15); }
};

// A row's step over CH chunks of 32 keys: its scores in tensor memory at ts to weights 2^(s sc - m), bf16 (see above), over the
// first half of the same columns; the row's maximum m and sum l; O at `to` rescaled where the maximum grew. Of the last chunk only the
// first `tail` keys are visible. With `masked` each score is cut at its key's bound, +inf or -inf (the minimum drops a NaN,
// and a visible NaN comes back as inf - inf). Straight code for each CH: the chunks' loads, exponentials and stores
// interleave.
template <int D, int CH>
__device__ __forceinline__ void softmax_step(uint32_t ts, uint32_t to, int tail, bool masked, const float* bound,
                                             float sc, bool first, float& m, float& l)
{
    uint32_t s[32 * CH];
#pragma unroll
    for (int c = 0; c < CH; ++c)
        tmem_ld32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
    tmem_wait_ld();
    if (masked) {
#pragma unroll
        for (int i = 0; i < 32 * CH; i += 4) {
            const float4 b = *reinterpret_cast<const float4*>(bound + i);
            s[i] = __float_as_uint(fminf(__uint_as_float(s[i]), b.x));
            s[i + 1] = __float_as_uint(fminf(__uint_as_float(s[i + 1]), b.y));
            s[i + 2] = __float_as_uint(fminf(__uint_as_float(s[i + 2]), b.z));
            s[i + 3] = __float_as_uint(fminf(__uint_as_float(s[i + 3]), b.w));
        }
    } else if (tail < 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i >= tail)
                s[32 * (CH - 1) + i] = __float_as_uint(-INFINITY);
    }
    // The maximum as 8 independent chains.
    float mc[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
        mc[u] = fmaxf(__uint_as_float(s[2 * u]), __uint_as_float(s[2 * u + 1]));
#pragma unroll
    for (int i = 16; i < 32 * CH; i += 16)
#pragma unroll
        for (int u = 0; u < 8; ++u)
            mc[u] = fmax3(mc[u], __uint_as_float(s[i + 2 * u]), __uint_as_float(s[i + 2 * u + 1]));
    const float mx = fmax3(fmax3(mc[0], mc[1], mc[2]), fmax3(mc[3], mc[4], mc[5]), fmaxf(mc[6], mc[7])) * sc;
    const bool need = mx > m + kRescaleThreshold;  // also the first step with a visible key
    if (__any_sync(0xffffffffu, need)) {
        const float m_new = need ? mx : m;
        const float f = m == -INFINITY ? 0.0f : ex2(m - m_new);
        l *= f;
        if (!first) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(to + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    tmem_st16(to + c * 32 + 16 * i, *reinterpret_cast<uint32_t(*)[16]>(&o[16 * i]));
            }
        }
        m = m_new;
    }
    // A row that has seen no key yet: 2^(-inf - 0) = 0 for all of them.
    const float shift = m == -INFINITY ? 0.0f : -m;
    const float2 sc2 = make_float2(sc, sc), sh2 = make_float2(shift, shift);
    float2 ls[4] = {};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int k = 32 * c + 2 * i;
            const float2 x = ffma2(make_float2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), sc2, sh2);
            const float2 e = make_float2(ex2(x.x), ex2(x.y));
            ls[i & 3] = fadd2(ls[i & 3], e);
            p[i] = pack_bf16x2(e.x, e.y);
        }
        tmem_st16(ts + 16 * c, p);
    }
    tmem_wait_st();
    const float2 l2 = fadd2(fadd2(ls[0], ls[1]), fadd2(ls[2], ls[3]));
    l += l2.x + l2.y;
}

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v)
{
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

__device__ __forceinline__ void st_cluster_f32x4(uint32_t addr, float4 v)
{
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}

constexpr int kMaxSplits = 8;

// HIDE: which keys may be hidden (the code for a mask, even where it is not run, costs a plain call 4 to 8%).
enum Hide : int { kHideNone = 0, kHideLengths = 1, kHideMask = 2 };
template <int D, bool SPLIT, int HIDE>
__global__ void __launch_bounds__(kThreads, 1) k_cross(const __grid_constant__ CrossParams P)
{
    using C = Cfg<D, SPLIT>;
    constexpr int TB = C::kTileBytes, NS = C::kSlots;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr uint32_t NQ = C::kQ;
    uint8_t* sQ = smem;             // [NQ]
    uint8_t* sKV = smem + NQ * TB;  // [NS]
    uint8_t* sO = sKV + NS * TB;    // [tiles][kPanel]
    float* bounds = reinterpret_cast<float*>(sO + C::kStage);  // [kHideSteps][kTile]
    volatile uint32_t* maskeds = reinterpret_cast<volatile uint32_t*>(bounds + kHideSteps * kTile);
    uint64_t* bars = reinterpret_cast<uint64_t*>(bounds + kHideSteps * (kTile + 4));
    // SPLIT: the rows' parts overlay the stages, this CTA's own result of a row stays in its softmax thread until then.
    float part_m = -INFINITY, part_l = 0.0f;
    bool part_here = false, part_any = false;
    uint64_t* q_full = bars;             // [NQ]
    uint64_t* q_empty = q_full + NQ;     // [NQ]
    uint64_t* kv_empty = q_empty + NQ;   // [NS]
    // By key step, not by slot: where K and V take turns in a slot, threads that follow only the V tiles would miss phases
    // of the slot's barrier.
    uint64_t* k_full = kv_empty + NS;    // [kSteps]
    uint64_t* v_full = k_full + kSteps;  // [kSteps]
    uint64_t* h_full = v_full + kSteps;  // [kHideSteps]
    uint64_t* h_empty = h_full + kHideSteps;
    uint64_t* s_full = h_empty + kHideSteps;  // [tiles]
    uint64_t* p_full = s_full + 2;       // [tiles]
    uint64_t* o_full = p_full + 2;       // [tiles]
    uint64_t* drain = o_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const CrossArgs& a = P.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int i = 0; i < int(NQ); ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < NS; ++i)
            mbar_init(&kv_empty[i], 1);
        for (int i = 0; i < kSteps; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&v_full[i], 1);
        }
        for (int i = 0; i < kHideSteps; ++i) {
            mbar_init(&h_full[i], 1);
            mbar_init(&h_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&P.tq);
        prefetch_tmap(&P.tk);
        prefetch_tmap(&P.tv);
        prefetch_tmap(&P.to);
    }
    grid_dep_wait();  // before TMEM allocation and the first global access
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_launch();
    const uint32_t tmem = *tmem_slot;

    if (warp < 4)
        regs_decrease<kRegsCtl>();
    if (warp == 0) {
        if (lane == 0) {
            Walk<SPLIT> w;
            uint32_t seq = 0, nq = 0;  // K and V tiles, Q tiles loaded
            bool ok = true;
            const auto load = [&](uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int row, int h, int b) {
                mbar_arrive_expect_tx(bar, TB);
#pragma unroll
                for (int p = 0; p < D / 64; ++p)
                    tma_load_4d(dst + p * kPanel, m, bar, p * 64, row, h, b);
            };
            for (w.first(P); w.more(P) && ok; w.next(P)) {
                const int hk = w.it.h / (a.H / a.Hkv);
                for (int t = 0; w.start() && t < w.it.tiles && ok; ++t) {
                    const uint32_t s = nq % NQ;
                    ok = mbar_wait(&q_empty[s], ((nq / NQ) & 1) ^ 1, a.status, kErrAttnWait, abort_flag);
                    if (ok) {
                        load(sQ + s * TB, &P.tq, &q_full[s], w.it.q0() + t * kTile, w.it.h * P.q_head,
                             w.it.b * P.q_sample);
                        ++nq;
                    }
                }
                for (int kv = 0; kv < 2 && ok; ++kv) {
                    const uint32_t s = seq % NS;
                    ok = mbar_wait(&kv_empty[s], ((seq / NS) & 1) ^ 1, a.status, kErrAttnWait, abort_flag);
                    if (ok) {
                        const uint32_t f = (seq >> 1) % kSteps;
                        if (kv == 0)
                            load(sKV + s * TB, &P.tk, &k_full[f], w.j * kTile, hk * P.kv_head_k, w.it.b * P.kv_sample_k);
                        else
                            load(sKV + s * TB, &P.tv, &v_full[f], w.j * kTile, hk * P.kv_head_v, w.it.b * P.kv_sample_v);
                        ++seq;
                    }
                }
            }
            if (!ok) {  // let the loads already issued land before the CTA can exit
                for (uint32_t i = nq > NQ ? nq - NQ : 0; i < nq; ++i)
                    mbar_wait(&q_full[i % NQ], (i / NQ) & 1, a.status, kErrWaitDrain, nullptr);
                for (uint32_t i = seq > NS ? seq - NS : 0; i < seq; ++i)
                    mbar_wait(&(i & 1 ? v_full : k_full)[(i >> 1) % kSteps], ((i >> 1) / kSteps) & 1, a.status,
                              kErrWaitDrain, nullptr);
            }
        }
    } else if (warp == 1) {
        // The whole warp walks and waits, so that addresses and descriptors stay in uniform registers; one lane issues.
        {
            constexpr uint32_t idesc_s0 = idesc_bf16_f32(128, 0), idesc_o = idesc_bf16_f32(128, D, 0, 1);
            const uint64_t dq0 = desc_kmajor_sw128(smem_u32(sQ)), dk0 = desc_kmajor_sw128(smem_u32(sKV)),
                           dv0 = desc_mnmajor_sw128(smem_u32(sKV), kPanel, 1024);  // in units of 16 bytes
            constexpr uint32_t kUnit = TB >> 4;
            uint32_t step = 0, nq = 0, np[2] = {0, 0};  // key steps; Q tile of the item's A; P tiles taken of A and B
            bool ok = true;
            const auto wait = [&](uint64_t* bar, uint32_t phase) {
                return bool(__all_sync(0xffffffffu, mbar_wait(bar, phase & 1, a.status, kErrAttnWait, abort_flag)));
            };
            constexpr std::integral_constant<int, 0> kA;
            constexpr std::integral_constant<int, 1> kB;
            // S_t = Q_t K^T; Q is waited for at an item's first step.
            const auto scores = [&](auto tile, bool first, bool last, uint64_t dk, uint32_t idesc, bool shared_q = false) {
                constexpr int t = decltype(tile)::value;
                const uint32_t n = shared_q ? 0 : nq + t, qi = n % NQ;
                const uint64_t dq = dq0 + qi * kUnit;
                if (first && !wait(&q_full[qi], n / NQ))
                    return false;
                tc_fence_after();
                if (elect_one_sync()) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t off = ((k >> 2) * kPanel + (k & 3) * 32) >> 4;
                        mma_bf16_ss(tmem + t * 128, dq + off, dk + off, idesc, k > 0);
                    }
                    mma_commit(&s_full[t]);
                    if (last)
                        mma_commit(&q_empty[qi]);
                }
                __syncwarp();
                return true;
            };
            // O_t += P_t V.
            const auto outputs = [&](auto tile, bool first, bool last, uint64_t dv, int width) {
                constexpr int t = decltype(tile)::value;
                if (!wait(&p_full[t], np[t]))
                    return false;
                ++np[t];
                tc_fence_after();
                if (elect_one_sync()) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (16 * k < width)
                            mma_bf16_ts(tmem + 256 + t * 128, tmem + t * 128 + 8 * k, dv + k * (2048 >> 4), idesc_o,
                                        !first || k > 0);
                    if (last)
                        mma_commit(&o_full[t]);
                }
                __syncwarp();
                return true;
            };
            Walk<SPLIT> w, x;
            w.first(P);
            if (SPLIT && w.more(P) && w.it.tiles == 1) {
                // One query tile: step g, of tile g % 2, is S_t as soon as its P of two steps before is spent.
                const int steps = w.it.hi - w.it.lo;
                const auto width = [&](int g) { return min(kTile, (w.it.n - (w.it.lo + g) * kTile + 15) & ~15); };
                const auto free_slot = [&](uint64_t* bar) {
                    if (elect_one_sync())
                        mma_commit(bar);
                    __syncwarp();
                };
                const auto score = [&](auto tile, int g) {
                    const uint32_t s = 2 * g % NS;
                    if (!wait(&k_full[g % kSteps], g / kSteps) ||
                        !scores(tile, g < 2, false, dk0 + s * kUnit, idesc_s0 | uint32_t(width(g) >> 3) << 17, true))
                        return false;
                    free_slot(&kv_empty[s]);
                    return true;
                };
                const auto output = [&](auto tile, int g) {
                    const uint32_t s = (2 * g + 1) % NS;
                    if (!wait(&v_full[g % kSteps], g / kSteps) ||
                        !outputs(tile, g < 2, g + 2 >= steps, dv0 + s * kUnit, width(g)))
                        return false;
                    free_slot(&kv_empty[s]);
                    if (HIDE == kHideMask)
                        free_slot(&h_empty[g % kHideSteps]);
                    return g + 2 >= steps || score(tile, g + 2);
                };
                ok = score(kA, 0) && (steps < 2 || score(kB, 1));
                for (int g = 0; g < steps && ok; g += 2)
                    ok = output(kA, g) && (g + 1 >= steps || output(kB, g + 1));
                w.it.item = P.items;  // done
            }
            if (w.more(P)) {
                const uint32_t idesc = idesc_s0 | uint32_t(w.width() >> 3) << 17;
                ok = wait(&k_full[0], 0) && scores(kA, true, w.last(), dk0, idesc) &&
                     (w.it.tiles < 2 || scores(kB, true, w.last(), dk0, idesc));
                if (ok && elect_one_sync())
                    mma_commit(&kv_empty[0]);
                __syncwarp();
            }
            // Per step: O_A += P_A V, S_A of the next step, then B: one tile's softmax runs under the other's products. What
            // the products need is worked out before the wait for P.
            for (; w.more(P) && ok; w = x, ++step) {
                x = w;
                x.next(P);
                const bool more = x.more(P), first = w.start(), last = w.last(), xfirst = x.start(), xlast = x.last();
                const bool b = w.it.tiles > 1, xb = more && x.it.tiles > 1;
                const int width = w.width();
                const uint32_t sv = (2 * step + 1) % NS, sk = (2 * step + 2) % NS;
                const uint64_t dv = dv0 + sv * kUnit, dk = dk0 + sk * kUnit;
                const uint32_t idesc = idesc_s0 | uint32_t(x.width() >> 3) << 17;
                if (last)
                    nq += w.it.tiles;  // the next scores are the next item's
                const auto next_k = [&] { return wait(&k_full[(step + 1) % kSteps], (step + 1) / kSteps); };
                ok = wait(&v_full[step % kSteps], step / kSteps) &&
                     outputs(kA, first, last, dv, width) && (!more || (next_k() && scores(kA, xfirst, xlast, dk, idesc))) &&
                     (!b || outputs(kB, first, last, dv, width)) && (!xb || scores(kB, xfirst, xlast, dk, idesc));
                if (!ok)
                    break;
                if (elect_one_sync()) {
                    if (HIDE == kHideMask)  // the step's weights are made, so its bounds have been read
                        mma_commit(&h_empty[step % kHideSteps]);
                    mma_commit(&kv_empty[sv]);
                    if (more)
                        mma_commit(&kv_empty[sk]);
                }
                __syncwarp();
            }
            if (elect_one_sync())
                mma_commit(drain);  // arrives once every MMA issued above has completed
            __syncwarp();
            mbar_wait(drain, 0, a.status, kErrWaitDrain, nullptr);
        }
    } else if (warp == 2) {
        if (HIDE == kHideMask) {
            Walk<SPLIT> w;
            uint32_t step = 0;
            for (w.first(P); w.more(P); w.next(P), ++step) {
                const uint32_t hs = step % kHideSteps;
                const uint8_t* bytes = a.key_mask + w.it.b * a.mask_stride + w.j * kTile;
                const int left = w.it.n - w.j * kTile;
                bool see[4];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    see[c] = 32 * c + lane < left && __ldg(bytes + 32 * c + lane) != 0;
                uint32_t masked = 0;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    masked |= __all_sync(0xffffffffu, see[c]) ? 0u : 1u << c;
                if (!mbar_wait(&h_empty[hs], ((step / kHideSteps) & 1) ^ 1, a.status, kErrAttnWait, abort_flag))
                    break;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    bounds[hs * kTile + 32 * c + lane] = see[c] ? INFINITY : -INFINITY;
                if (lane == 0)
                    maskeds[hs] = masked;
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&h_full[hs]);
            }
        }
    } else if (warp >= 4) {
        regs_increase<kRegsSoftmax>();
        const int t = (warp - 4) >> 2, w32 = (warp & 3) * 32, r = w32 + lane;
        const uint32_t lanes = tmem + (uint32_t(w32) << 16);
        const uint32_t ts = lanes + t * 128, to = lanes + 256 + t * 128;
        uint32_t ns = 0, no = 0, step = 0;  // S and O tiles taken; key steps of all items so far
        Items<SPLIT> it, nx;  // this item and, worked out while its scores are on their way, the next
        bool ok = true;
        it.first(P);
        for (; it.more(P) && ok; it = nx) {
            nx = it;
            nx.next(P);
            const bool both = SPLIT && it.tiles == 1;  // both groups on one tile, its steps in turn
            if (t >= it.tiles && !both) {
                step += it.hi - it.lo;
                continue;
            }
            const int row0 = it.q0() + (both ? 0 : t * kTile) + w32;  // of the warp
            if (both)
                step = t;
            if (it.n == 0) {  // no keys: zeros, a row's 16-byte pieces side by side
                constexpr int per = D / 8;
                for (int i = lane; i < 32 * per; i += 32) {
                    const long row = row0 + i / per;
                    if (row < a.Lq)
                        *reinterpret_cast<uint4*>(a.out + it.b * a.so.sample + it.h * a.so.head + row * a.so.row +
                                                  i % per * 8) = make_uint4(0, 0, 0, 0);
                }
                continue;
            }
            float m = -INFINITY, l = 0.0f;
            const int stride = both ? 2 : 1, begin = it.lo + (both ? t : 0);
            for (int j = begin; j < it.hi; j += stride, step += stride) {
                const int valid = it.n - j * kTile;
                int tail = valid >= kTile || valid % 32 == 0 ? 32 : valid % 32;
                uint32_t masked = 0;
                const float* bound = bounds + step % kHideSteps * kTile;
                uint64_t* v_here = &v_full[step % kSteps];
                const uint32_t v_phase = (step / kSteps) & 1;
                // Rows of V that are multiplied (those up to valid, in sixteens) and belong to hidden keys: both tiles' threads
                // clear them, whichever comes first. V stays until both tiles' products have read it.
                const auto clear = [&] {
                    if (r < ((valid + 15) & ~15) && (HIDE == kHideMask ? bound[r] < 0.0f : r >= valid)) {
                        uint8_t* row = sKV + (2 * step + 1) % NS * TB + r * 128;
#pragma unroll
                        for (int p = 0; p < D / 64; ++p)
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                *reinterpret_cast<uint4*>(row + p * kPanel + ((i ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                };
                const auto look = [&] {  // the mask's word on this step
                    if (HIDE != kHideMask)
                        return true;
                    const uint32_t s = step % kHideSteps;
                    if (!mbar_wait(&h_full[s], (step / kHideSteps) & 1, a.status, kErrAttnWait, abort_flag))
                        return false;
                    masked = maskeds[s];
                    tail = 32;  // the bounds know of it
                    return true;
                };
                // While the scores are on their way, as far as the mask and V are there. Not where this group may have skipped
                // items: until its scores have come it could then take an older phase of a barrier for its own.
                bool cleared = false;
                if (HIDE == kHideMask && P.in_step) {
                    ok = look();
                    if (ok && (masked || (valid < kTile && it.n < a.Lk)) &&
                        __all_sync(0xffffffffu, mbar_try_wait(smem_u32(v_here), v_phase))) {
                        clear();
                        cleared = true;
                    }
                }
                if (!ok || !mbar_wait(&s_full[t], ns & 1, a.status, kErrAttnWait, abort_flag)) {
                    ok = false;
                    break;
                }
                ++ns;
                tc_fence_after();
                if (HIDE == kHideMask && !P.in_step && !look()) {
                    ok = false;
                    break;
                }
                switch (min(4, (valid + 31) >> 5)) {
                case 1: softmax_step<D, 1>(ts, to, tail, masked, bound, a.scale_log2, j == begin, m, l); break;
                case 2: softmax_step<D, 2>(ts, to, tail, masked, bound, a.scale_log2, j == begin, m, l); break;
                case 3: softmax_step<D, 3>(ts, to, tail, masked, bound, a.scale_log2, j == begin, m, l); break;
                default: softmax_step<D, 4>(ts, to, tail, masked, bound, a.scale_log2, j == begin, m, l); break;
                }
                if (HIDE && !cleared && (masked || (valid < kTile && it.n < a.Lk))) {
                    if (!mbar_wait(v_here, v_phase, a.status, kErrAttnWait, abort_flag)) {
                        ok = false;
                        break;
                    }
                    clear();
                }
                tc_fence_before();
                mbar_arrive(&p_full[t]);
            }
            if (!ok || (begin < it.hi && !mbar_wait(&o_full[t], no & 1, a.status, kErrAttnWait, abort_flag))) {
                ok = false;
                break;
            }
            tc_fence_after();
            if constexpr (SPLIT) {  // merged below
                part_m = m;
                part_l = l;
                part_here = true;
                part_any = begin < it.hi;
                break;
            }
            ++no;
            uint8_t* stage = sO + t * kPanel + w32 * 128;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
            for (int p = 0; p < D / 64; ++p) {
                uint32_t o[64];
                tmem_ld32(to + p * 64, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
                tmem_ld32(to + p * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&o[32]));
                tmem_wait_ld();
                if (lane == 0)
                    bulk_wait_read<0>();  // the warp's last store has read the stage
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(
                        pack_bf16x2(__uint_as_float(o[8 * i]) * inv, __uint_as_float(o[8 * i + 1]) * inv),
                        pack_bf16x2(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv),
                        pack_bf16x2(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv),
                        pack_bf16x2(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv));
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (row0 < a.Lq)
                        tma_store_4d(&P.to, stage, p * 64, row0, it.h * P.o_head, it.b * P.o_sample);
                    bulk_commit();
                }
                __syncwarp();
            }
            tc_fence_before();  // O has been read before the P that lets the next item's product overwrite it
        }
        if (lane == 0)
            bulk_wait_all();  // the last rows are written before the CTA and its shared memory go
    }

    if constexpr (SPLIT) {
        // Each CTA holds, for every row, its part's maximum m, sum l and O (two parts where both groups shared a tile). With M
        // the largest m, the row's result is sum O 2^(m - M) / sum l 2^(m - M). The tiles' valid rows are dealt out over the
        // CTAs; every CTA sends its scaled rows to their owners, and those add and write them. The stages' memory takes the
        // parts: all products that read it are done (o_full) before the first cluster barrier.
        const int S = P.splits, me = int(cluster_ctarank());
        const int t = max((warp - 4) >> 2, 0), r = (warp & 3) * 32 + lane;
        Items<true> it;
        it.first(P);
        const bool both = it.tiles == 1;
        const int q0 = it.q0() + (both ? 0 : t * kTile), rows = min(kTile, a.Lq - q0);
        const int per = (kTile + S - 1) / S;                             // owned rows at most
        float* parts = reinterpret_cast<float*>(smem);                    // [tiles][S][per][D]
        float* ml = reinterpret_cast<float*>(smem) + 2 * (S * per * D);  // [tiles][S][kTile][2]
        // The parts of this group's rows: S of its own tile, or the 2 S of both.
        const int from = both ? 0 : t * S, to_part = both ? 2 * S : from + S;
        __syncwarp();
        __syncthreads();
        cluster_sync_all();
        if (part_here && r < rows)
            for (int o = 0; o < S; ++o) {
                const uint32_t at = map_to_cta(smem_u32(ml + ((t * S + me) * kTile + r) * 2), o);
                st_cluster_f32(at, part_m);
                st_cluster_f32(at + 4, part_l);
            }
        cluster_sync_all();
        if (part_here && __any_sync(0xffffffffu, r < rows)) {
            float M = -INFINITY, L = 0.0f;
            for (int o = from; o < to_part && r < rows; ++o)
                M = fmaxf(M, ml[(o * kTile + r) * 2]);
            const auto weight = [&](float m) { return m == -INFINITY ? 0.0f : ex2(m - M); };
            for (int o = from; o < to_part && r < rows; ++o) {
                const float* e = ml + (o * kTile + r) * 2;
                L += e[1] * weight(e[0]);
            }
            // A part without a visible key adds nothing (its O may never have been written); NaN parts stay NaN.
            const bool add = part_any && !(part_m == -INFINITY && part_l == 0.0f);
            const float f = weight(part_m) * (L == 0.0f ? 0.0f : 1.0f / L);
            int owner = 0;  // of row r: rows * owner / S <= r < rows * (owner + 1) / S
            while (owner + 1 < S && rows * (owner + 1) / S <= r)
                ++owner;
            const int lr = r - rows * owner / S;
            const uint32_t dst = map_to_cta(smem_u32(parts + ((t * S + me) * per + lr) * D), owner);
            const uint32_t to = tmem + (uint32_t((warp & 3) * 32) << 16) + 256 + t * 128;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
                uint32_t v[16];
                tmem_ld16(to + c, v);
                tmem_wait_ld();
                if (r < rows) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        st_cluster_f32x4(dst + (c + i) * 4,
                                         add ? make_float4(__uint_as_float(v[i]) * f, __uint_as_float(v[i + 1]) * f,
                                                           __uint_as_float(v[i + 2]) * f, __uint_as_float(v[i + 3]) * f)
                                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f));
                }
            }
        }
        __syncwarp();
        cluster_sync_all();
        if (part_here) {
            const int first = rows * me / S, count = rows * (me + 1) / S - first;
            __nv_bfloat16* out = a.out + it.b * a.so.sample + it.h * a.so.head;
            for (int i = r + (both ? t * kTile : 0); i < count * (D / 8); i += both ? 2 * kTile : kTile) {
                const int lr = i / (D / 8), c = i % (D / 8) * 8;
                float4 x = make_float4(0, 0, 0, 0), y = x;
#pragma unroll 1
                for (int o = from; o < to_part; ++o) {
                    const float4* e = reinterpret_cast<const float4*>(parts + (o * per + lr) * D + c);
                    const float4 u = e[0], v = e[1];
                    x = make_float4(x.x + u.x, x.y + u.y, x.z + u.z, x.w + u.w);
                    y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
                }
                *reinterpret_cast<uint4*>(out + long(q0 + first + lr) * a.so.row + c) =
                    make_uint4(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w), pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------------------ few query rows

constexpr int kFewRows = 4;    // query rows that share a key head
constexpr int kFewWarps = 8;
// K and V rows a lane takes a round, each, and the rounds in flight: 64 KB a CTA, so that three of one or two rows fit an SM
// (96 KB: 27 against 22 us at 2 x 24 heads of 128 over 4096 keys). Several query rows leave registers for two rows a round (two rows: 23 against 29 us).
template <int R>
struct FewCfg {
    static constexpr int kDepth = R == 1 ? 4 : 2, kRounds = 8 / kDepth;
};
constexpr int kFewSmem = kFewWarps * 8 * 2 * 32 * 16;  // a warp's rounds: [round][K, V][depth][lane] of 16 bytes

// 16 bytes to shared memory behind the thread's back; zeros where `on` is false (nothing is read).
__device__ __forceinline__ void copy16(void* dst, const void* src, bool on)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0)
                 : "memory");
}

__device__ __forceinline__ void unpack8(uint4 u, float (&f)[8])
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// A few query rows of the heads that share a key head: with so few, K and V pass the CUDA cores once and HBM is the bound. A
// cluster takes one (sample, key head), each CTA a run of its keys; D / 8 lanes take a key, 8 values each, so that a warp's
// load is whole rows. Each lane copies what it will use itself into shared memory ahead of its use (in registers alone too
// little is in flight where there are few CTAs: 28 against 17 us at 8 heads of 128 over 8192 keys). Each warp keeps its own
// running maximum, sum and outputs; the warps' parts meet in shared memory, the CTAs' in the first CTA's.
template <int D, int R>
__global__ void __launch_bounds__(32 * kFewWarps) k_cross_few(const CrossArgs a, int splits)
{
    constexpr int kLanes = D / 8, kKeys = 32 / kLanes;  // lanes a key, keys a load
    constexpr int kFewDepth = FewCfg<R>::kDepth, kFewRounds = FewCfg<R>::kRounds;
    __shared__ float po[kFewWarps][R][D];
    __shared__ float pm[kFewWarps][R], pl[kFewWarps][R];
    grid_dep_wait();
    grid_dep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = splits > 1 ? int(cluster_ctarank()) : 0, pair = blockIdx.x / splits;
    const int b = pair / a.Hkv, hk = pair % a.Hkv, group = a.H / a.Hkv, rows = group * a.Lq;
    const int n = a.key_len ? min(max(__ldg(a.key_len + b), 0), a.Lk) : a.Lk;
    const int lo = int(long(n) * part / splits), hi = int(long(n) * (part + 1) / splits);
    const int dim = lane % kLanes * 8;  // of this lane
    const auto head = [&](int r) { return hk * group + r / a.Lq; };

    float q[R][8], o[R][8] = {}, m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < rows)
            u = __ldg(reinterpret_cast<const uint4*>(a.q + b * a.sq.sample + head(r) * a.sq.head + r % a.Lq * a.sq.row + dim));
        unpack8(u, q[r]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            q[r][i] *= a.scale_log2;
    }
    const __nv_bfloat16* kb = a.k + b * a.sk.sample + hk * a.sk.head + dim;
    const __nv_bfloat16* vb = a.v + b * a.sv.sample + hk * a.sv.head + dim;
    const uint8_t* mask = a.key_mask ? a.key_mask + b * a.mask_stride : nullptr;
    extern __shared__ __align__(16) uint4 few_ring[];
    uint4* ring = few_ring + warp * (kFewRounds * 2 * kFewDepth * 32) + lane;
    constexpr int kRound = kFewWarps * kKeys * kFewDepth;  // keys a round of the CTA
    const int first = lo + warp * kKeys + lane / kLanes;   // this lane's first key
    // Which of a round's keys are visible, a bit each.
    const auto look = [&](int j0) {
        uint32_t see = 0;
#pragma unroll
        for (int u = 0; u < kFewDepth; ++u) {
            const int j = j0 + u * kFewWarps * kKeys;
            if (j < hi && (!mask || __ldg(mask + j) != 0))
                see |= 1u << u;
        }
        return see;
    };
    const auto fetch = [&](int slot, int j0, uint32_t see) {
        uint4* dst = ring + slot * (2 * kFewDepth * 32);
#pragma unroll
        for (int u = 0; u < kFewDepth; ++u) {
            const bool on = (see >> u) & 1;
            const long j = on ? j0 + u * kFewWarps * kKeys : 0;
            copy16(dst + u * 32, kb + j * a.sk.row, on);
            copy16(dst + (kFewDepth + u) * 32, vb + j * a.sv.row, on);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // sees: the rounds in flight, four bits each, the next to come lowest; ahead: of the round to be fetched next, looked up
    // a round early.
    uint32_t sees = 0;
#pragma unroll
    for (int i = 0; i < kFewRounds - 1; ++i) {
        const uint32_t see = look(first + i * kRound);
        sees |= see << (4 * i);
        fetch(i, first + i * kRound, see);
    }
    uint32_t ahead = look(first + (kFewRounds - 1) * kRound);
    int slot = 0;
    for (int j0 = first; j0 - lane / kLanes < hi; j0 += kRound) {
        const int next = j0 + (kFewRounds - 1) * kRound;
        fetch(slot == 0 ? kFewRounds - 1 : slot - 1, next, ahead);
        sees |= ahead << (4 * (kFewRounds - 1));
        ahead = look(next + kRound);
        asm volatile("cp.async.wait_group %0;" ::"n"(kFewRounds - 1) : "memory");
        uint4 ku[kFewDepth], vu[kFewDepth];
        bool see[kFewDepth];
#pragma unroll
        for (int u = 0; u < kFewDepth; ++u) {
            see[u] = (sees >> u) & 1;
            ku[u] = ring[(slot * 2 * kFewDepth + u) * 32];
            vu[u] = ring[(slot * 2 * kFewDepth + kFewDepth + u) * 32];
        }
        sees >>= 4;
        slot = slot == kFewRounds - 1 ? 0 : slot + 1;
        float s[kFewDepth][R];
#pragma unroll
        for (int u = 0; u < kFewDepth; ++u) {
            float k[8];
            unpack8(ku[u], k);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float x = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x = fmaf(q[r][i], k[i], x);
                s[u][r] = x;
            }
        }
#pragma unroll
        for (int w = kLanes / 2; w > 0; w >>= 1)
#pragma unroll
            for (int u = 0; u < kFewDepth; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    s[u][r] += __shfl_xor_sync(0xffffffffu, s[u][r], w);
        float shift[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = m[r];
#pragma unroll
            for (int u = 0; u < kFewDepth; ++u) {
                if (!see[u])
                    s[u][r] = -INFINITY;
                top = fmaxf(top, s[u][r]);
            }
#pragma unroll
            for (int w = 16; w >= kLanes; w >>= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float f = m[r] == -INFINITY ? 0.0f : ex2(m[r] - top);
            m[r] = top;
            shift[r] = top == -INFINITY ? 0.0f : top;  // no visible key yet: 2^(-inf - 0) = 0
            l[r] *= f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                o[r][i] *= f;
        }
#pragma unroll
        for (int u = 0; u < kFewDepth; ++u) {
            float v[8];
            unpack8(vu[u], v);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float p = ex2(s[u][r] - shift[r]);
                l[r] += p;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    o[r][i] = fmaf(p, v[i], o[r][i]);
            }
        }
    }
    // Sum over the keys that the warp's lane groups took; every lane of a group has the same l.
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int w = 16; w >= kLanes; w >>= 1) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                o[r][i] += __shfl_xor_sync(0xffffffffu, o[r][i], w);
        }
        if (lane < kLanes) {
#pragma unroll
            for (int i = 0; i < 8; i += 4)
                *reinterpret_cast<float4*>(&po[warp][r][dim + i]) = make_float4(o[r][i], o[r][i + 1], o[r][i + 2], o[r][i + 3]);
        }
        if (lane == 0) {
            pm[warp][r] = m[r];
            pl[warp][r] = l[r];
        }
    }
    __syncthreads();
    // The parts of `count` warps or CTAs to one: element e of R * D, with the row's maximum and sum.
    const auto join = [&](int count, int e, float& M, float& L) {
        const int r = e / D;
        M = -INFINITY;
        for (int w = 0; w < count; ++w)
            M = fmaxf(M, pm[w][r]);
        float x = 0.0f;
        L = 0.0f;
        for (int w = 0; w < count; ++w) {
            const float f = pm[w][r] == -INFINITY ? 0.0f : ex2(pm[w][r] - M);
            L = fmaf(pl[w][r], f, L);
            x = fmaf(po[w][r][e % D], f, x);
        }
        return x;
    };
    constexpr int kPer = (R * D + 32 * kFewWarps - 1) / (32 * kFewWarps);
    float x[kPer], M[kPer], L[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = threadIdx.x + i * 32 * kFewWarps;
        if (e < R * D)
            x[i] = join(kFewWarps, e, M[i], L[i]);
    }
    if (splits > 1) {
        __syncthreads();
        cluster_sync_all();  // every CTA has read its warps' parts
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = threadIdx.x + i * 32 * kFewWarps;
            if (e < R * D) {
                st_cluster_f32(map_to_cta(smem_u32(&po[part][e / D][e % D]), 0), x[i]);
                if (e % D == 0) {
                    st_cluster_f32(map_to_cta(smem_u32(&pm[part][e / D]), 0), M[i]);
                    st_cluster_f32(map_to_cta(smem_u32(&pl[part][e / D]), 0), L[i]);
                }
            }
        }
        cluster_sync_all();
        if (part)
            return;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = threadIdx.x + i * 32 * kFewWarps;
            if (e < R * D)
                x[i] = join(splits, e, M[i], L[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = threadIdx.x + i * 32 * kFewWarps, r = e / D;
        if (e < R * D && r < rows)
            a.out[b * a.so.sample + head(r) * a.so.head + r % a.Lq * a.so.row + e % D] =
                __float2bfloat16(x[i] * (L[i] == 0.0f ? 0.0f : 1.0f / L[i]));
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

// [samples][heads][rows][d] with its strides as a 4-D map, box 64 x box_rows with the 128-byte swizzle; rows past the
// tensor read as zeros. A shared dimension (stride 0) is one element long and its use flag 0.
bool encode_heads(CUtensorMap* m, const void* p, const HeadStrides& s, int rows, int heads, int samples, int d, int box_rows,
                  int* use_head, int* use_sample)
{
    auto fn = encode_fn();
    *use_head = heads > 1 && s.head > 0;
    *use_sample = samples > 1 && s.sample > 0;
    const cuuint64_t dims[4] = {cuuint64_t(d), cuuint64_t(std::max(rows, 1)), cuuint64_t(*use_head ? heads : 1),
                                cuuint64_t(*use_sample ? samples : 1)};
    const cuuint64_t strides[3] = {cuuint64_t(s.row) * 2, cuuint64_t(*use_head ? s.head : s.row) * 2,
                                   cuuint64_t(*use_sample ? s.sample : s.row) * 2};
    const cuuint32_t box[4] = {64, cuuint32_t(box_rows), 1, 1}, es[4] = {1, 1, 1, 1};
    return fn && fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A one-time check that the compiled register count holds the warpgroups' split (otherwise the softmax groups' increase
// could never be granted), and the shared memory limit on each device.
template <int D, bool SPLIT, int HIDE>
cudaError_t setup()
{
    static const cudaError_t regs = [] {
        cudaFuncAttributes fa{};
        const cudaError_t e = cudaFuncGetAttributes(&fa, k_cross<D, SPLIT, HIDE>);
        if (e != cudaSuccess)
            return e;
        return fa.numRegs * kThreads < 128 * kRegsCtl + 256 * kRegsSoftmax ? cudaErrorInvalidConfiguration
                                                                          : cudaSuccess;
    }();
    if (regs != cudaSuccess)
        return regs;
    static std::atomic<uint64_t> devs{0};
    return smem_limit_once(devs, k_cross<D, SPLIT, HIDE>, Cfg<D, SPLIT>::kSmem);
}

// Clusters of `size` CTAs of the split kernel that the current device runs at once (they have to fit its GPCs), kept for
// devices 0..63 once asked.
template <int D>
int clusters_at_once(int size)
{
    static std::atomic<int> known[64][kMaxSplits + 1];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess)
        return 0;
    const bool keep = dev >= 0 && dev < 64;
    if (keep && known[dev][size].load(std::memory_order_relaxed))
        return known[dev][size].load(std::memory_order_relaxed);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<D, true>::kSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = size;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (setup<D, true, kHideMask>() != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, k_cross<D, true, kHideMask>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (keep)
        known[dev][size].store(n, std::memory_order_relaxed);
    return n;
}

// CTAs an item: as many as run at once for all items, with two key steps each or more; 1 where that is not even two.
template <int D>
int splits_of(int items, int steps)
{
    for (int s = std::min({kMaxSplits, num_sms() / items, steps / 2}); s > 1; --s)
        if (clusters_at_once<D>(s) >= items)
            return s;
    return 1;
}

template <int D, int HIDE>
cudaError_t launch(const CrossParams& P, cudaStream_t st)
{
    if (P.splits > 1) {
        const cudaError_t e = setup<D, true, HIDE>();
        return e != cudaSuccess ? e
                                : launch_k_cluster(k_cross<D, true, HIDE>, dim3(P.items * P.splits), P.splits, kThreads,
                                                   Cfg<D, true>::kSmem, st, P);
    }
    const cudaError_t e = setup<D, false, HIDE>();
    return e != cudaSuccess ? e
                            : launch_k(k_cross<D, false, HIDE>, dim3(std::min(P.items, num_sms())), kThreads,
                                       Cfg<D, false>::kSmem, st, P);
}

template <int D>
cudaError_t launch(const CrossParams& P, cudaStream_t st)
{
    return P.a.key_mask  ? launch<D, kHideMask>(P, st)
           : P.a.key_len ? launch<D, kHideLengths>(P, st)
                         : launch<D, kHideNone>(P, st);
}

// k_cross_few CTAs that an SM of the current device holds: three, but two of four rows' (128 registers a thread, and at D = 128
// the warps' parts take 16 KB beside the rounds). Kept for devices 0..63 once asked.
template <int D, int R>
int few_at_once()
{
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess)
        return 1;
    const bool keep = dev >= 0 && dev < 64;
    if (keep && known[dev].load(std::memory_order_relaxed))
        return known[dev].load(std::memory_order_relaxed);
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_cross_few<D, R>, 32 * kFewWarps, kFewSmem) != cudaSuccess) {
        cudaGetLastError();
        return 1;
    }
    n = std::max(1, n);
    if (keep)
        known[dev].store(n, std::memory_order_relaxed);
    return n;
}

template <int D, int R>
cudaError_t launch_few(const CrossArgs& a, cudaStream_t st)
{
    static std::atomic<uint64_t> devs{0};
    const cudaError_t e = smem_limit_once(devs, k_cross_few<D, R>, kFewSmem);
    if (e != cudaSuccess)
        return e;
    // The keys over as many CTAs as the SMs hold at once, 128 keys a CTA or more (more than that leave a second wave: 128 key
    // heads of 4096 keys 61 against 51 us, 148 of 512 keys with four rows each 24.7 against 16.4; the size that divides the CTAs most evenly over the SMs instead, 6 for 8 at 48 key
    // heads, was slower: 23.6 against 22.4 us).
    const int pairs = a.B * a.Hkv;
    const int splits = std::max(1, std::min({kMaxSplits, kFewWarps, few_at_once<D, R>() * num_sms() / pairs, a.Lk / 128}));
    return launch_k_cluster(k_cross_few<D, R>, dim3(pairs * splits), splits, 32 * kFewWarps, kFewSmem, st, a, splits);
}

template <int D>
cudaError_t launch_few(const CrossArgs& a, cudaStream_t st)
{
    const int rows = a.H / a.Hkv * a.Lq;
    return rows == 1   ? launch_few<D, 1>(a, st)
           : rows == 2 ? launch_few<D, 2>(a, st)
                       : launch_few<D, 4>(a, st);
}

}  // namespace

cudaError_t cross_attention(const CrossArgs& args, const char** err, cudaStream_t st)
{
    CrossArgs a = args;
    if (a.Lk == 0) {  // no key is read; addresses are still made
        a.k = a.v = a.q;
        a.sk = a.sv = HeadStrides{a.d, 0, 0};
    }
    // The CUDA cores keep up with HBM for one or two rows; up to four they still win where the keys are few (four rows over 4096
    // keys of 48 heads: 46 against 29 us).
    const long few = long(a.H / a.Hkv) * a.Lq;
    if (few <= 2 || (few <= kFewRows && a.Lk <= 512)) {
        const cudaError_t e = a.d == 64 ? launch_few<64>(a, st) : launch_few<128>(a, st);
        if (e != cudaSuccess)
            return e;
        count_launch();
        return cudaGetLastError();
    }
    CrossParams P;
    P.a = a;
    P.blocks = (a.Lq + 2 * kTile - 1) / (2 * kTile);
    P.items = a.B * a.H * P.blocks;
    P.in_step = a.Lq > kTile && (a.Lq - 1) % (2 * kTile) >= kTile;
    const int steps = (a.Lk + kTile - 1) / kTile;
    P.splits = a.d == 64 ? splits_of<64>(P.items, steps) : splits_of<128>(P.items, steps);
    if (!encode_heads(&P.tq, a.q, a.sq, a.Lq, a.H, a.B, a.d, kTile, &P.q_head, &P.q_sample) ||
        !encode_heads(&P.tk, a.k, a.sk, a.Lk, a.Hkv, a.B, a.d, kTile, &P.kv_head_k, &P.kv_sample_k) ||
        !encode_heads(&P.tv, a.v, a.sv, a.Lk, a.Hkv, a.B, a.d, kTile, &P.kv_head_v, &P.kv_sample_v) ||
        !encode_heads(&P.to, a.out, a.so, a.Lq, a.H, a.B, a.d, 32, &P.o_head, &P.o_sample)) {
        *err = "cross_attention: tensor map encoding failed";
        return cudaErrorInvalidValue;
    }
    const cudaError_t e = a.d == 64 ? launch<64>(P, st) : launch<128>(P, st);
    if (e != cudaSuccess)
        return e;
    count_launch();
    return cudaGetLastError();
}

}  // namespace mkb
