// Attention to another stream's keys (see cross_attention.cuh) on tcgen05.
//
// Keys are few and queries many, so the work is a stream of query tiles past small sets of keys: persistent CTAs walk
// items of (sample, head, 256 query rows) as two 128-row tiles A and B, and every stage runs ahead into the next item, so
// that one item's loads, another's products and a third's stores overlap. Twelve warps:
//   warp 0     TMA: Q tiles (double-buffered) and K and V tiles of 128 keys into one ring
//   warp 1     MMA: S = Q K^T, then O += P V with P in tensor memory, for A and B in turn
//   warp 2     with key lengths or masks: clears the V rows of keys that no query sees (0 * NaN would spread)
//   warps 4-7  softmax of tile A, 8-11 of tile B: a thread a row, the running maximum and sum of one pass
// Only ceil(visible / 16) * 16 keys of the last tile are multiplied and exponentiated (77 keys cost 80, not 128).
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

namespace mkb {

namespace {

constexpr int kThreads = 384;
// The launch gives every thread 168 registers; the control warpgroup drops to kRegsCtl and the softmax warpgroups rise to
// kRegsSoftmax, enough for a row's 128 scores.
constexpr int kLaunchRegs = (65536 / kThreads) / 8 * 8;
constexpr int kRegsCtl = 56, kRegsSoftmax = 216;
static_assert(128 * kRegsCtl + 256 * kRegsSoftmax <= kThreads * kLaunchRegs, "register split exceeds the CTA pool");
constexpr int kTile = 128;              // query rows a tile, keys a tile
constexpr int kPanel = kTile * 64 * 2;  // 64 bf16 columns of 128 rows
constexpr int kSteps = 4;               // full barriers of K and of V: no more key steps than that are ever in flight
constexpr float kRescaleThreshold = 8.0f;  // log2 units: O is rescaled only when a row's maximum grows by more

template <int D>
struct Cfg {
    static constexpr int kTileBytes = (D / 64) * kPanel;
    static constexpr int kSlots = D == 64 ? 8 : 3;  // K and V tiles in flight beside the four Q tiles
    static constexpr int kSmem = 1024 + (4 + kSlots) * kTileBytes + 512;
    static_assert(kSmem <= 227 * 1024);
    static_assert((kSlots + 1) / 2 <= kSteps);
};

struct CrossParams {
    CUtensorMap tq, tk, tv;
    CrossArgs a;
    // 0 where a dimension is shared (stride 0): its coordinate stays 0.
    int q_head, q_sample, kv_head_k, kv_sample_k, kv_head_v, kv_sample_v;
    int items, blocks;  // work items, query blocks of 256 rows
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One (sample, head, query block) and its keys.
struct Item {
    int b, h, q0, n, steps, tiles;  // n: keys up to the last that may be visible; steps of 128; 1 or 2 query tiles
    __device__ __forceinline__ void set(const CrossParams& P, int item)
    {
        const CrossArgs& a = P.a;
        const int bh = item / P.blocks;
        q0 = (item - bh * P.blocks) * 2 * kTile;
        b = bh / a.H;
        h = bh - b * a.H;
        n = a.key_len ? min(max(__ldg(a.key_len + b), 0), a.Lk) : a.Lk;
        steps = (n + kTile - 1) / kTile;
        tiles = q0 + kTile < a.Lq ? 2 : 1;
    }
};

// The walk over all key steps of a CTA's items that have keys.
struct Walk {
    Item it;
    int item, j;
    __device__ __forceinline__ void settle(const CrossParams& P)  // on to an item with keys
    {
        j = 0;
        for (; item < P.items; item += gridDim.x) {
            it.set(P, item);
            if (it.steps > 0)
                return;
        }
    }
    __device__ __forceinline__ void first(const CrossParams& P)
    {
        item = blockIdx.x;
        settle(P);
    }
    __device__ __forceinline__ void next(const CrossParams& P)
    {
        if (++j == it.steps) {
            item += gridDim.x;
            settle(P);
        }
    }
    __device__ __forceinline__ bool more(const CrossParams& P) const { return item < P.items; }
    __device__ __forceinline__ bool last() const { return j + 1 == it.steps; }
    // Keys of the step that are multiplied: those up to n, in sixteens.
    __device__ __forceinline__ int width() const { return min(kTile, (it.n - j * kTile + 15) & ~15); }
};

// Bit i of the 32 keys from `key` on: visible (below n and not masked). All lanes of a warp take part and get the word.
__device__ __forceinline__ uint32_t visible_word(const CrossArgs& a, int b, int n, int key)
{
    const int left = n - key;
    uint32_t w = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1;
    if (a.key_mask) {
        const int k = key + int(threadIdx.x & 31);
        w &= __ballot_sync(0xffffffffu, k < n && __ldg(a.key_mask + b * a.mask_stride + k) != 0);
    }
    return w;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) k_cross(const __grid_constant__ CrossParams P)
{
    using C = Cfg<D>;
    constexpr int TB = C::kTileBytes, NS = C::kSlots;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;            // [2 buffers][2 tiles]
    uint8_t* sKV = smem + 4 * TB;  // [slots]
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (4 + NS) * TB);
    uint64_t* q_full = bars;             // [2 buffers][2 tiles]
    uint64_t* q_empty = q_full + 4;      // [2 buffers][2 tiles]
    uint64_t* kv_empty = q_empty + 4;    // [slots]
    // By key step, not by slot: where K and V take turns in a slot, a warp that follows only the V tiles would miss phases
    // of the slot's barrier.
    uint64_t* k_full = kv_empty + NS;    // [kSteps]
    uint64_t* v_full = k_full + kSteps;  // [kSteps]
    uint64_t* v_ready = v_full + kSteps; // [kSteps] V with its unseen rows cleared
    uint64_t* s_full = v_ready + kSteps; // [tiles]
    uint64_t* p_full = s_full + 2;       // [tiles]
    uint64_t* o_full = p_full + 2;       // [tiles]
    uint64_t* drain = o_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const CrossArgs& a = P.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const bool clear_v = a.key_len || a.key_mask;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < NS; ++i)
            mbar_init(&kv_empty[i], 1);
        for (int i = 0; i < kSteps; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_ready[i], 1);
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
            Walk w;
            uint32_t seq = 0, nq[2] = {0, 0};  // ring position; Q tiles issued of A and B
            bool ok = true;
            const auto load = [&](uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int row, int h, int b) {
                mbar_arrive_expect_tx(bar, TB);
#pragma unroll
                for (int p = 0; p < D / 64; ++p)
                    tma_load_4d(dst + p * kPanel, m, bar, p * 64, row, h, b);
            };
            for (w.first(P); w.more(P) && ok; w.next(P)) {
                const int hk = w.it.h / (a.H / a.Hkv);
                if (w.j == 0)
                    for (int t = 0; t < w.it.tiles && ok; ++t) {
                        const uint32_t buf = nq[t] & 1, i = buf * 2 + t;
                        ok = mbar_wait(&q_empty[i], ((nq[t] >> 1) & 1) ^ 1, a.status, kErrAttnWait, abort_flag);
                        if (ok) {
                            load(sQ + i * TB, &P.tq, &q_full[i], w.it.q0 + t * kTile, w.it.h * P.q_head,
                                 w.it.b * P.q_sample);
                            ++nq[t];
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
                for (int t = 0; t < 2; ++t)
                    for (uint32_t i = nq[t] > 2 ? nq[t] - 2 : 0; i < nq[t]; ++i)
                        mbar_wait(&q_full[(i & 1) * 2 + t], (i >> 1) & 1, a.status, kErrWaitDrain, nullptr);
                for (uint32_t i = seq > NS ? seq - NS : 0; i < seq; ++i)
                    mbar_wait(&(i & 1 ? v_full : k_full)[(i >> 1) % kSteps], ((i >> 1) / kSteps) & 1, a.status,
                              kErrWaitDrain, nullptr);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc_s0 = idesc_bf16_f32(128, 0), idesc_o = idesc_bf16_f32(128, D, 0, 1);
            const uint32_t q_addr = smem_u32(sQ), kv_addr = smem_u32(sKV);
            uint32_t seq = 0, nq[2] = {0, 0}, np[2] = {0, 0};  // as the producer's; P tiles taken of A and B
            bool ok = true;
            // S_t of step w, K in slot s. The item's first step waits for Q, its last frees it.
            const auto scores = [&](const Walk& w, int t, uint32_t s) {
                const uint32_t i = (nq[t] & 1) * 2 + t;
                if (w.j == 0 && !mbar_wait(&q_full[i], (nq[t] >> 1) & 1, a.status, kErrAttnWait, abort_flag))
                    return false;
                tc_fence_after();
                const uint32_t idesc = idesc_s0 | uint32_t(w.width() >> 3) << 17;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (k >> 2) * kPanel + (k & 3) * 32;
                    mma_bf16_ss(tmem + t * 128, desc_kmajor_sw128(q_addr + i * TB + off),
                                desc_kmajor_sw128(kv_addr + s * TB + off), idesc, k > 0);
                }
                mma_commit(&s_full[t]);
                if (w.last()) {
                    mma_commit(&q_empty[i]);
                    ++nq[t];
                }
                return true;
            };
            const auto wait_kv = [&](uint64_t* bars, uint32_t step) {
                return mbar_wait(&bars[step % kSteps], (step / kSteps) & 1, a.status, kErrAttnWait, abort_flag);
            };
            Walk w, x;
            w.first(P);
            if (w.more(P)) {
                ok = wait_kv(k_full, 0);
                for (int t = 0; t < w.it.tiles && ok; ++t)
                    ok = scores(w, t, 0);
                if (ok)
                    mma_commit(&kv_empty[0]);
            }
            // Per step: O_A += P_A V, S_A of the next step, then B: one tile's softmax runs under the other's products.
            for (; w.more(P) && ok; w = x, seq += 2) {
                x = w;
                x.next(P);
                const bool more = x.more(P);
                const uint32_t sv = (seq + 1) % NS, sk = (seq + 2) % NS;
                ok = wait_kv(clear_v ? v_ready : v_full, seq >> 1);
                const int tiles = more ? max(w.it.tiles, x.it.tiles) : w.it.tiles;
                for (int t = 0; t < tiles && ok; ++t) {
                    if (t < w.it.tiles) {
                        ok = mbar_wait(&p_full[t], np[t] & 1, a.status, kErrAttnWait, abort_flag);
                        if (!ok)
                            break;
                        ++np[t];
                        tc_fence_after();
                        const int steps = w.width() >> 4;
#pragma unroll 1
                        for (int k = 0; k < steps; ++k)
                            mma_bf16_ts(tmem + 256 + t * 128, tmem + t * 128 + 8 * k,
                                        desc_mnmajor_sw128(kv_addr + sv * TB + k * 2048, kPanel, 1024), idesc_o,
                                        (w.j > 0) || (k > 0));
                        if (w.last())
                            mma_commit(&o_full[t]);
                    }
                    if (more && t == 0)
                        ok = wait_kv(k_full, (seq >> 1) + 1);
                    if (more && ok && t < x.it.tiles)
                        ok = scores(x, t, sk);
                }
                if (!ok)
                    break;
                mma_commit(&kv_empty[sv]);
                if (more)
                    mma_commit(&kv_empty[sk]);
            }
            mma_commit(drain);  // arrives once every MMA issued above has completed
            mbar_wait(drain, 0, a.status, kErrWaitDrain, nullptr);
        }
    } else if (warp == 2) {
        if (clear_v) {
            Walk w;
            uint32_t step = 0;
            for (w.first(P); w.more(P); w.next(P), ++step) {
                const uint32_t s = (2 * step + 1) % NS;
                uint32_t hide[4];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    hide[c] = ~visible_word(a, w.it.b, w.it.n, w.j * kTile + 32 * c);
                if (!mbar_wait(&v_full[step % kSteps], (step / kSteps) & 1, a.status, kErrAttnWait, abort_flag))
                    break;
                const int width = w.width();
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (32 * c < width && hide[c]) {
                        if ((hide[c] >> lane) & 1) {
                            uint8_t* row = sKV + s * TB + (32 * c + lane) * 128;
#pragma unroll
                            for (int p = 0; p < D / 64; ++p)
#pragma unroll
                                for (int i = 0; i < 8; ++i)
                                    *reinterpret_cast<uint4*>(row + p * kPanel + i * 16) = make_uint4(0, 0, 0, 0);
                        }
                    }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&v_ready[step % kSteps]);
            }
        }
    } else if (warp >= 4) {
        regs_increase<kRegsSoftmax>();
        const int t = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
        const uint32_t ts = lanes + t * 128, to = lanes + 256 + t * 128;
        const float sc = a.scale_log2;
        uint32_t ns = 0, no = 0;  // S and O tiles taken
        Item it;
        for (int item = blockIdx.x; item < P.items; item += gridDim.x) {
            it.set(P, item);
            if (t >= it.tiles)
                continue;
            float m = -INFINITY, l = 0.0f;
            bool ok = true;
            for (int j = 0; j < it.steps; ++j) {
                uint32_t see[4];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    see[c] = visible_word(a, it.b, it.n, j * kTile + 32 * c);
                const int chunks = min(4, (it.n - j * kTile + 31) >> 5);
                if (!mbar_wait(&s_full[t], ns & 1, a.status, kErrAttnWait, abort_flag)) {
                    ok = false;
                    break;
                }
                ++ns;
                tc_fence_after();
                uint32_t s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c < chunks)
                        tmem_ld32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
                tmem_wait_ld();
                float mc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c < chunks) {
                        if (see[c] != 0xffffffffu) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!((see[c] >> i) & 1))
                                    s[32 * c + i] = __float_as_uint(-INFINITY);
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
#pragma unroll
                            for (int u = 0; u < 4; ++u)
                                mc[u] = fmax3(mc[u], __uint_as_float(s[32 * c + i + 2 * u]),
                                              __uint_as_float(s[32 * c + i + 2 * u + 1]));
                    }
                const float mx = fmaxf(fmax3(mc[0], mc[1], mc[2]), mc[3]) * sc;
                const bool need = mx > m + kRescaleThreshold;  // also the first tile with a visible key
                if (__any_sync(0xffffffffu, need)) {
                    const float m_new = need ? mx : m;
                    const float f = m == -INFINITY ? 0.0f : ex2(m - m_new);
                    l *= f;
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(to + c * 16, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st16(to + c * 16, o);
                        }
                    }
                    m = m_new;
                }
                // A row that has seen no key yet: 2^(-inf - 0) = 0 for all of them.
                const float shift = m == -INFINITY ? 0.0f : -m;
                const float2 sc2 = make_float2(sc, sc), sh2 = make_float2(shift, shift);
                float2 ls[4] = {};
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c < chunks) {
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
                tc_fence_before();
                mbar_arrive(&p_full[t]);
                const float2 l2 = fadd2(fadd2(ls[0], ls[1]), fadd2(ls[2], ls[3]));
                l += l2.x + l2.y;
            }
            if (!ok)
                break;
            const int row = it.q0 + t * kTile + r;
            __nv_bfloat16* dst = a.out + it.b * a.so.sample + it.h * a.so.head + long(row) * a.so.row;
            const bool in = row < a.Lq;
            if (it.steps == 0) {
                if (in)
#pragma unroll
                    for (int i = 0; i < D / 8; ++i)
                        reinterpret_cast<uint4*>(dst)[i] = make_uint4(0, 0, 0, 0);
                continue;
            }
            if (!mbar_wait(&o_full[t], no & 1, a.status, kErrAttnWait, abort_flag))
                break;
            ++no;
            tc_fence_after();
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(to + c * 32, o);
                tmem_wait_ld();
                if (in) {
                    uint4* d = reinterpret_cast<uint4*>(dst + c * 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        d[i] = make_uint4(
                            pack_bf16x2(__uint_as_float(o[8 * i]) * inv, __uint_as_float(o[8 * i + 1]) * inv),
                            pack_bf16x2(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv),
                            pack_bf16x2(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv),
                            pack_bf16x2(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv));
                }
            }
            tc_fence_before();  // O has been read before the P that lets the next item's product overwrite it
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
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

// [samples][heads][rows][d] with its strides as a 4-D map, box 64 x 128 rows with the 128-byte swizzle; rows past the
// tensor read as zeros. A shared dimension (stride 0) is one element long and its use flag 0.
bool encode_heads(CUtensorMap* m, const void* p, const HeadStrides& s, int rows, int heads, int samples, int d,
                  int* use_head, int* use_sample)
{
    auto fn = encode_fn();
    *use_head = heads > 1 && s.head > 0;
    *use_sample = samples > 1 && s.sample > 0;
    const cuuint64_t dims[4] = {cuuint64_t(d), cuuint64_t(std::max(rows, 1)), cuuint64_t(*use_head ? heads : 1),
                                cuuint64_t(*use_sample ? samples : 1)};
    const cuuint64_t strides[3] = {cuuint64_t(s.row) * 2, cuuint64_t(*use_head ? s.head : s.row) * 2,
                                   cuuint64_t(*use_sample ? s.sample : s.row) * 2};
    const cuuint32_t box[4] = {64, kTile, 1, 1}, es[4] = {1, 1, 1, 1};
    return fn && fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A one-time check that the compiled register count holds the warpgroups' split (otherwise the softmax groups' increase
// could never be granted), and the shared memory limit on each device.
template <int D>
cudaError_t setup()
{
    static const cudaError_t regs = [] {
        cudaFuncAttributes fa{};
        const cudaError_t e = cudaFuncGetAttributes(&fa, k_cross<D>);
        if (e != cudaSuccess)
            return e;
        return fa.numRegs * kThreads < 128 * kRegsCtl + 256 * kRegsSoftmax ? cudaErrorInvalidConfiguration
                                                                          : cudaSuccess;
    }();
    if (regs != cudaSuccess)
        return regs;
    static std::atomic<uint64_t> devs{0};
    return smem_limit_once(devs, k_cross<D>, Cfg<D>::kSmem);
}

template <int D>
cudaError_t launch(const CrossParams& P, cudaStream_t st)
{
    const cudaError_t e = setup<D>();
    if (e != cudaSuccess)
        return e;
    return launch_k(k_cross<D>, dim3(std::min(P.items, num_sms())), kThreads, Cfg<D>::kSmem, st, P);
}

}  // namespace

cudaError_t cross_attention(const CrossArgs& a, const char** err, cudaStream_t st)
{
    CrossParams P;
    P.a = a;
    P.blocks = (a.Lq + 2 * kTile - 1) / (2 * kTile);
    P.items = a.B * a.H * P.blocks;
    const void* k = a.Lk ? a.k : a.q;  // no keys: the maps are not used
    const void* v = a.Lk ? a.v : a.q;
    if (!encode_heads(&P.tq, a.q, a.sq, a.Lq, a.H, a.B, a.d, &P.q_head, &P.q_sample) ||
        !encode_heads(&P.tk, k, a.sk, a.Lk, a.Hkv, a.B, a.d, &P.kv_head_k, &P.kv_sample_k) ||
        !encode_heads(&P.tv, v, a.sv, a.Lk, a.Hkv, a.B, a.d, &P.kv_head_v, &P.kv_sample_v)) {
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
