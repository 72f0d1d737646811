// Attention of long 16-bit prompts over the 4-bit paged cache, on the fifth
// generation tensor cores (tcgen05, sm_100a).
//
// A CTA holds 256 rows (query token x query head of the group) of one kv head
// as two tiles of 128.  Keys come into shared memory 128 at a time, and a tile
// takes 64 of them a step:
//   S_w = Q_w K^T     A: Q in shared memory, B: K, D in tensor memory
//   P_w = 2^(S_w - m) the softmax warps, row by row in a thread
//   O_w += P_w V      A: P in tensor memory (beside S_w, twice), B: V^T
// Warps 0-3 and 4-7 are the softmax of tile 0 and 1, so one tile's
// exponentials run while the other's products do; warps 8-15 turn the next
// keys' 4-bit K and V into halves in shared memory (K as it lies, V
// transposed by interleaving the nibbles of two keys), straight from global
// memory through registers; a thread of warps 16 and 17 each issues a tile's products.  All
// operands are K-major with the 128-byte swizzle.
//
// Roundings.  K and V are exact in half.  fp16 queries stay as they are; bf16
// ones are scaled by a power of two a row, their largest into [2^14, 2^15):
// exact down to 2^-31 of it, and within 2^-39 of it below that.  P is rounded
// once to half, by at most 2^-11 of itself (its sum is taken before): in fp16
// that is the output's own half unit for a row of few keys, and averages out
// over many (2.3e-4 against 2.1e-4 with P in fp32, on 262143 keys); a second
// half for the rest would double the P V products.  The running maximum moves
// only when a logit exceeds it by 2^7, since O has to be read and written back
// then.  What the matrix unit cuts off O: see kAside.
//
// What bounds it, 3 chunks of about 2000 tokens over 4.7k-6.6k keys, 32 heads
// over 8, dim 128, bf16 (464 GFLOP, 281 us at the card's matrix rate): 698 us,
// 665 TFLOP/s.  No unit is full (tensor pipe 32 %, exponentials 33 %, issue
// 50 %; leaving out half the P V products changes nothing, all
// dequantisation 7 %): a step is the softmax warps' chain of about 2600
// clocks for 64 keys (scores' barrier, tensor-memory load, maximum,
// exponentials at 1225, store) with two of its warps a scheduler, and a CTA's
// start and end are 30k of about 230k clocks.  With P over S in tensor memory
// and 128 keys a step, the scores waited for the P V product: 758 us.
//
// Every wait is bounded: one that gives up sets the workspace's error word,
// every role leaves its loop, the rows are written as NaN and the tensor
// memory is freed.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kernels.cuh"
#include "kv4_attention.cuh"
#include "kv4_stage.cuh"
#include "sili_b200.h"

namespace sili {
int set_error(int code, const std::string& msg);
}

namespace {

using namespace sili::mma;
using sili::AttendArgs;
using sili::ex2;
using sili::kLift;
using sili::kLn2;
using sili::kLog2e;
using sili::kSlack;
using sili::mul2;
using sili::pack2;

#define CKP(x)                                                                                          \
    do {                                                                                                \
        const cudaError_t e_ = (x);                                                                     \
        if (e_ != cudaSuccess) return sili::set_error(SILI_ECUDA, std::string(#x) + ": " + cudaGetErrorString(e_)); \
    } while (0)

constexpr int kM = 128;               // rows of a tile (MMA M)
constexpr int kTiles = 2;
constexpr int kSub = 64;              // keys a step of a tile (MMA N of S, K of P V)
constexpr int kSoftmax = kTiles * 128, kDequant = 256;
constexpr int kThreads = kSoftmax + kDequant + 128;     // whole warpgroups: each sets its share of the registers
// registers a thread after the split; together what the launch holds: 96 * 640
constexpr int kRegsSoftmax = 144, kRegsDequant = 72, kRegsRest = 48;
static_assert(kSoftmax * kRegsSoftmax + kDequant * kRegsDequant + 128 * kRegsRest <= 96 * kThreads, "register split");
constexpr int kMmaWarp = (kSoftmax + kDequant) / 32;
// Steps after which a row tile's O leaves tensor memory.  The matrix unit cuts what it adds to an accumulator towards
// zero: with V of one sign the output was short by 6e-9 a key, 1.6e-3 over 262144 keys.  So long rows' sums are added
// outside, rounded, in a slot of the workspace: every 16384 keys in fp16, 65536 in bf16, which leaves a fifth of the
// output's half unit (1e-4, 4e-4).  1184 queries of 32 heads over 8, dim 128, over 262144 keys: 11.9 ms in bf16, 12.1 in
// fp16, 11.5 with the sums left where they were; up to 16384 keys the same.
template <typename T>
constexpr int kAside = std::is_same<T, __half>::value ? 256 : 1024;
constexpr int kPolls = 4096;          // polls of a wait, each asleep for up to kNap ns, before it gives up
std::atomic<int> g_polls{kPolls}, g_output_polls{kPolls};     // sili_kv4_attention_wait_limit

template <int D>
struct Smem {
    alignas(1024) uint8_t q[kTiles][kM * D * 2];
    alignas(1024) uint8_t k[2][kKeys * D * 2];
    alignas(1024) uint8_t v[2][kKeys * D * 2];
    alignas(8) unsigned long long kv_full[2], kv_free[2];                                  // by stage
    unsigned long long s_full[2], s_free[2], p_free[2], o_full[2], drained[2];   // by tile
    // by tile and the step's parity: a warp may be a step ahead of its tile's others, and must not count for their step
    unsigned long long p_full[2][2];
    uint8_t odd_keys[2][16][4];       // [stage][8 keys][group]: bits of keys whose V scale is not a number
    int odd[2];                       // the last stage that had any, plus one
    alignas(8) uint8_t there[2][8];   // [stage][16 keys]: their page exists
    uint32_t tmem;
    int dead;
    int hit[3];                       // the CTA's request, kv head and row tile pair
    int slot;                         // of the workspace, for rows of more than kAside steps; -1: none
};

// What every role knows of the CTA's work.
struct Work {
    int r, h, group, rows, row0, len;
    int64_t pos0;          // position of the request's first query
    int j0, last;              // stages [j0, last) of keys
    int n[kTiles];             // each tile's steps, from stage j0 on

    __device__ __forceinline__ int64_t pos_of(int row) const { return pos0 + min(row, rows - 1) / group; }
};

struct Span {
    int row0, nq, len, pairs;
    int64_t pos0;
};
__device__ __forceinline__ Span span_of(const AttendArgs& a, int r) {
    Span q;
    const int64_t s0 = min(max((int64_t)a.starts[r], (int64_t)0), a.tokens);
    const int64_t past = a.starts[r + 1], s1 = min(max(past, s0), a.tokens);     // (rows that q lacks keep their positions)
    const int all = max(a.lens[r], 0);
    q.row0 = (int)s0;
    q.nq = (int)(s1 - s0);
    q.len = (int)min(min((int64_t)all, (int64_t)a.width * a.page), (int64_t)0x7FFFFF00);
    q.pos0 = all - (past - s0);
    q.pairs = (q.nq * (a.heads / a.kv_heads) + kTiles * kM - 1) / (kTiles * kM);
    return q;
}

// Items (a kv head's pair of row tiles) are numbered by level, and a request's
// last rows, which have the most keys, are its level 0: the long items start
// first and the short ones fill the card's last round.  Within a level the
// requests that reach it follow one another, their kv heads together.  One
// warp finds item `id`: the level by bisection of the items before it,
// kv heads * sum over requests of min(pairs, level).
__device__ __forceinline__ bool find_item(const AttendArgs& a, int64_t id, int (&hit)[3]) {
    const int lane = threadIdx.x & 31;
    const int64_t want = id / a.kv_heads;       // among pairs
    const int mine = lane < a.requests ? span_of(a, lane).pairs : 0;       // (32 requests need one look at the lengths)
    auto before = [&](int level) {
        int64_t n = min(mine, level);
        for (int r = lane + 32; r < a.requests; r += 32) n += min(span_of(a, r).pairs, level);
        return sili::warp_sum(n);
    };
    int most = mine;
    for (int r = lane + 32; r < a.requests; r += 32) most = max(most, span_of(a, r).pairs);
#pragma unroll
    for (int o = 16; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (want >= before(most)) return false;
    int lo = 0, hi = most;                      // before(lo) <= want < before(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before(mid) <= want) lo = mid; else hi = mid;
    }
    int64_t rank = want - before(lo);           // among the requests that reach level lo
    for (int base = 0; base < a.requests; base += 32) {
        const int r = base + lane, pairs = base == 0 ? mine : r < a.requests ? span_of(a, r).pairs : 0;
        const unsigned reach = __ballot_sync(0xffffffffu, pairs > lo);
        if (rank < __popc(reach)) {
            if ((reach >> lane & 1) && __popc(reach & ((1u << lane) - 1u)) == (int)rank) {
                hit[0] = r;
                hit[1] = (int)(id % a.kv_heads);
                hit[2] = pairs - 1 - lo;
            }
            return true;
        }
        rank -= __popc(reach);
    }
    return false;
}

template <typename T, int D>
struct Prompt {
    static constexpr int E = D / 32;
    const AttendArgs& a;
    Smem<D>& s;
    Work w;

    // tensor memory: S (64 columns a tile), P (two of 32), O (dim)
    __device__ __forceinline__ uint32_t s_col(int t) const { return s.tmem + t * kSub; }
    __device__ __forceinline__ uint32_t p_col(int t) const { return s.tmem + kTiles * kSub + t * kSub; }
    __device__ __forceinline__ uint32_t o_col(int t) const { return s.tmem + 2 * kTiles * kSub + t * D; }

    // ── warps 8-15: 4-bit keys and values of step j into stage j & 1 ──
    __device__ __forceinline__ void dequantise() { dequantise_stages<D>(a, s, w, kSoftmax, 0); }

    // ── one thread of warps 16 and 17 each: the products of tile t ──
    // (a thread a tile: neither waits behind the other's products being queued).  The thread's instructions are the chain
    // that its tile waits for, so it computes nothing per product but an addition to a descriptor's low word.
    __device__ __forceinline__ void products(int t) {
        constexpr uint32_t kStage = kKeys * D * 2 / 16;
        const uint32_t q = desc_low(s.q[t]), k0 = desc_low(s.k[0]), v0 = desc_low(s.v[0]), d = s_col(t), p = p_col(t), o = o_col(t);
        const int mine = w.n[t], stages = w.last - w.j0;
        const int over = s.slot >= 0 ? kAside<T> - 1 : 0x7FFFFFFF;      // O starts anew at steps that have none of these bits
        auto scores = [&](int i) {      // step i: the keys' rows 64 (i & 1) on of stage (i >> 1) & 1
            const uint32_t k = k0 + (i >> 1 & 1) * kStage + (i & 1) * (kSub * 8);
            mma_ss<false>(d, q, k, idesc(kM, kSub));
#pragma unroll
            for (int c = 1; c < D / 16; ++c)
                mma_ss<true>(d, q + (c >> 2) * (kM * 8) + 2 * (c & 3), k + (c >> 2) * (kKeys * 8) + 2 * (c & 3), idesc(kM, kSub));
            commit(&s.s_full[t]);
        };
        if (mine > 0) {
            if (!bar_wait(&s.kv_full[0], 0, &s.dead, a.polls)) return;
            asm volatile("tcgen05.fence::after_thread_sync;");
            scores(0);
        }
        for (int i = 0; i < mine; ++i) {
            if (i + 1 < mine) {
                if (((i + 1) & 1) == 0 && !bar_wait(&s.kv_full[(i + 1) >> 1 & 1], (i + 1) >> 2 & 1, &s.dead, a.polls)) return;
                if (!bar_wait(&s.s_free[t], i & 1, &s.dead, a.polls)) return;
                asm volatile("tcgen05.fence::after_thread_sync;");
                scores(i + 1);
            }
            if (!bar_wait(&s.p_full[t][i & 1], (i >> 1) & 1, &s.dead, a.polls)) return;
            asm volatile("tcgen05.fence::after_thread_sync;");
            const uint32_t v = v0 + (i >> 1 & 1) * kStage + (i & 1) * (D * 8);
#pragma unroll
            for (int c = 0; c < kSub / 16; ++c) mma_ts(o, p + (i & 1) * (kSub / 2) + 8 * c, v + 2 * c, idesc(kM, D), c > 0 || (i & over));
            commit(&s.p_free[t]);
            if (i + 1 == mine || ((i + 1) & over) == 0) commit(&s.o_full[t]);
            if ((i & 1) || i + 1 == mine) commit(&s.kv_free[i >> 1 & 1]);
        }
        // the other tile's stages: this one is done with them as soon as they are filled
        for (int n = (mine + 1) >> 1; n < stages; ++n) {
            if (!bar_wait(&s.kv_full[n & 1], (n >> 1) & 1, &s.dead, a.polls)) return;
            bar_arrive(&s.kv_free[n & 1]);
        }
    }

    // O's row times f
    __device__ __forceinline__ void rescale(int t, uint32_t lanes, float f) {
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
            float x[16];
            tmem_ld16(o_col(t) + lanes + 16 * c, x);
            tmem_wait(x);
            uint32_t r[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(x[i] * f);
            tmem_st16(o_col(t) + lanes + 16 * c, r);
        }
    }

    // this thread's part of the CTA's slot: 16 of its row's sums at a time, and the maximum they stand over
    __device__ __forceinline__ float4* aside(int t, int c) const {
        float* at = (float*)((uint8_t*)a.workspace + sili::kTicketBytes) + s.slot * sili::kSlotFloats;
        return (float4*)(at + ((t * (D / 16) + c) * kM + (threadIdx.x & 127)) * 16);
    }
    __device__ __forceinline__ float* aside_base() const {
        return (float*)((uint8_t*)a.workspace + sili::kTicketBytes) + (s.slot + 1) * sili::kSlotFloats - kSoftmax + threadIdx.x;
    }
    // x += the row's 16 sums of chunk c, taken from the maximum they stand over by f
    __device__ __forceinline__ void add_aside(int t, int c, float f, float (&x)[16]) const {
        const float4* at = aside(t, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = __ldcg(at + i);
            x[4 * i] = fmaf(v.x, f, x[4 * i]);
            x[4 * i + 1] = fmaf(v.y, f, x[4 * i + 1]);
            x[4 * i + 2] = fmaf(v.z, f, x[4 * i + 2]);
            x[4 * i + 3] = fmaf(v.w, f, x[4 * i + 3]);
        }
    }
    __device__ __forceinline__ float aside_factor(float base) const {
        const float was = __ldcg(aside_base());
        return was == base ? 1.f : ex2(was - base);      // (both -inf: nothing seen yet)
    }
    // O's row joins its sum in the slot; the next product overwrites O
    __device__ __forceinline__ void set_aside(int t, uint32_t lanes, float base, bool first) const {
        const float f = first ? 0.f : aside_factor(base);
        // 64 columns at a time, their loads in flight together
#pragma unroll 1
        for (int c = 0; c < D / 16; c += 4) {
            float x[64];
#pragma unroll
            for (int k = 0; k < 4; ++k) tmem_ld16(o_col(t) + lanes + 16 * (c + k), reinterpret_cast<float(&)[16]>(x[16 * k]));
            tmem_wait(x);
            if (!first)
#pragma unroll
                for (int k = 0; k < 4; ++k) add_aside(t, c + k, f, reinterpret_cast<float(&)[16]>(x[16 * k]));
#pragma unroll
            for (int i = 0; i < 16; ++i)
                __stcg(aside(t, c + i / 4) + i % 4, make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]));
        }
        __stcg(aside_base(), base);
    }

    // A slot for a CTA with rows of more than kAside steps.  There are more slots than CTAs can be resident, so one of
    // them is free; none found within the bound (never seen): the CTA goes on without.
    __device__ __forceinline__ int take_slot() const {
        if (max(w.n[0], w.n[1]) <= kAside<T>) return -1;
        uint32_t* bits = (uint32_t*)a.workspace + sili::kSlotWord;
        for (int i = 0; i < 64 * sili::kSlotWords; ++i) {
            const int word = (blockIdx.x + i) % sili::kSlotWords;
            for (uint32_t left = ~*(volatile uint32_t*)(bits + word); left; left &= left - 1) {
                const uint32_t bit = left & (0u - left);
                if (!(atomicOr(bits + word, bit) & bit)) {
                    __threadfence();
                    return word * 32 + __ffs(bit) - 1;
                }
            }
        }
        return -1;
    }

    // ── warps 0-7: one row a thread ──
    __device__ __forceinline__ void softmax() {
        const int t = threadIdx.x >> 7, row = w.row0 + t * kM + (threadIdx.x & 127);
        const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;     // this warp's quarter of the tensor memory's lanes
        const int warp_row0 = w.row0 + t * kM + (threadIdx.x & 96);
        const bool real = row < w.rows;
        const int64_t q_row = span_row() + (real ? row / w.group : 0);
        const int head = w.h * w.group + (real ? row % w.group : 0);
        // the row sees keys [from, to); every row of the warp sees those in [all_from, all_to)
        const int64_t pos = w.pos_of(row);
        const int to = (int)min(pos + 1, (int64_t)w.len), from = a.window ? (int)max(pos - a.window + 1, (int64_t)0) : 0;
        const int all_to = (int)min(w.pos_of(warp_row0) + 1, (int64_t)w.len);
        const int all_from = a.window ? (int)max(w.pos_of(warp_row0 + 31) - a.window + 1, (int64_t)0) : 0;
        // Q into shared memory as halves
        // (with the scale's sign, so that the logits' factor is never negative)
        float cf = fabsf(a.scale) * kLog2e;
        {
            // the whole row at once: its loads are in flight together
            const T* src = (const T*)a.q + q_row * a.qt + head * a.qh;
            const int m = threadIdx.x & 127;
            sili::Pack<T, 4> row4[D / 4];
#pragma unroll
            for (int i = 0; i < D / 4; ++i) {
                if (real) row4[i] = *(const sili::Pack<T, 4>*)(src + 4 * i);
                else
#pragma unroll
                    for (int k = 0; k < 4; ++k) row4[i].v[k] = sili::from_f32<T>(0.f);
            }
            float f = a.scale < 0.f ? -1.f : 1.f;
            if (!std::is_same<T, __half>::value) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < D / 4; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) top = max(top, __float_as_uint(sili::to_f32(row4[i].v[k])) & 0x7FFFFFFFu);
                if (top && top < 0x7F800000u) {
                    const int e = 14 - max((int)(top >> 23) - 127, -100);
                    f *= __int_as_float((127 + e) << 23);
                    cf *= __int_as_float((127 - e) << 23);
                }
            }
#pragma unroll
            for (int i = 0; i < D; i += 8) {
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const sili::Pack<T, 4>& p = row4[i / 4 + k / 2];
                    o[k] = pack2(sili::to_f32(p.v[2 * (k & 1)]) * f, sili::to_f32(p.v[2 * (k & 1) + 1]) * f);
                }
                *(uint4*)(s.q[t] + (i >> 6) * (kM * 128) + chunk_at(m, (i & 63) >> 3)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
        cf = fmaxf(cf, 0x1p-126f);      // not 0, which would undo a mask's -inf
        if (threadIdx.x == 0) s.slot = take_slot();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();       // Q is there: the products may begin
        float base = -INFINITY, l = 0.f;       // base: the running maximum - lift
        uint32_t poisoned = 0;                 // groups of 32 elements in which the row saw a NaN
        bool ok = true;
        const int steps = w.n[t], block = s.slot >= 0 ? kAside<T> : steps;
        int i = 0, filled = 0;                 // filled: how often O has been whole, once a block
        for (int end = min(block, steps); i < steps; end = min(end + block, steps)) {
            if (i > 0) {
                ok = __all_sync(0xffffffffu, bar_wait(&s.o_full[t], filled & 1, &s.dead, a.polls));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;");
                set_aside(t, lanes, base, filled++ == 0);
            }
            for (; i < end; ++i) {
                const int j = w.j0 + (i >> 1), st = i >> 1 & 1, half = i & 1, key0 = j * kKeys + half * kSub;
                ok = __all_sync(0xffffffffu, bar_wait(&s.s_full[t], i & 1, &s.dead, a.polls));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;");
                float x[kSub];
#pragma unroll
                for (int c = 0; c < kSub; c += 16) tmem_ld16(s_col(t) + lanes + c, reinterpret_cast<float(&)[16]>(x[c]));
                tmem_wait(x);
                asm volatile("tcgen05.fence::before_thread_sync;");
                bar_arrive(&s.s_free[t]);          // the next scores may come while these are worked on
                // keys [lo, hi) of the step are the row's; pages that are not there, a byte per 16 keys
                const uint32_t there = *(const volatile uint32_t*)&s.there[st][4 * half];
                const int hi = to - key0, lo = from - key0;
                if (there != 0x01010101u || key0 + kSub > all_to || key0 < all_from) {
#pragma unroll
                    for (int k = 0; k < kSub; ++k)
                        if (k < lo || k >= hi || !(there >> (k / 16 * 8) & 1)) x[k] = -INFINITY;
                }
                // The running maximum moves when a logit exceeds it by 2^7: P stays within a half, and O is seldom read and
                // written back.  (The maximum comes first although the sum of P would tell as well: P then takes the place
                // of S in the registers, and the exponentials have room to overlap: 1225 against 1700 clocks.)
                float top = fmaxf(x[0], x[1]), top1 = fmaxf(x[2], x[3]);
#pragma unroll
                for (int k = 4; k < kSub; k += 4) {
                    top = fmaxf(top, fmaxf(x[k], x[k + 1]));
                    top1 = fmaxf(top1, fmaxf(x[k + 2], x[k + 3]));
                }
                top = fmaxf(top, top1);
                if (top != -INFINITY) top = top * cf - kLift;
                if (__any_sync(0xffffffffu, top > base + kSlack)) {       // (NaN compares false)
                    const float fresh = fmaxf(base, top);
                    const float f = fresh == base ? 1.f : ex2(base - fresh);
                    base = fresh;
                    l *= f;
                    if (i > 0) {
                        ok = __all_sync(0xffffffffu, bar_wait(&s.p_free[t], (i - 1) & 1, &s.dead, a.polls));
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;");
                        rescale(t, lanes, f);     // (for nothing where O has just been set aside)
                    }
                }
                const float shift = base == -INFINITY ? 0.f : base;
                // P's buffer was last read by the product two steps ago, which was queued before these scores
                uint32_t p[2][16];
                float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
                for (int k = 0; k < kSub; k += 2) {
                    const float u = ex2(fmaf(x[k], cf, -shift)), v = ex2(fmaf(x[k + 1], cf, -shift));
                    sum0 += u; sum1 += v;
                    p[k / 32][k / 2 % 16] = pack2(u, v);
                }
                tmem_st16(p_col(t) + lanes + (i & 1) * (kSub / 2), p[0]);
                tmem_st16(p_col(t) + lanes + (i & 1) * (kSub / 2) + 16, p[1]);
                l += sum0 + sum1;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                if (*(volatile int*)&s.odd[st] == (i >> 1) + 1) {
                    for (int k = max(lo, 0); k < min(hi, kSub); ++k) {
                        if (!(there >> (k / 16 * 8) & 1)) continue;
                        for (int g = 0; g < E; ++g)
                            if (s.odd_keys[st][(half * kSub + k) >> 3][g] >> (k & 7) & 1) poisoned |= 1u << g;
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;");
                bar_arrive(&s.p_full[t][i & 1]);
            }
            if (!ok) break;
        }
        // (a barrier of its own: p_free may be one or two phases behind here, which a parity does not tell apart)
        if (ok && steps > 0) ok = __all_sync(0xffffffffu, bar_wait(&s.o_full[t], filled & 1, &s.dead, a.output_polls));
        asm volatile("tcgen05.fence::after_thread_sync;");
        // l 0: the row saw nothing
        float inv = l == 0.f ? 0.f : 1.f / l;
        const bool more = filled > 0 && ok;
        const float f = more ? aside_factor(base) : 0.f;
        const int64_t id = q_row * a.heads + head;
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
            float x[16];
            __syncwarp();
            if (steps > 0) {
                tmem_ld16(o_col(t) + lanes + 16 * c, x);
                tmem_wait(x);
                if (more) add_aside(t, c, f, x);
            } else
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = 0.f;
            const bool bad = !ok || (poisoned >> (c / 2) & 1);
            if (real)
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    sili::Pack<T, 8> o;
#pragma unroll
                    for (int k = 0; k < 8; ++k) o.v[k] = sili::from_f32<T>(bad ? __int_as_float(0x7FC00000) : x[i + k] * inv);
                    *(sili::Pack<T, 8>*)((T*)a.out + id * D + 16 * c + i) = o;
                }
        }
        if (real && a.lse) a.lse[id] = !ok ? __int_as_float(0x7FC00000) : l == 0.f ? -INFINITY : kLn2 * (base + log2f(l));
    }

    int first_row;
    __device__ __forceinline__ int64_t span_row() const { return first_row; }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) k_prompt(const __grid_constant__ AttendArgs a) {
    extern __shared__ uint8_t raw[];
    Smem<D>& s = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5;
    // rows of q that belong to no request
    {
        const int64_t from = a.requests ? min(max((int64_t)a.starts[0], (int64_t)0), a.tokens) : 0;
        const int64_t to = a.requests ? min(max((int64_t)a.starts[a.requests], from), a.tokens) : 0;
        const int64_t per = (int64_t)a.heads * D, n = (a.tokens - (to - from)) * per;
        for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
            const int64_t x = i < from * per ? i : i + (to - from) * per;
            ((T*)a.out)[x] = sili::from_f32<T>(0.f);
            if (a.lse && x % D == 0) a.lse[x / D] = -INFINITY;
        }
    }
    if (warp == 0) {
        int hit[3] = {-1, 0, 0};
        const bool found = find_item(a, blockIdx.x, hit);
        if (!found && threadIdx.x == 0) s.hit[0] = -1;
        if (hit[0] >= 0) { s.hit[0] = hit[0]; s.hit[1] = hit[1]; s.hit[2] = hit[2]; }
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&s.kv_full[i], kDequant);
            bar_init(&s.kv_free[i], kTiles);
            bar_init(&s.s_full[i], 1);
            bar_init(&s.o_full[i], 1);
            bar_init(&s.drained[i], 1);
            bar_init(&s.s_free[i], 128);
            bar_init(&s.p_full[i][0], 128);
            bar_init(&s.p_full[i][1], 128);
            bar_init(&s.p_free[i], 1);
            s.odd[i] = 0;
        }
        s.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    if (s.hit[0] < 0) return;
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(addr(&s.tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const Span q = span_of(a, s.hit[0]);
    Prompt<T, D> k{a, s};
    Work& w = k.w;
    w.r = s.hit[0];
    w.h = s.hit[1];
    w.group = a.heads / a.kv_heads;
    w.rows = q.nq * w.group;
    w.row0 = s.hit[2] * (kTiles * kM);
    w.len = q.len;
    w.pos0 = q.pos0;
    k.first_row = q.row0;
    w.j0 = a.window ? (int)(max((int64_t)0, w.pos_of(w.row0) - a.window + 1) / kKeys) : 0;
    w.last = w.j0;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        w.n[t] = 0;
        if (w.row0 + t * kM < w.rows) {
            const int64_t hi = min((int64_t)w.len, w.pos_of(w.row0 + t * kM + kM - 1) + 1) - (int64_t)w.j0 * kKeys;
            w.n[t] = max(0, (int)((hi + kSub - 1) / kSub));
        }
        w.last = max(w.last, w.j0 + (w.n[t] + 1) / 2);
    }
    if (warp < kSoftmax / 32) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        k.softmax();
    } else if (warp < kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsDequant));
        __syncthreads();       // Q is there
        if (w.last > w.j0) k.dequantise();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
        __syncthreads();       // Q is there
        const int t = warp - kMmaWarp;
        if (w.last > w.j0 && t < kTiles && (threadIdx.x & 31) == 0) k.products(t);
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (*(volatile int*)&s.dead) {     // (every role has left its loop: it is the same for all threads)
        // Whichever role gave up: the products that a thread has queued may still run, so that thread waits for them
        // (bounded) before the tensor memory is freed and the shared memory with it.
        const int t = warp - kMmaWarp;
        if (t >= 0 && t < kTiles && (threadIdx.x & 31) == 0) {
            atomicOr((unsigned*)a.workspace + sili::kErrorWord, 1u);
            int quiet = 0;
            commit(&s.drained[t]);
            bar_wait(&s.drained[t], 0, &quiet, kPolls);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0 && s.slot >= 0) {
        __threadfence();       // the next owner's sums come after this one's
        atomicAnd((uint32_t*)a.workspace + sili::kSlotWord + s.slot / 32, ~(1u << s.slot % 32));
    }
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem), "r"(512));
}

template <typename T, int D>
int launch(const AttendArgs& a, cudaStream_t s) {
    constexpr int smem = (int)sizeof(Smem<D>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    static_assert(kSoftmax == sili::kSlotRows && D <= sili::kSlotDim, "a slot holds a CTA's rows");
    auto kernel = k_prompt<T, D>;
    static std::atomic<uint64_t> set{0};
    CKP(sili::allow_smem(kernel, smem, set));
    // no more items than every request's rows rounded up; CTAs past the last leave at once
    const int64_t rows = a.tokens * (a.heads / a.kv_heads);
    const int64_t items = (rows / (kTiles * kM) + a.requests + 1) * a.kv_heads;
    if (items > 0x7fffffffLL) return sili::set_error(SILI_EINVAL, "kv4_attention: sizes out of range");
    kernel<<<(unsigned)items, kThreads, smem, s>>>(a);
    sili::count_launch();
    CKP(cudaGetLastError());
    return SILI_OK;
}

}  // namespace

namespace sili {

// Full row pairs from which on this kernel is taken: half the SMs' worth, where it is ahead at every size measured.  us
// of one request in bf16, this kernel | the other, which splits the keys:
//   32 heads over 8 x 128,  1024 keys: 48 pairs 47 |  74, 72: 47 |  94, 128:  47 |  149
//                           4096 keys: 32 117 | 117, 48 118 | 162, 72 118 | 229, 128 119 | 389
//                          16384 keys: 24 399 | 275, 32 399 | 354, 48 398 | 518, 72 399 | 762
//   32 over 4 x 64,         4096 keys: 32 104 |  78, 48 104 | 105, 72 104 | 145
//                          16384 keys: 48 362 | 312, 64 361 | 406, 72 360 | 453
//   14 over 14 x 64,       16384 keys: 42 354 | 276, 70 359 | 439
// They cross between 20 pairs (1024 keys) and 60 (dim 64 over 16384), so calls between there and 74 pairs take up to
// twice the time that this kernel would.  The rule looks at all rows of a batch: a request with one query beside a long
// prompt is walked here by one CTA a kv head, however long it is (262143 keys beside 2048 queries: 5.8 ms; in two calls
// 0.18 + 0.09).
bool kv4_prompt_takes(int dtype, int dim, int64_t tokens, int heads, int kv_heads, int64_t most_new) {
    const int64_t group = heads / kv_heads;
    return dtype != SILI_F32 && (dim == 64 || dim == 128) && most_new * group >= 128 &&
           tokens * group / (kTiles * kM) * kv_heads >= 74;
}
void kv4_polls(AttendArgs& a) {
    a.polls = g_polls.load(std::memory_order_relaxed);
    a.output_polls = g_output_polls.load(std::memory_order_relaxed);
}
int kv4_prompt_launch(int dtype, int dim, const AttendArgs& args, cudaStream_t s) {
    AttendArgs a = args;
    kv4_polls(a);
    if (dtype == SILI_F16) return dim == 64 ? launch<__half, 64>(a, s) : launch<__half, 128>(a, s);
    return dim == 64 ? launch<__nv_bfloat16, 64>(a, s) : launch<__nv_bfloat16, 128>(a, s);
}

}  // namespace sili

extern "C" int sili_kv4_attention_wait_limit(int polls, int output_polls) {
    g_polls.store(polls < 0 ? kPolls : std::min(polls, kPolls), std::memory_order_relaxed);
    g_output_polls.store(output_polls < 0 ? kPolls : std::min(output_polls, kPolls), std::memory_order_relaxed);
    return SILI_OK;
}
