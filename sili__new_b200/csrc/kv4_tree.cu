// Attention of drafted tokens' trees over the 4-bit paged cache where a
// request brings many rows (query token x query head of the group), in 16
// bits, on the fifth generation tensor cores (tcgen05, sm_100a).
//
// The units of 128 keys of all (request, kv head, row tile) segments are
// numbered and cut evenly over one CTA an SM, whatever the lengths; a segment
// that several CTAs share leaves its parts in the workspace, and a second
// launch joins them, in CTA order, many CTAs a segment.  Within a CTA the work
// is kv4_prompt.cu's, as a pipeline that runs on from segment to segment: two
// groups of four softmax warps with a row a thread, S and a double-buffered P
// in tensor memory, eight warps that turn the next keys into halves in shared
// memory, a thread each for the two groups' products.  Where a request has
// more than 128 rows, the groups are two tiles of 128 rows over the same keys
// (PAIR), 64 at a time; else they have the same rows and the keys' halves (64 of
// 128 each), and are joined at a segment's end.
//
// A row sees the committed keys, as its window leaves them, and of the request's
// own, which follow, those that its mask names: a step of 64 keys that not all
// of a warp's rows see whole gets its 64 bits from those two.  Roundings as in
// kv4_prompt.cu; a row's sums leave tensor memory every kPiece units.
//
// What bounds it, 40 requests of up to 64 drafts over 2k-12k keys, 32 heads over
// 8, dim 128, bf16 (233 GFLOP, 143 us at the card's matrix rate): 444-459 us
// from card to card, 520 TFLOP/s, tensor pipe 35 %, issue 50 %.  With the conversions, loads,
// exponentials and most products left out it took 328: a step is the softmax
// warps' chain (scores' barrier, tensor-memory load, maximum, exponentials,
// store), two of its warps a scheduler.  24 drafts over 131071 keys (52 GFLOP):
// 173 us; there the conversion of the keys, for 96 rows, weighs as much (125
// without it).
//
// Every wait is bounded: one that gives up sets the workspace's error word; from
// there on the rows of the CTA's run, and its parts of shared segments, become NaN.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kernels.cuh"
#include "kv4_stage.cuh"
#include "sili_b200.h"

namespace sili {
int set_error(int code, const std::string& msg);
}

namespace {

using namespace sili::mma;
using sili::AttendArgs;
using sili::Cursor;
using sili::ex2;
using sili::kLift;
using sili::kLn2;
using sili::kLog2e;
using sili::kSlack;
using sili::pack2;

#define CKT(x)                                                                                          \
    do {                                                                                                \
        const cudaError_t e_ = (x);                                                                     \
        if (e_ != cudaSuccess) return sili::set_error(SILI_ECUDA, std::string(#x) + ": " + cudaGetErrorString(e_)); \
    } while (0)

constexpr int kM = 128;               // rows of a tile (MMA M)
constexpr int kSub = 64;              // keys of a step of a group
constexpr int kSoftmax = 256, kDequant = 256, kThreads = kSoftmax + kDequant + 128;
// registers a thread after the split; together what the launch holds: 96 * 640
constexpr int kRegsSoftmax = 144, kRegsDequant = 72, kRegsRest = 48;
static_assert(kSoftmax * kRegsSoftmax + kDequant * kRegsDequant + 128 * kRegsRest <= 96 * kThreads, "register split");
static_assert(kKeys == sili::kUnit, "a unit is a stage");
constexpr int kMmaWarp = (kSoftmax + kDequant) / 32;
constexpr int kCtas = 148;
// Units after which a row's sums leave tensor memory: the matrix unit cuts what it adds to an accumulator towards zero,
// 6e-9 a key where V has one sign (kv4_prompt.cu: 16384 keys leave a fifth of fp16's half unit, 65536 of bf16's).
template <typename T>
constexpr int kPiece = std::is_same<T, __half>::value ? 128 : 512;

// The workspace: the error word within the first kTicketBytes; what the join needs to know, a record a CTA; the parts.
struct Shared {
    int parts;             // of the segment that begins in the CTA and does not end there; 0: none
    int row0, rows, h, tile;
    int pad[3];
};
constexpr int64_t kPartsAt = sili::kTicketBytes + (int64_t)kCtas * sizeof(Shared);
// A part: [row][dim] sums, then the rows' maxima and the sums of their probabilities; those twice, so that the pieces of a
// run write the one while the other is read.
__host__ __device__ constexpr int64_t part_floats(int rows, int dim) { return (int64_t)rows * (dim + 4); }
__device__ __forceinline__ float* part_of(const AttendArgs& a, int rows, int dim, int cta, int which) {
    return (float*)((uint8_t*)a.workspace + kPartsAt) + (cta * 2 + which) * part_floats(rows, dim);
}

template <int D>
struct Smem {
    alignas(1024) uint8_t q[2][kM * D * 2];      // (then the second group's sums, where the groups have the same rows)
    alignas(1024) uint8_t k[2][kKeys * D * 2];
    alignas(1024) uint8_t v[2][kKeys * D * 2];
    alignas(8) unsigned long long kv_full[2], kv_free[2];                         // by stage
    unsigned long long s_full[2], s_free[2], p_free[2], o_full[2], drained[2];    // by group
    unsigned long long p_full[2][2];                                              // by group and the step's parity
    unsigned long long q_full;
    float base[kM], sum[kM];          // the second group's
    uint8_t odd_keys[2][16][4];       // [stage][8 keys][group]: bits of keys whose V scale is not a number
    int odd[2];                       // the last stage that had any, plus one
    alignas(8) uint8_t there[2][8];   // [stage][16 keys]: their page exists
    uint32_t tmem;
    int dead;
};

// true when the phase of this parity is complete; false, at once, when any role has given up
__device__ __forceinline__ bool wait(unsigned long long* b, uint32_t parity, int* dead, int polls) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(addr(b)), "r"(parity) : "memory");
    return done || (!*(volatile int*)dead && bar_wait(b, parity, dead, polls));
}
// one arrival a warp
__device__ __forceinline__ void warp_arrive(unsigned long long* b) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(b);
}
// two floats at a time
__device__ __forceinline__ uint64_t two(float x, float y) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ void halves(uint64_t d, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(d)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kSoftmax) : "memory"); }
__device__ __forceinline__ bool softmax_any(bool is) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((uint32_t)is), "n"(kSoftmax) : "memory");
    return any;
}
// bits [lo, hi) of 64
__device__ __forceinline__ uint64_t range_bits(int64_t lo, int64_t hi) {
    if (hi <= 0 || lo >= 64 || lo >= hi) return 0;
    const uint64_t below = hi >= 64 ? ~0ull : (1ull << hi) - 1;
    return lo <= 0 ? below : below & (~0ull << lo);
}

template <typename T, int D, bool PAIR>
struct Tree {
    static constexpr int E = D / 32, kRows = PAIR ? 2 * kM : kM;
    using Cur = Cursor<kRows>;
    const AttendArgs& a;
    Smem<D>& s;
    int64_t begin, end, all;

    // What every role knows of a piece of a segment: stages [j0, last) of request r's and kv head h's keys.
    struct Work {
        int r, h, len, j0, last;
    };
    // The walk over the run's pieces, the same for every role: f(cursor, its stages, whether the segment has begun before, the
    // pieces of it that follow, stages done before).
    template <typename F>
    __device__ __forceinline__ void pieces(Cur c, F f) const {
        const int n = (int)(end - begin);
        bool again = false;
        for (int done = 0; done < n;) {
            const int rest = min(c.left(), n - done), here = min(rest, kPiece<T>);
            const Work w{c.r, c.h, c.q.len, c.u, c.u + here};
            if (!f(c, w, again, (rest - here + kPiece<T> - 1) / kPiece<T>, done)) return;
            done += here;
            again = here < rest;
            if (again) c.u += here;
            else if (done < n) c.next_segment(a);
        }
    }
    __device__ __forceinline__ int rows_of(const Cur& c) const { return c.q.nq * (a.heads / a.kv_heads) - c.tile * kRows; }
    // steps of group t in a piece of so many stages: none where it has no rows
    __device__ __forceinline__ int steps_of(const Cur& c, int t, int stages) const {
        return PAIR ? (t * kM < rows_of(c) ? 2 * stages : 0) : stages;
    }

    // tensor memory: S (64 columns a group), P (two of 32), O (dim)
    __device__ __forceinline__ uint32_t s_col(int t) const { return s.tmem + t * kSub; }
    __device__ __forceinline__ uint32_t p_col(int t) const { return s.tmem + 2 * kSub + t * kSub; }
    __device__ __forceinline__ uint32_t o_col(int t) const { return s.tmem + 4 * kSub + t * D; }

    // ── warps 8-15 ──
    __device__ __forceinline__ void dequantise(const Cur& c0) {
        pieces(c0, [&](const Cur&, const Work& w, bool, int, int done) { return dequantise_stages<D>(a, s, w, kSoftmax, done); });
    }

    // ── a thread of warps 16 and 17 each: the products of group t ──
    // Step i of a piece is half i & 1 of its stage i / 2 (PAIR), or half t of its stage i.
    __device__ __forceinline__ void products(int t, const Cur& c0) {
        constexpr uint32_t kStage = kKeys * D * 2 / 16;
        const uint32_t q = desc_low(s.q[PAIR ? t : 0]), k0 = desc_low(s.k[0]), v0 = desc_low(s.v[0]);
        const uint32_t d = s_col(t), p = p_col(t), o = o_col(t);
        int u = 0, piece = 0;      // steps and pieces done
        pieces(c0, [&](const Cur& c, const Work& w, bool, int, int done) {
            const int stages = w.last - w.j0, mine = steps_of(c, t, stages);
            if (!wait(&s.q_full, piece++ & 1, &s.dead, a.polls)) return false;
            auto scores = [&](int i) {
                const int n = done + (PAIR ? i >> 1 : i), half = PAIR ? i & 1 : t;
                if ((!PAIR || half == 0) && !wait(&s.kv_full[n & 1], (n >> 1) & 1, &s.dead, a.polls)) return false;
                if (u + i > 0 && !wait(&s.s_free[t], (u + i - 1) & 1, &s.dead, a.polls)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const uint32_t k = k0 + (n & 1) * kStage + half * (kSub * 8);
                mma_ss<false>(d, q, k, idesc(kM, kSub));
#pragma unroll
                for (int x = 1; x < D / 16; ++x)
                    mma_ss<true>(d, q + (x >> 2) * (kM * 8) + 2 * (x & 3), k + (x >> 2) * (kKeys * 8) + 2 * (x & 3), idesc(kM, kSub));
                commit(&s.s_full[t]);
                return true;
            };
            if (mine > 0 && !scores(0)) return false;
            for (int i = 0; i < mine; ++i) {
                if (i + 1 < mine && !scores(i + 1)) return false;
                const int n = done + (PAIR ? i >> 1 : i), half = PAIR ? i & 1 : t, at = u + i;
                if (!wait(&s.p_full[t][at & 1], (at >> 1) & 1, &s.dead, a.polls)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const uint32_t v = v0 + (n & 1) * kStage + half * (D * 8);
#pragma unroll
                for (int x = 0; x < kSub / 16; ++x)
                    mma_ts(o, p + (at & 1) * (kSub / 2) + 8 * x, v + 2 * x, idesc(kM, D), x > 0 || i > 0);
                commit(&s.p_free[t]);
                if (!PAIR || half == 1) commit(&s.kv_free[n & 1]);
                if (i + 1 == mine) commit(&s.o_full[t]);
            }
            if (mine == 0) {
                // the other group's stages: this one is done with them as soon as they are filled
                for (int n = done; n < done + stages; ++n) {
                    if (!wait(&s.kv_full[n & 1], (n >> 1) & 1, &s.dead, a.polls)) return false;
                    bar_arrive(&s.kv_free[n & 1]);
                }
                bar_arrive(&s.o_full[t]);      // (the softmax does not go on to the next piece without this thread)
            }
            u += mine;
            return true;
        });
    }

    // ── warps 0-7: one row a thread ──
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

    // What a thread knows of its row.
    struct Row {
        const int64_t* mask;
        int id;                // its place in lse; -1: none
        int to, from, own, len;     // committed keys [from, to) that it sees; the request's first drafted key, its keys
        float cf;              // logit = S * cf, in powers of two
    };

    // the keys of [key0, key0 + 64) that the row sees, without those whose page is not there
    __device__ __forceinline__ uint64_t visible(const Row& r, int key0, uint32_t there) const {
        uint64_t bits = range_bits((int64_t)r.from - key0, (int64_t)r.to - key0);
        const int64_t d = (int64_t)key0 - r.own;           // the window's first key among the drafts
        if (r.id >= 0 && d > -64 && d < 64 * a.words) {
            uint64_t own = 0;
            if (d < 0) own = (uint64_t)r.mask[0] << -d;
            else {
                const int w = (int)(d >> 6), b = (int)(d & 63);
                own = (uint64_t)r.mask[w] >> b;
                if (b && w + 1 < a.words) own |= (uint64_t)r.mask[w + 1] << (64 - b);
            }
            bits |= own & range_bits((int64_t)r.own - key0, (int64_t)r.len - key0);
        }
        uint64_t pages = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (there >> (8 * k) & 1) pages |= 0xFFFFull << (16 * k);
        return bits & pages;
    }

    // this thread's row of a segment; its query into shared memory as halves
    __device__ __forceinline__ Row begin_segment(const Cur& c, const Work& w) {
        const int t = threadIdx.x >> 7, m = threadIdx.x & 127, group = a.heads / a.kv_heads;
        const int at = (PAIR ? t * kM : 0) + m, row = c.tile * kRows + at;
        const bool real = at < rows_of(c);
        const int64_t token = c.q.row0 + (real ? row / group : 0);
        const int head = c.h * group + (real ? row % group : 0);
        Row r;
        r.id = real ? (int)(token * a.heads + head) : -1;
        r.mask = a.masks + token * a.words;
        r.len = w.len;
        r.own = (int)min(max(c.q.pos0, (int64_t)-0x7FFFFFFF), (int64_t)0x7FFFFFFF);
        int some = 0;
        if (real)
            for (int i = 0; i < a.words; ++i) some += __popcll((unsigned long long)r.mask[i]);
        r.to = !real ? w.len : some ? min(max(r.own, 0), w.len) : 0;
        r.from = real && a.window ? (int)min(max(c.q.pos0 + some - a.window, (int64_t)0), (int64_t)0x7FFFFFFF) : 0;
        // (with the scale's sign, so that the logits' factor is never negative)
        r.cf = fabsf(a.scale) * kLog2e;
        const T* src = (const T*)a.q + token * a.qt + head * a.qh;
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
                r.cf *= __int_as_float((127 - e) << 23);
            }
        }
        if (PAIR || t == 0)
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
        r.cf = fmaxf(r.cf, 0x1p-126f);      // not 0, which would undo a mask's -inf
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;");
        __syncwarp();
        if ((threadIdx.x & 31) == 0) bar_arrive(&s.q_full);
        return r;
    }

    __device__ __forceinline__ void softmax(const Cur& c0) {
        const int t = threadIdx.x >> 7;
        const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;     // this warp's quarter of the tensor memory's lanes
        int u = 0, filled = 0;                                         // steps and pieces done
        bool alive = true;     // no wait has given up: behind one that has, a barrier's parity says nothing about its phase
        pieces(c0, [&](const Cur& c, const Work& w, bool again, int left, int done) {
            const Row r = begin_segment(c, w);
            const int all_from = __reduce_max_sync(0xffffffffu, r.from), all_to = __reduce_min_sync(0xffffffffu, r.to);
            float base = -INFINITY, l = 0.f;       // base: the running maximum - lift
            uint32_t poisoned = 0;                 // groups of 32 elements in which the row saw a NaN
            const int steps = steps_of(c, t, w.last - w.j0);
            bool ok = alive;
            for (int i = 0; ok && i < steps; ++i) {
                const int n = done + (PAIR ? i >> 1 : i), st = n & 1, half = PAIR ? i & 1 : t, at = u + i;
                const int key0 = (w.j0 + (PAIR ? i >> 1 : i)) * kKeys + half * kSub;
                ok = __all_sync(0xffffffffu, wait(&s.s_full[t], at & 1, &s.dead, a.polls));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;");
                // (both were written before the stage was given to the products; asked for here, they come beside the scores)
                const uint32_t there = *(const volatile uint32_t*)&s.there[st][4 * half];
                const int odd_stage = *(const volatile int*)&s.odd[st];
                float x[kSub];
#pragma unroll
                for (int k = 0; k < kSub; k += 16) tmem_ld16(s_col(t) + lanes + k, reinterpret_cast<float(&)[16]>(x[k]));
                tmem_wait(x);
                asm volatile("tcgen05.fence::before_thread_sync;");
                warp_arrive(&s.s_free[t]);         // the next scores may come while these are worked on
                const bool masked = there != 0x01010101u || key0 + kSub > all_to || key0 < all_from;
                uint64_t bits = ~0ull;
                if (masked) {
                    bits = visible(r, key0, there);
                    const uint32_t low = (uint32_t)bits, high = (uint32_t)(bits >> 32);
#pragma unroll
                    for (int k = 0; k < kSub; ++k)
                        if (!((k < 32 ? low : high) >> (k & 31) & 1)) x[k] = -INFINITY;
                }
                // The running maximum moves when a logit exceeds it by 2^7: P stays within a half, and O is seldom read and
                // written back.
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < kSub; k += 2) tops[k / 2 & 3] = max3(tops[k / 2 & 3], x[k], x[k + 1]);
                float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
                if (top != -INFINITY) top = top * r.cf - kLift;
                if (__any_sync(0xffffffffu, top > base + kSlack)) {       // (NaN compares false)
                    const float fresh = fmaxf(base, top);
                    const float f = fresh == base ? 1.f : ex2(base - fresh);
                    base = fresh;
                    l *= f;
                    if (i > 0) {
                        ok = __all_sync(0xffffffffu, wait(&s.p_free[t], (at - 1) & 1, &s.dead, a.polls));
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;");
                        rescale(t, lanes, f);
                    }
                }
                const float shift = base == -INFINITY ? 0.f : base;
                // P's buffer was last read by the product two steps ago, which was queued before these scores
                uint32_t p[2][16];
                const uint64_t cf2 = two(r.cf, r.cf), shift2 = two(-shift, -shift);
                uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < kSub; k += 2) {
                    float y, z;
                    halves(fma2(two(x[k], x[k + 1]), cf2, shift2), y, z);
                    y = ex2(y);
                    z = ex2(z);
                    sum[k / 2 & 3] = add2(sum[k / 2 & 3], two(y, z));
                    p[k / 32][k / 2 % 16] = pack2(y, z);
                }
                tmem_st16(p_col(t) + lanes + (at & 1) * (kSub / 2), p[0]);
                tmem_st16(p_col(t) + lanes + (at & 1) * (kSub / 2) + 16, p[1]);
                float sum0, sum1;
                halves(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), sum0, sum1);
                l += sum0 + sum1;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                if (odd_stage == n + 1) {
                    if (!masked) bits = visible(r, key0, there);
                    for (int g = 0; g < E; ++g) {
                        uint64_t odd = 0;
                        for (int k = 0; k < 8; ++k) odd |= (uint64_t)s.odd_keys[st][half * 8 + k][g] << (8 * k);
                        if (odd & bits) poisoned |= 1u << g;
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;");
                warp_arrive(&s.p_full[t][at & 1]);
            }
            u += steps;
            // (a barrier of its own: p_free may be one or two phases behind here, which a parity does not tell apart)
            // (voted as the others are: the barrier and the loads that follow take a warp's lanes together)
            if (ok) ok = __all_sync(0xffffffffu, wait(&s.o_full[t], filled & 1, &s.dead, a.output_polls));
            ++filled;
            asm volatile("tcgen05.fence::after_thread_sync;");
            alive = !softmax_any(!ok);
            end_piece(c, r, base, l, poisoned, steps, !alive, again, left, begin + done - (c.u - c.q.k0));
            return true;
        });
    }

    // The end of a piece of a segment: its rows, or its part of them.  seg0: the number of the segment's first unit.
    __device__ __forceinline__ void end_piece(const Cur& c, const Row& r, float base, float l, uint32_t poisoned, int steps,
                                              bool dead, bool again, int left, int64_t seg0) {
        const int t = threadIdx.x >> 7, m = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;
        float* mine = (float*)s.q[0] + m;            // the second group's sums, [dim][row], where the rows are the same
        if (!PAIR) {
            if (t == 1) {
                s.base[m] = base;
                s.sum[m] = l;
#pragma unroll 1
                for (int d = 0; d < D; d += 16) {
                    float x[16];
                    tmem_ld16(o_col(1) + lanes + d, x);
                    tmem_wait(x);
#pragma unroll
                    for (int i = 0; i < 16; ++i) mine[(d + i) * kM] = poisoned >> (d >> 5) & 1 ? __int_as_float(0x7FC00000) : x[i];
                }
            }
            softmax_sync();
        }
        if (PAIR || t == 0) {
            float h = 1.f, f = 0.f;
            if (!PAIR) {       // the other group's keys
                const float other = s.base[m], most = fmaxf(base, other);
                h = base == most ? 1.f : ex2(base - most);
                f = other == most ? 1.f : ex2(other - most);
                l = l * h + s.sum[m] * f;
                base = most;
            }
            const int64_t seg1 = seg0 + c.q.units, ctas = min((int64_t)gridDim.x, all);
            const bool whole = seg0 >= begin && seg1 <= end, out = whole && !left;
            const int cta = blockIdx.x, lead = whole ? cta : (int)(((seg0 + 1) * ctas - 1) / all);
            const int row = (PAIR ? t * kM : 0) + m;
            // (a whole segment's pieces use the place of the segment that this CTA begins last)
            float* part = part_of(a, kRows, D, cta, cta == lead);
            float* tops = part + kRows * (D + 2 * (left & 1));
            const float* before = part + kRows * (D + 2 * (~left & 1));
            float was_f = 0.f;
            if (again) {
                const float was = __ldcg(before + row), most = fmaxf(was, base);
                was_f = was == most ? 1.f : ex2(was - most);
                const float now = base == most ? 1.f : ex2(base - most);
                l = l * now + __ldcg(before + kRows + row) * was_f;
                h *= now;
                f *= now;
                base = most;
            }
            if (dead) l = h = __int_as_float(0x7FC00000);
            if (out) {
                // l 0: the row saw nothing; NaN goes through
                const float inv = l == 0.f ? 0.f : 1.f / l;
                h *= inv;
                f *= inv;
                was_f *= inv;
                if (r.id >= 0 && a.lse) a.lse[r.id] = l == 0.f ? -INFINITY : kLn2 * (base + log2f(l));
            } else if (r.id >= 0) {
                __stcg(tops + row, base);
                __stcg(tops + kRows + row, l);
            }
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
                float x[16];
                __syncwarp();          // (lanes without a row left the last turn early)
                if (steps > 0) {
                    tmem_ld16(o_col(t) + lanes + d, x);
                    tmem_wait(x);
                }
                if (r.id < 0) continue;
                const bool bad = poisoned >> (d >> 5) & 1;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    x[i] = bad ? __int_as_float(0x7FC00000) : x[i] * h;
                    if (!PAIR) x[i] = fmaf(mine[(d + i) * kM], f, x[i]);
                }
                float4* at = (float4*)(part + (int64_t)row * D + d);
                if (again)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 v = __ldcg(at + i);
                        x[4 * i] = fmaf(v.x, was_f, x[4 * i]);
                        x[4 * i + 1] = fmaf(v.y, was_f, x[4 * i + 1]);
                        x[4 * i + 2] = fmaf(v.z, was_f, x[4 * i + 2]);
                        x[4 * i + 3] = fmaf(v.w, was_f, x[4 * i + 3]);
                    }
                if (out)
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        sili::Pack<T, 8> o;
#pragma unroll
                        for (int k = 0; k < 8; ++k) o.v[k] = sili::from_f32<T>(x[i + k]);
                        *(sili::Pack<T, 8>*)((T*)a.out + (int64_t)r.id * D + d + i) = o;
                    }
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) __stcg(at + i, make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]));
            }
            if (threadIdx.x == 0 && !whole && lead == cta && !left) {
                Shared& to = ((Shared*)((uint8_t*)a.workspace + sili::kTicketBytes))[cta];
                to.row0 = c.q.row0;
                to.rows = c.q.nq * (a.heads / a.kv_heads);
                to.h = c.h;
                to.tile = c.tile;
                to.parts = (int)((seg1 * ctas - 1) / all) - lead + 1;
            }
        }
        __syncwarp();
        if (!PAIR) softmax_sync();         // (the next segment's queries come over the sums)
    }
};

template <typename T, int D, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) k_tree(const __grid_constant__ AttendArgs a) {
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
    if (threadIdx.x == 0) ((Shared*)((uint8_t*)a.workspace + sili::kTicketBytes))[blockIdx.x].parts = 0;
    using K = Tree<T, D, PAIR>;
    typename K::Cur c;
    K k{a, s};
    k.all = sili::locate<K::kRows, kThreads / 32>(a, c, blockIdx.x, gridDim.x, k.begin, k.end);
    if (k.begin >= k.end) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&s.kv_full[i], kDequant);
            bar_init(&s.kv_free[i], 2);
            bar_init(&s.s_full[i], 1);
            bar_init(&s.o_full[i], 1);
            bar_init(&s.drained[i], 1);
            bar_init(&s.s_free[i], kM / 32);
            bar_init(&s.p_full[i][0], kM / 32);
            bar_init(&s.p_full[i][1], kM / 32);
            bar_init(&s.p_free[i], 1);
            s.odd[i] = 0;
        }
        bar_init(&s.q_full, kSoftmax / 32);
        s.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(addr(&s.tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    if (warp < kSoftmax / 32) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        k.softmax(c);
    } else if (warp < kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsDequant));
        k.dequantise(c);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
        const int t = warp - kMmaWarp;
        if (t < 2 && (threadIdx.x & 31) == 0) k.products(t, c);
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (*(volatile int*)&s.dead) {     // (every role has left its loop: it is the same for all threads)
        // Whichever role gave up: the products that a thread has queued may still run, so that thread waits for them
        // (bounded) before the tensor memory is freed and the shared memory with it.
        const int t = warp - kMmaWarp;
        if (t >= 0 && t < 2 && (threadIdx.x & 31) == 0) {
            atomicOr((unsigned*)a.workspace + sili::kErrorWord, 1u);
            int quiet = 0;
            commit(&s.drained[t]);
            bar_wait(&s.drained[t], 0, &quiet, 4096);
        }
        __syncthreads();
    }
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem), "r"(512));
}

// The parts of the segments that several CTAs shared, joined: CTA (lead, y) takes kJoinRows rows of the one that began in
// CTA `lead`.
constexpr int kJoinRows = 16, kJoinThreads = 256;

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kJoinThreads) k_tree_join(const __grid_constant__ AttendArgs a) {
    __shared__ float s_weight[kJoinRows][kCtas], s_inv[kJoinRows];
    const int lead = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = a.heads / a.kv_heads;
    const Shared g = ((const Shared*)((const uint8_t*)a.workspace + sili::kTicketBytes))[lead];
    const int first = blockIdx.y * kJoinRows, n = g.parts;
    if (n == 0 || g.tile * ROWS + first >= g.rows) return;
    auto id_of = [&](int row) {      // -1: none
        const int at = g.tile * ROWS + first + row;
        return at < g.rows ? (g.row0 + at / group) * a.heads + g.h * group + at % group : -1;
    };
    for (int row = warp; row < kJoinRows; row += kJoinThreads / 32) {
        const int id = id_of(row);
        if (id < 0) continue;
        auto tops = [&](int i) { return part_of(a, ROWS, D, lead + i, i == 0) + ROWS * D + first + row; };
        float top = -INFINITY, sum = 0.f;
        for (int i = lane; i < n; i += 32) top = fmaxf(top, __ldcg(tops(i)));
#pragma unroll
        for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        for (int i = lane; i < n; i += 32) {
            const float mine = __ldcg(tops(i)), f = mine == top ? 1.f : ex2(mine - top);
            s_weight[row][i] = f;
            sum += __ldcg(tops(i) + ROWS) * f;
        }
        sum = sili::warp_sum(sum);
        if (lane == 0) {
            s_inv[row] = sum == 0.f ? 0.f : 1.f / sum;
            if (a.lse) a.lse[id] = sum == 0.f ? -INFINITY : kLn2 * (top + log2f(sum));
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kJoinRows * (D / 4); i += kJoinThreads) {
        const int row = i / (D / 4), d = i % (D / 4) * 4, id = id_of(row);
        if (id < 0) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int k = 0; k < n; ++k) {
            const float f = s_weight[row][k];
            const float4 p = __ldcg((const float4*)(part_of(a, ROWS, D, lead + k, k == 0) + (int64_t)(first + row) * D + d));
            v[0] += p.x * f; v[1] += p.y * f; v[2] += p.z * f; v[3] += p.w * f;
        }
        sili::Pack<T, 4> o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o.v[k] = sili::from_f32<T>(v[k] * s_inv[row]);
        *(sili::Pack<T, 4>*)((T*)a.out + (int64_t)id * D + d) = o;
    }
}

template <typename T, int D, bool PAIR>
int launch(const AttendArgs& a, cudaStream_t s) {
    constexpr int smem = (int)sizeof(Smem<D>) + 1024, rows = PAIR ? 2 * kM : kM;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    static_assert(D * kM * 4 <= (int)sizeof(Smem<D>::q), "the second group's sums fit the queries' place");
    auto kernel = k_tree<T, D, PAIR>;
    static std::atomic<uint64_t> set{0};
    CKT(sili::allow_smem(kernel, smem, set));
    kernel<<<kCtas, kThreads, smem, s>>>(a);
    k_tree_join<T, D, rows><<<dim3(kCtas, rows / kJoinRows), kJoinThreads, 0, s>>>(a);
    sili::count_launch(2);
    CKT(cudaGetLastError());
    return SILI_OK;
}
template <typename T, int D>
int by_rows(const AttendArgs& a, int64_t rows, cudaStream_t s) {
    return rows <= kM ? launch<T, D, false>(a, s) : launch<T, D, true>(a, s);
}

}  // namespace

namespace sili {

// us of this kernel | the one of kv4_attention.cu, by rows that every request has (32 heads over 8):
//   dim 128, 1 request, 131071 keys, fp16:    32 rows 166 | 119, 36: 166 | 200, 64: 168 | 200, 128: 178 | 368
//   dim 128, 40 requests, 2k-12k keys, bf16:  32 rows 344 | 264, 36: 343 | 487, 64: 349 | 495, 128: 378 | 978, 256: 460 | 1898
//   dim 128, the same up to 1000 keys:        32 rows 124 | 114, 36: 127 | 181, 64: 121 | 181, 256: 209 | 799
//   dim 128, 4 requests up to 700 keys:       32 rows  30 |  27, 36:  30 |  41, 64:  30 |  44, 256:  40 |  59
//   dim 64, 1 request, 131071 keys, fp16:     32 rows 114 |  78, 36: 114 | 126, 64: 116 | 126, 128: 121 | 226
//   dim 64, 40 requests, 2k-12k keys, bf16:   32 rows 237 | 170, 36: 235 | 307, 64: 239 | 314, 256: 365 | 1178
//   dim 64, the same up to 1000 keys:         32 rows  79 |  83, 36:  81 | 130, 64:  77 | 130, 256: 127 | 546
//   dim 64, 4 requests up to 700 keys:        32 rows  24 |  22, 36:  24 |  33, 64:  24 |  34, 256:  32 |  44
// The other one walks tiles of up to 32 rows, so it is taken up to there.  `rows` comes from the caller's largest number of
// queries (or their average, without a hint); requests that have fewer, up to 32 rows, would be faster in the other one.
bool kv4_tree_takes(int dtype, int dim, int64_t rows) { return dtype != SILI_F32 && (dim == 64 || dim == 128) && rows > 32; }

int64_t kv4_tree_workspace(int dim, int64_t rows) {
    return kPartsAt + kCtas * 2 * part_floats(rows <= kM ? kM : 2 * kM, dim) * 4;
}

int kv4_tree_launch(int dtype, int dim, const AttendArgs& args, int64_t rows, cudaStream_t s) {
    AttendArgs a = args;
    kv4_polls(a);
    if (dtype == SILI_F16) return dim == 64 ? by_rows<__half, 64>(a, rows, s) : by_rows<__half, 128>(a, rows, s);
    return dim == 64 ? by_rows<__nv_bfloat16, 64>(a, rows, s) : by_rows<__nv_bfloat16, 128>(a, rows, s);
}

}  // namespace sili
