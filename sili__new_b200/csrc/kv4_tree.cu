// Attention of drafted tokens' trees over the 4-bit paged cache where a
// request brings many rows (query token x query head of the group), in 16
// bits, on the fifth generation tensor cores (tcgen05, sm_100a).
//
// As in kv4_attention.cu the products are transposed, so that the cache is the
// 128-row operand and the rows only make it as wide as there are,
//   S^T [128 keys, N rows] = K Q^T,   O^T [dim, N rows] += V^T P^T,
// and the units of 128 keys of all (request, kv head, row tile) segments are
// numbered and cut evenly over one CTA an SM; a segment that several CTAs share
// is joined by whichever finishes last, in CTA order.  A CTA is a pipeline over
// its run of units:
//   warps 8-15  turn K into halves in tensor memory (a lane a key: the first
//               operand may lie there, which saves shared memory 64 KB of
//               traffic a unit) and V, transposed by interleaving the nibbles
//               of two keys, into shared memory;
//   warp 16     a thread issues the products, the next unit's scores before
//               this one's P V;
//   warps 0-7   a lane a key and half of the rows each: exponentials over the
//               rows' running maxima, P into shared memory, where the rows are
//               consecutive (8 of them a 16-byte store);
//   warp 17     asks the second-level cache for the keys four units ahead.
// The maxima are shared by all keys of a unit; they move only when a logit
// exceeds one by 2^7, which a vote of the four warps tells.  Rows' sums are
// taken by lanes and joined at a segment's end.  Roundings as in kv4_prompt.cu:
// K and V exact, bf16 queries scaled by a power of two a row, P rounded once to
// a half after its sum is taken.
//
// Every wait is bounded: one that gives up sets the workspace's error word; the
// rows of the CTA's run become NaN, its parts of shared segments too, so that
// the joins stay complete.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kernels.cuh"
#include "kv4_attention.cuh"
#include "kv4_mma.cuh"
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
using sili::kUnit;
using sili::mul2;
using sili::pack2;

#define CKT(x)                                                                                          \
    do {                                                                                                \
        const cudaError_t e_ = (x);                                                                     \
        if (e_ != cudaSuccess) return sili::set_error(SILI_ECUDA, std::string(#x) + ": " + cudaGetErrorString(e_)); \
    } while (0)

constexpr int kSoftmax = 256, kDequant = 256, kThreads = kSoftmax + kDequant + 128;
constexpr int kRegsSoftmax = 144, kRegsDequant = 72, kRegsRest = 48;
static_assert(kSoftmax * kRegsSoftmax + kDequant * kRegsDequant + 128 * kRegsRest <= 96 * kThreads, "register split");
constexpr int kMmaWarp = (kSoftmax + kDequant) / 32, kFetchWarp = kMmaWarp + 1;
constexpr int kCtas = 148;
constexpr int kAhead = 4;               // units that the cache is asked for ahead
constexpr float kNoMaximum = -3e38f;    // below every finite logit, and finite: a masked key's -inf over it is -inf
// Units after which a row's sums leave tensor memory: the matrix unit cuts what it adds to an accumulator towards zero,
// 6e-9 a key where V has one sign (kv4_prompt.cu: 16384 keys leave a fifth of fp16's half unit, 65536 of bf16's).
template <typename T>
constexpr int kPiece = std::is_same<T, __half>::value ? 128 : 512;

template <int D, int N>
struct Smem {
    alignas(1024) uint8_t q[N * D * 2];
    alignas(1024) uint8_t v[2][kUnit * D * 2];      // (a product of 128 rows reads on behind 64 of V^T: into P, unused)
    alignas(1024) uint8_t p[(N + 63) / 64][kUnit * 128];
    float weight[N * (kCtas + 2)];                   // the parts' weights of a shared segment
    alignas(16) float4 cn[N / 2];                    // two rows: logit factors, negated bases (the running maximum - lift)
    unsigned long long mask[N][4];
    int from[N], to[N];                              // the row's committed keys
    float f[N];                                      // what a moved maximum multiplies the sums by
    int top[N];                                      // a unit's largest logits, as ordered integers
    float sum[4][N];
    unsigned poison[N];                              // groups of 32 elements in which the row saw a NaN
    alignas(8) unsigned long long k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], s_free[2], p_full, p_free, q_full, o_full,
        drained;
    uint8_t there[4][8];                             // [unit & 3][16 keys]: their page exists
    uint8_t odd_keys[4][16][4];                      // [unit & 3][8 keys][group]: bits of keys whose V scale is not a number
    int odd[4];                                      // the last unit that had any, plus one
    int progress;                                    // units dequantised
    uint32_t tmem;
    int dead, last;
};

// true when the phase of this parity is complete; false, at once, when any role has given up
__device__ __forceinline__ bool wait(unsigned long long* b, uint32_t parity, int* dead, int polls) {
    return !*(volatile int*)dead && bar_wait(b, parity, dead, polls);
}
__device__ __forceinline__ void group_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool group_any(int id, int threads, bool is) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((uint32_t)is), "r"(id), "r"(threads) : "memory");
    return any;
}
// a * b + c, two at a time
__device__ __forceinline__ void fma2(float& x, float& y, float a0, float a1, float b0, float b1, float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(x), "=f"(y) : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
// floats as integers of the same order (NaN apart)
__device__ __forceinline__ int ordered(float x) {
    const int u = __float_as_int(x);
    return u ^ (u >> 31 & 0x7FFFFFFF);
}
__device__ __forceinline__ float unordered(int u) { return __int_as_float(u ^ (u >> 31 & 0x7FFFFFFF)); }

template <typename T, int D, int N>
struct Tree {
    static constexpr int E = D / 32, kCols = N / 2, kChunk = kCols < 32 ? kCols : 32;
    using Cur = Cursor<N>;
    using S = Smem<D, N>;
    const AttendArgs& a;
    S& s;
    int64_t begin, end, all;

    // tensor memory: K twice (dim / 2 columns), S twice (N), O (N)
    __device__ __forceinline__ uint32_t k_col(int st) const { return s.tmem + st * (D / 2); }
    __device__ __forceinline__ uint32_t s_col(int st) const { return s.tmem + D + st * N; }
    __device__ __forceinline__ uint32_t o_col() const { return s.tmem + D + 2 * N; }

    // ── warps 8-15 ──
    // What a thread loads of a unit, once the pages are known.
    struct Ahead {
        int pk, pv, offk, offv, len, key0;
    };
    __device__ __forceinline__ void dequantise(Cur c) {
        const int n = (int)(end - begin), tid = threadIdx.x - kSoftmax, dw = tid >> 5, lane = tid & 31;
        // K: a lane a key, half of its elements
        const int key = tid & 127, part = tid >> 7;
        const uint32_t lanes = (uint32_t)(tid & 96) << 16;
        // V: 8 keys x 8 elements a thread; lane & 7 numbers the keys, so a store instruction fills whole rows
        const int half = dw & 1, ck = lane & 7, db = (dw >> 1) * 4 + (lane >> 3), vkey = half * 64 + ck * 8, vg = db >> 2;
        const bool has_v = db < D / 8;
        constexpr int kWide = D / 64;          // 16-byte parts of half a K row
        uint4 rk[kWide], sv[E / 2];
        uint32_t sk = 0, rv[8];
        int left = c.left();
        auto pages = [&](Ahead& h) {
            h.key0 = c.u * kUnit;
            h.len = c.q.len;
            const int* row = a.table + c.r * a.stride;
            const int head = c.h * a.page;
            int ok, ov;
            const int colk = a.column(h.key0 + key, ok), colv = a.column(h.key0 + vkey, ov);
            // (whole runs of 16 keys, which share a page; the last may reach past the end)
            h.pk = ((h.key0 + key) & ~15) < h.len ? __ldg(row + colk) : -1;
            h.pv = ((h.key0 + vkey) & ~15) < h.len ? __ldg(row + colv) : -1;
            h.offk = head + ok;
            h.offv = head + ov;
            if (--left == 0) {
                c.next_segment(a);
                left = c.left();
            } else ++c.u;
        };
        bool there;
        auto load_k = [&](const Ahead& h) {
            there = (unsigned)h.pk < (unsigned)a.n_pages;
            if (there) {
                const int64_t row = (int64_t)h.pk * (2 * (int64_t)a.half_rows) + h.offk;
                const uint8_t* codes = a.codes + row * (D / 2) + part * (D / 4);
#pragma unroll
                for (int i = 0; i < kWide; ++i) rk[i] = __ldg((const uint4*)(codes + 16 * i));
                const uint8_t* scales = a.scales + row * E + part * (E / 2);
                if (E == 4) sk = __ldg((const uint16_t*)scales);
                else sk = __ldg(scales);
            }
        };
        auto load_v = [&](const Ahead& h) {
            if (has_v && (unsigned)h.pv < (unsigned)a.n_pages) {
                const int64_t row = (int64_t)h.pv * (2 * (int64_t)a.half_rows) + a.half_rows + h.offv;
                const uint8_t* codes = a.codes + row * (D / 2) + db * 4;
                const uint8_t* scales = a.scales + row * E;
#pragma unroll
                for (int i = 0; i < 8; ++i) rv[i] = __ldg((const uint32_t*)(codes + i * (D / 2)));
#pragma unroll
                for (int i = 0; i < E / 2; ++i) sv[i] = __ldg((const uint4*)(scales + 16 * i));
            } else {
#pragma unroll
                for (int i = 0; i < E / 2; ++i) sv[i] = make_uint4(0, 0, 0, 0);
            }
        };
        // the scales of keys 2p and 2p + 1 as bytes 0 and 2
        const uint32_t pick = E == 4 ? (uint32_t)(vg | (4 + vg) << 8) : (uint32_t)(vg | (2 + vg) << 8);
        auto pair_of = [&](int p) {
            if constexpr (E == 4) {
                const uint4 v = sv[p >> 1 & (E / 2 - 1)];
                return __byte_perm(p & 1 ? v.z : v.x, p & 1 ? v.w : v.y, pick) & 0x00FF00FFu;
            } else {
                const uint32_t v = p == 0 ? sv[0].x : p == 1 ? sv[0].y : p == 2 ? sv[0].z : sv[0].w;
                return __byte_perm(v, 0, pick) & 0x00FF00FFu;
            }
        };
        Ahead next;
        pages(next);
        load_k(next);
        load_v(next);
        if (n > 1) pages(next);
        for (int i = 0; i < n; ++i) {
            const int st = i & 1, slot = i & 3;
            const uint32_t again = ((i >> 1) - 1) & 1;
            if (i >= 2 && !wait(&s.k_free[st], again, &s.dead, a.polls)) return;
            asm volatile("tcgen05.fence::after_thread_sync;");
            // (slots are four: a unit's are read before the scores of the one two further on are asked for)
            if (part == 0 && (lane & 15) == 0) s.there[slot][key >> 4] = there;
            uint32_t pairs[4], bits = 0, odd_any = 0;
            if (has_v) {
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    pairs[p] = pair_of(p);
                    odd_any |= pairs[p] + 0x00080008u;      // carries into bit 8 of a byte of at least 0xF8
                }
                if (odd_any & 0x01000100u) {
                    // scales that are no numbers are left out and noted
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        if ((pairs[p] & 0xFFu) >= 0xF8u) { bits |= 1u << (2 * p); pairs[p] &= 0xFFFF0000u; }
                        if ((pairs[p] >> 16) >= 0xF8u) { bits |= 2u << (2 * p); pairs[p] &= 0xFFFFu; }
                    }
                    *(volatile int*)&s.odd[slot] = i + 1;
                }
                if ((db & 3) == 0) s.odd_keys[slot][half * 8 + ck][vg] = (uint8_t)bits;
            }
#pragma unroll
            for (int q = 0; q < kWide; ++q) {
                const uint32_t sc = (sk >> (8 * q) & 0xFFu) * 0x00800080u, w[4] = {rk[q].x, rk[q].y, rk[q].z, rk[q].w};
                uint32_t r[16];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t f[4];
                    sili::kv4_decode4(w[k], f);
#pragma unroll
                    for (int b = 0; b < 4; ++b) r[4 * k + b] = mul2(f[b], sc);
                }
                tmem_st16(k_col(st) + lanes + part * (D / 4) + 16 * q, r);
            }
            if (i + 1 < n) load_k(next);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;");
            bar_arrive(&s.k_full[st]);
            if (i >= 2 && !wait(&s.v_free[st], again, &s.dead, a.polls)) return;
            if (has_v) {
                constexpr uint32_t kLow = 0x0F0F0F0Fu;
                uint32_t even[4][4], odd[4][4];
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const uint32_t x = rv[2 * p], y = rv[2 * p + 1], sc = pairs[p] << 7;
                    sili::kv4_decode4((x & kLow) | ((y << 4) & ~kLow), even[p]);
                    sili::kv4_decode4(((x >> 4) & kLow) | (y & ~kLow), odd[p]);
#pragma unroll
                    for (int b = 0; b < 4; ++b) { even[p][b] = mul2(even[p][b], sc); odd[p][b] = mul2(odd[p][b], sc); }
                }
                uint8_t* block = s.v[st] + half * (D * 128);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int d = db * 8 + 2 * b;
                    *(uint4*)(block + chunk_at(d, ck)) = make_uint4(even[0][b], even[1][b], even[2][b], even[3][b]);
                    *(uint4*)(block + chunk_at(d + 1, ck)) = make_uint4(odd[0][b], odd[1][b], odd[2][b], odd[3][b]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            bar_arrive(&s.v_full[st]);
            if (i + 1 < n) {
                load_v(next);
                if (i + 2 < n) pages(next);
            }
            if (tid == 0) *(volatile int*)&s.progress = i + 1;
        }
    }

    // ── warp 17: the codes and scales of the units ahead into the second-level cache (a hint: nothing waits for it) ──
    __device__ __forceinline__ void fetch(Cur c) {
        const int n = (int)(end - begin), lane = threadIdx.x & 31, run = lane & 7, kind = lane >> 3;
        int left = c.left();
        for (int i = 0; i < n; ++i) {
            if (i >= 2) {
                const int key = c.u * kUnit + run * 16;
                int off;
                const int col = a.column(key, off);
                const int pg = key < c.q.len ? __ldg(a.table + c.r * a.stride + col) : -1;
                if ((unsigned)pg < (unsigned)a.n_pages) {
                    const int64_t row = (int64_t)pg * (2 * (int64_t)a.half_rows) + (kind & 1) * (int64_t)a.half_rows +
                                        c.h * a.page + off;
                    const uint8_t* at = kind < 2 ? a.codes + row * (D / 2) : a.scales + row * E;
                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(at), "r"(kind < 2 ? 16 * (D / 2) : 16 * E)
                                 : "memory");
                }
            }
            if (--left == 0) {
                if (i + 1 < n) c.next_segment(a);
                left = c.left();
            } else ++c.u;
            for (int k = 0; *(volatile int*)&s.progress + kAhead < i + 1; ++k) {
                if (*(volatile int*)&s.dead || k > 1000000) return;
                __nanosleep(100);
            }
        }
    }

    // The walk over the run's pieces of segments, the same for every role: f(cursor, units, first of its segment here, pieces
    // that follow in it, units done before).
    template <typename F>
    __device__ __forceinline__ void pieces(Cur c, F f) {
        const int n = (int)(end - begin);
        bool again = false;
        for (int done = 0; done < n;) {
            const int rest = min(c.left(), n - done), here = min(rest, kPiece<T>);
            if (!f(c, here, again, (rest - here + kPiece<T> - 1) / kPiece<T>, done)) return;
            done += here;
            again = here < rest;
            if (again) c.u += here;
            else if (done < n) c.next_segment(a);
        }
    }

    // ── a thread of warp 16 ──
    __device__ __forceinline__ void products(const Cur& c0) {
        const uint32_t q = desc_low(s.q), v0 = desc_low(s.v[0]);
        // P: rows consecutive (MN-major), 64 of them 128 bytes; the next 64 a block further on
        const uint32_t p = ((addr(s.p[0]) >> 4) & 0x3FFFu) | ((uint32_t)(kUnit * 128 / 16) << 16);
        constexpr uint32_t kIdO = idesc(128, N) | 1u << 16;
        int piece = 0;
        auto scores = [&](int u) {
            const int st = u & 1;
            if (!wait(&s.k_full[st], (u >> 1) & 1, &s.dead, a.polls)) return false;
            if (u >= 2 && !wait(&s.s_free[st], ((u >> 1) - 1) & 1, &s.dead, a.polls)) return false;
            asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
                mma_ts(s_col(st), k_col(st) + 8 * c, q + (c >> 2) * (N * 8) + 2 * (c & 3), idesc(128, N), c > 0);
            commit(&s.s_full[st]);
            commit(&s.k_free[st]);
            return true;
        };
        pieces(c0, [&](const Cur&, int here, bool, int, int u) {
            if (!wait(&s.q_full, piece++ & 1, &s.dead, a.polls) || !scores(u)) return false;
            for (int i = 0; i < here; ++i, ++u) {
                if (i + 1 < here && !scores(u + 1)) return false;
                const int st = u & 1;
                if (!wait(&s.v_full[st], (u >> 1) & 1, &s.dead, a.polls) || !wait(&s.p_full, u & 1, &s.dead, a.polls)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const uint32_t v = v0 + st * (kUnit * D * 2 / 16);
#pragma unroll
                for (int c = 0; c < kUnit / 16; ++c) {
                    const uint32_t x = v + (c >> 2) * (D * 8) + 2 * (c & 3);
                    if (c > 0 || i > 0) mma_ss<true>(o_col(), x, p + c * 128, kIdO);
                    else mma_ss<false>(o_col(), x, p + c * 128, kIdO);
                }
                commit(&s.p_free);
                commit(&s.v_free[st]);
                if (i + 1 == here) commit(&s.o_full);
            }
            return true;
        });
    }

    // ── warps 0-7 ──  (l: a lane's part of its rows' sums)
    // rows, masks and queries of a segment
    __device__ __forceinline__ void begin_segment(const Cur& c, float (&l)[kCols], int& all_from, int& all_to) {
        const int tid = threadIdx.x, group = a.heads / a.kv_heads;
        const int rows = c.q.nq * group, row0 = c.tile * N;
        if (tid < 2 * N) {
            // two lanes a row
            const int row = row0 + (tid >> 1), part = tid & 1;
            const bool real = row < rows;
            const int64_t token = c.q.row0 + (real ? row / group : 0);
            const int head = c.h * group + (real ? row % group : 0);
            const T* src = (const T*)a.q + token * a.qt + head * a.qh + part * (D / 2);
            sili::Pack<T, 4> x[D / 8];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                if (real) x[i] = *(const sili::Pack<T, 4>*)(src + 4 * i);
                else
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[i].v[k] = sili::from_f32<T>(0.f);
            }
            // (with the scale's sign, so that the logits' factor is never negative)
            float f = a.scale < 0.f ? -1.f : 1.f, cf = fabsf(a.scale) * kLog2e;
            if (!std::is_same<T, __half>::value) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) top = max(top, __float_as_uint(sili::to_f32(x[i].v[k])) & 0x7FFFFFFFu);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                if (top && top < 0x7F800000u) {
                    const int e = 14 - max((int)(top >> 23) - 127, -100);
                    f *= __int_as_float((127 + e) << 23);
                    cf *= __int_as_float((127 - e) << 23);
                }
            }
#pragma unroll
            for (int i = 0; i < D / 2; i += 8) {
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const sili::Pack<T, 4>& p = x[i / 4 + k / 2];
                    o[k] = pack2(sili::to_f32(p.v[2 * (k & 1)]) * f, sili::to_f32(p.v[2 * (k & 1) + 1]) * f);
                }
                const int d = part * (D / 2) + i;
                *(uint4*)(s.q + (d >> 6) * (N * 128) + chunk_at(tid >> 1, (d & 63) >> 3)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
            if (part == 0) {
                const int r = tid >> 1;
                cf = fmaxf(cf, 0x1p-126f);      // not 0, which would undo a mask's -inf
                ((float*)&s.cn[r >> 1])[r & 1] = cf;
                ((float*)&s.cn[r >> 1])[2 + (r & 1)] = -kNoMaximum;
                int some = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned long long m = real && i < a.words ? (unsigned long long)a.masks[token * a.words + i] : 0;
                    s.mask[r][i] = m;
                    some += __popcll(m);
                }
                s.to[r] = some ? (int)min(max(c.q.pos0, (int64_t)0), (int64_t)c.q.len) : 0;
                s.from[r] = a.window ? (int)min(max(c.q.pos0 + some - a.window, (int64_t)0), (int64_t)0x7FFFFFFF) : 0;
                s.top[r] = ordered(-INFINITY);
                s.poison[r] = 0;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;");
        bar_arrive(&s.q_full);
        group_sync(1, kSoftmax);
        // keys that every (real) row sees
        all_from = 0;
        all_to = 0x7FFFFFFF;
        for (int i = threadIdx.x & 31; i < min(rows - row0, N); i += 32) {
            all_from = max(all_from, s.from[i]);
            all_to = min(all_to, s.to[i]);
        }
        all_from = __reduce_max_sync(0xffffffffu, all_from);
        all_to = __reduce_min_sync(0xffffffffu, all_to);
#pragma unroll
        for (int k = 0; k < kCols; ++k) l[k] = 0.f;
    }

    __device__ __forceinline__ void load(uint32_t at, float (&x)[kChunk]) const {
#pragma unroll
        for (int k = 0; k < kChunk; k += 16) tmem_ld16(at + k, reinterpret_cast<float(&)[16]>(x[k]));
#pragma unroll
        for (int k = 0; k < kChunk; k += 16) tmem_wait(reinterpret_cast<float(&)[16]>(x[k]));
    }

    // A unit's exponentials.  g: which half of the rows; i: the unit's place in its piece, u: in the run.
    __device__ __forceinline__ void unit(const Cur& c, float (&l)[kCols], int key0, int i, int u, int all_from, int all_to) {
        const int g = threadIdx.x >> 7, lane_key = threadIdx.x & 127, key = key0 + lane_key, st = u & 1, slot = u & 3;
        const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16, scores = s_col(st) + lanes + g * kCols;
        const int col0 = g * kCols;
        wait(&s.s_full[st], (u >> 1) & 1, &s.dead, a.polls);
        asm volatile("tcgen05.fence::after_thread_sync;");
        const bool exists = key < c.q.len && *(volatile uint8_t*)&s.there[slot][lane_key >> 4];
        const bool masked = !exists || key0 + kUnit > all_to || key0 < all_from;
        const int64_t own = c.q.pos0;
        const int64_t d = (int64_t)key - own;
        auto hide = [&](float (&x)[kChunk], int c0) {
            if (!masked) return;
            if (d >= 0) {
                const bool in = exists && d < 64 * 4;
                const int w = in ? (int)(d >> 6) : 0, b = (int)(d & 63);
#pragma unroll
                for (int k = 0; k < kChunk; ++k)
                    if (!in || !(s.mask[c0 + k][w] >> b & 1)) x[k] = -INFINITY;
            } else {
#pragma unroll
                for (int k = 0; k < kChunk; ++k)
                    if (!exists || key >= s.to[c0 + k] || key < s.from[c0 + k]) x[k] = -INFINITY;
            }
        };
        float above = -INFINITY;
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += kChunk) {
            float x[kChunk];
            load(scores + c0, x);
            hide(x, col0 + c0);
#pragma unroll
            for (int k = 0; k < kChunk; k += 2) {
                const float4 cn = s.cn[(col0 + c0 + k) / 2];
                float e0, e1;
                fma2(e0, e1, x[k], x[k + 1], cn.x, cn.y, cn.z, cn.w);
                above = fmaxf(above, fmaxf(e0, e1));
            }
        }
        if (group_any(2 + g, 128, above > kLift + kSlack)) raise(l, scores, col0, i, u, lanes, hide);
        // the product before this one has read P
        if (u > 0) wait(&s.p_free, (u - 1) & 1, &s.dead, a.polls);
        const unsigned odd = *(volatile int*)&s.odd[slot] == u + 1 ? odd_bits(slot, lane_key) : 0u;
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += kChunk) {
            float x[kChunk];
            load(scores + c0, x);
            if (c0 + kChunk == kCols) {
                asm volatile("tcgen05.fence::before_thread_sync;");
                bar_arrive(&s.s_free[st]);
            }
            hide(x, col0 + c0);
            if (odd)
#pragma unroll
                for (int k = 0; k < kChunk; ++k)
                    if (x[k] != -INFINITY) atomicOr(&s.poison[col0 + c0 + k], odd);
#pragma unroll
            for (int k = 0; k < kChunk; k += 8) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 cn = s.cn[(col0 + c0 + k) / 2 + j];
                    float e0, e1;
                    fma2(e0, e1, x[k + 2 * j], x[k + 2 * j + 1], cn.x, cn.y, cn.z, cn.w);
                    e0 = ex2(e0);
                    e1 = ex2(e1);
                    l[c0 + k + 2 * j] += e0;
                    l[c0 + k + 2 * j + 1] += e1;
                    o[j] = pack2(e0, e1);
                }
                const int col = col0 + c0 + k;
                *(uint4*)(s.p[col >> 6] + chunk_at(lane_key, (col & 63) >> 3)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;");
        bar_arrive(&s.p_full);
    }
    __device__ __forceinline__ unsigned odd_bits(int slot, int lane_key) const {
        unsigned b = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) b |= (unsigned)(s.odd_keys[slot][lane_key >> 3][e] >> (lane_key & 7) & 1) << e;
        return b;
    }

    // Moves the rows' maxima to those of this unit's logits where they are larger, and the sums along.
    template <typename H>
    __device__ __forceinline__ void raise(float (&l)[kCols], uint32_t scores, int col0, int i, int u, uint32_t lanes, const H& hide) {
        const int g = threadIdx.x >> 7;
#pragma unroll 1
        for (int c0 = 0; c0 < kCols; c0 += kChunk) {
            float x[kChunk];
            load(scores + c0, x);
            hide(x, col0 + c0);
#pragma unroll
            for (int k = 0; k < kChunk; ++k) {
                const float cf = ((const float*)&s.cn[(col0 + c0 + k) / 2])[k & 1], e = x[k] * cf;
                const int top = __reduce_max_sync(0xffffffffu, e != e ? ordered(-INFINITY) : ordered(e));
                if ((threadIdx.x & 31) == 0) atomicMax(&s.top[col0 + c0 + k], top);
            }
        }
        group_sync(2 + g, 128);
        const int r = threadIdx.x & 127;
        if (r < kCols) {
            const int c = col0 + r;
            float* nb = (float*)&s.cn[c >> 1] + 2 + (c & 1);
            const float base = -*nb, top = unordered(s.top[c]), fresh = top == -INFINITY ? base : fmaxf(base, top - kLift);
            s.f[c] = fresh == base ? 1.f : ex2(base - fresh);
            *nb = -fresh;
            s.top[c] = ordered(-INFINITY);
        }
        group_sync(2 + g, 128);
#pragma unroll
        for (int k = 0; k < kCols; ++k) l[k] *= s.f[col0 + k];
        if (i > 0) {
            wait(&s.p_free, (u - 1) & 1, &s.dead, a.polls);
            asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll 1
            for (int c0 = 0; c0 < kCols; c0 += 16) {
                float x[16];
                tmem_ld16(o_col() + lanes + col0 + c0, x);
                tmem_wait(x);
                uint32_t r16[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) r16[k] = __float_as_uint(x[k] * s.f[col0 + c0 + k]);
                tmem_st16(o_col() + lanes + col0 + c0, r16);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
    }

    // a CTA's part of a segment: [row][dim] sums, then the rows' maxima and the sums of their probabilities; those twice, so
    // that the pieces of a run write the one while the other is read
    __device__ __forceinline__ float* partial(int cta, int which) const {
        return (float*)((uint8_t*)a.workspace + sili::kTicketBytes) + (int64_t)(cta * 2 + which) * N * (D + 4);
    }
    __device__ __forceinline__ int64_t row_id(const Cur& c, int row) const {      // -1: none
        const int group = a.heads / a.kv_heads, at = c.tile * N + row;
        return at < c.q.nq * group ? (int64_t)(c.q.row0 + at / group) * a.heads + c.h * group + at % group : -1;
    }
    __device__ __forceinline__ void store(const Cur& c, int row, int d, float v, float top, float sum) const {
        const int64_t id = row_id(c, row);
        if (id < 0) return;
        // sum 0: the row saw nothing; NaN goes through
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        ((T*)a.out)[id * D + d] = sili::from_f32<T>(v * inv);
        if (d == 0 && a.lse) a.lse[id] = sum == 0.f ? -INFINITY : kLn2 * (top + log2f(sum));
    }

    // The end of a piece of a segment: as in kv4_attention.cu, with the sums coming from tensor memory.
    __device__ __forceinline__ void end_piece(const Cur& c, float (&l)[kCols], int piece, int64_t seg0, int64_t seg1, bool again, int left) {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = tid >> 7, dim = tid & 127;
        const uint32_t lanes = (uint32_t)(tid & 96) << 16;
        wait(&s.o_full, piece & 1, &s.dead, a.output_polls);
        asm volatile("tcgen05.fence::after_thread_sync;");
        // the rows' sums over the warp's keys: halves of the rows exchanged, until a lane has kCols / 32 of them (or, of fewer
        // rows, some lanes one)
#pragma unroll
        for (int o = 16, w = kCols; o; o >>= 1) {
            const bool up = lane & o;
            if (w > 1) {
                w >>= 1;
#pragma unroll
                for (int k = 0; k < kCols; ++k)
                    if (k < w) {
                        const float mine = up ? l[k + w] : l[k], other = up ? l[k] : l[k + w];
                        l[k] = mine + __shfl_xor_sync(0xffffffffu, other, o);
                    }
            } else l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
        }
        {
            // lane bits from 16 on chose the upper halves
            constexpr int kLeft = kCols >= 32 ? kCols / 32 : 1, kSteps = kCols >= 32 ? 5 : kCols == 16 ? 4 : 3;
            int col = 0;
#pragma unroll
            for (int k = 0, o = 16, w = kCols / 2; k < kSteps; ++k, o >>= 1, w >>= 1)
                if (lane & o) col += w;
            if (kSteps == 5 || (lane & ((32 >> kSteps) - 1)) == 0)
#pragma unroll
                for (int k = 0; k < kLeft; ++k) s.sum[warp & 3][g * kCols + col + k] = l[k];
        }
        const bool dead = group_any(1, kSoftmax, *(volatile int*)&s.dead);
        const bool whole = seg0 >= begin && seg1 <= end;
        const int64_t ctas = min((int64_t)gridDim.x, all);
        const int cta = blockIdx.x, lead = whole ? cta : (int)(((seg0 + 1) * ctas - 1) / all);
        // (a whole segment's pieces use the place of the segment that this CTA begins last)
        float* part = partial(cta, cta == lead);
        float* tops = part + N * (D + 2 * (left & 1));
        const float* before = part + N * (D + 2 * (~left & 1));
#pragma unroll 1
        for (int c0 = 0; c0 < kCols; c0 += 16) {
            float x[16];
            tmem_ld16(o_col() + lanes + g * kCols + c0, x);
            tmem_wait(x);
            if (dim < D)
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int row = g * kCols + c0 + k;
                    float v = x[k], top = -((const float*)&s.cn[row >> 1])[2 + (row & 1)];
                    float sum = s.sum[0][row] + s.sum[1][row] + s.sum[2][row] + s.sum[3][row];
                    if (dead) v = sum = __int_as_float(0x7FC00000);
                    else if (s.poison[row] >> (dim >> 5) & 1) v = __int_as_float(0x7FC00000);
                    if (again) {
                        const float was = __ldcg(before + row), most = fmaxf(was, top);
                        const float f = was == most ? 1.f : ex2(was - most), h = top == most ? 1.f : ex2(top - most);
                        sum = fmaf(sum, h, __ldcg(before + N + row) * f);
                        v = fmaf(v, h, __ldcg(part + row * D + dim) * f);
                        top = most;
                    }
                    if (whole && !left) store(c, row, dim, v, top, sum);
                    else {
                        __stcg(part + row * D + dim, v);
                        if (dim == 0) { __stcg(tops + row, top); __stcg(tops + N + row, sum); }
                    }
                }
        }
        asm volatile("tcgen05.fence::before_thread_sync;");
        if (whole || left) {
            group_sync(1, kSoftmax);       // (the next segment's rows come over these)
            return;
        }
        const int last = (int)((seg1 * ctas - 1) / all), n = last - lead + 1;
        __threadfence();
        group_sync(1, kSoftmax);
        if (tid == 0) {
            int* ticket = (int*)a.workspace + lead;
            const int seen = atomicAdd(ticket, 1);
            if (seen == n - 1) {
                *ticket = 0;       // as the next call wants it
                __threadfence();
            }
            s.last = seen == n - 1;
        }
        group_sync(1, kSoftmax);
        if (!s.last) return;
        // the weights of the parts, [row][part]
        float* tw = s.weight + N * kCtas;
        for (int row = warp; row < N; row += kSoftmax / 32) {
            float top = kNoMaximum, sum = 0.f;
            for (int i = lane; i < n; i += 32) top = fmaxf(top, __ldcg(partial(lead + i, i == 0) + N * D + row));
#pragma unroll
            for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
            for (int i = lane; i < n; i += 32) {
                const float* p = partial(lead + i, i == 0) + N * D + row;
                const float mi = __ldcg(p), f = mi == top ? 1.f : ex2(mi - top);
                s.weight[row * kCtas + i] = f;
                sum += __ldcg(p + N) * f;
            }
            sum = sili::warp_sum(sum);
            if (lane == 0) { tw[row] = top; tw[N + row] = sum; }
        }
        group_sync(1, kSoftmax);
        constexpr int kQuads = D / 4;
        for (int i = tid; i < N * kQuads; i += kSoftmax) {
            const int row = i / kQuads, d = i % kQuads * 4;
            if (row_id(c, row) < 0) continue;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
            for (int k = 0; k < n; ++k) {
                const float f = s.weight[row * kCtas + k];
                const float4 p = __ldcg((const float4*)(partial(lead + k, k == 0) + row * D + d));
                v[0] += p.x * f; v[1] += p.y * f; v[2] += p.z * f; v[3] += p.w * f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) store(c, row, d + k, v[k], tw[row], tw[N + row]);
        }
        group_sync(1, kSoftmax);
    }

    __device__ __forceinline__ void softmax(const Cur& c0) {
        int piece = 0;
        pieces(c0, [&](const Cur& c, int here, bool again, int left, int done) {
            int all_from, all_to;
            float l[kCols];
            begin_segment(c, l, all_from, all_to);
            for (int i = 0; i < here; ++i) unit(c, l, (c.u + i) * kUnit, i, done + i, all_from, all_to);
            const int64_t seg0 = begin + done - (c.u - c.q.k0);
            end_piece(c, l, piece++, seg0, seg0 + c.q.units, again, left);
            return true;
        });
    }
};

template <typename T, int D, int N>
__global__ void __launch_bounds__(kThreads, 1) k_tree(const __grid_constant__ AttendArgs a) {
    extern __shared__ uint8_t raw[];
    using S = Smem<D, N>;
    S& s = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
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
    Cursor<N> c;
    Tree<T, D, N> k{a, s};
    k.all = sili::locate<N, kThreads / 32>(a, c, blockIdx.x, gridDim.x, k.begin, k.end);
    if (k.begin >= k.end) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&s.k_full[i], kDequant);
            bar_init(&s.k_free[i], 1);
            bar_init(&s.v_full[i], kDequant);
            bar_init(&s.v_free[i], 1);
            bar_init(&s.s_full[i], 1);
            bar_init(&s.s_free[i], kSoftmax);
        }
        bar_init(&s.p_full, kSoftmax);
        bar_init(&s.p_free, 1);
        bar_init(&s.q_full, kSoftmax);
        bar_init(&s.o_full, 1);
        bar_init(&s.drained, 1);
        for (int i = 0; i < 4; ++i) s.odd[i] = 0;
        s.progress = s.dead = 0;
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
        if (warp == kMmaWarp && (threadIdx.x & 31) == 0) k.products(c);
        else if (warp == kFetchWarp) k.fetch(c);
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (*(volatile int*)&s.dead) {     // (every role has left its loop: it is the same for all threads)
        // the products that the thread has queued may still run: it waits for them (bounded) before the tensor memory is freed
        if (threadIdx.x == kMmaWarp * 32) {
            atomicOr((unsigned*)a.workspace + sili::kErrorWord, 1u);
            int quiet = 0;
            commit(&s.drained);
            bar_wait(&s.drained, 0, &quiet, 4096);
        }
        __syncthreads();
    }
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem), "r"(512));
}

template <typename T, int D, int N>
int launch(const AttendArgs& a, cudaStream_t s) {
    constexpr int smem = (int)sizeof(Smem<D, N>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    static_assert((int64_t)kCtas * 2 * N * (D + 4) * 4 <= sili::kSlotBytes, "the workspace holds the parts");
    auto kernel = k_tree<T, D, N>;
    static std::atomic<uint64_t> set{0};
    CKT(sili::allow_smem(kernel, smem, set));
    kernel<<<kCtas, kThreads, smem, s>>>(a);
    sili::count_launch();
    CKT(cudaGetLastError());
    return SILI_OK;
}
template <typename T, int D>
int by_rows(const AttendArgs& a, int64_t rows, cudaStream_t s) {
    return rows <= 32 ? launch<T, D, 32>(a, s) : rows <= 64 ? launch<T, D, 64>(a, s) : launch<T, D, 128>(a, s);
}

}  // namespace

namespace sili {

bool kv4_tree_takes(int dtype, int dim, int64_t rows) { return dtype != SILI_F32 && (dim == 64 || dim == 128) && rows > 16; }

int kv4_tree_launch(int dtype, int dim, const AttendArgs& args, int64_t rows, cudaStream_t s) {
    AttendArgs a = args;
    kv4_polls(a);
    if (dtype == SILI_F16) return dim == 64 ? by_rows<__half, 64>(a, rows, s) : by_rows<__half, 128>(a, rows, s);
    return dim == 64 ? by_rows<__nv_bfloat16, 64>(a, rows, s) : by_rows<__nv_bfloat16, 128>(a, rows, s);
}

}  // namespace sili
