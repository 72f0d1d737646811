// Attention over the 4-bit paged cache on the warp's matrix instructions, for
// decode steps (one or a few queries a request), for fp32 activations, and
// for short prompts; long 16-bit prompts run in kv4_prompt.cu.
//
// For one kv head of one request, with rows rho = (query token, query head of
// the group), the kernel accumulates the transposed products
//   S^T [keys, rows] = K Q^T,   O^T [dim, rows] += V^T P^T
// so that the cache is always the 16-row operand of mma.m16n8k16 and few
// query rows fill the 8-wide one.  The 4-bit operands are turned into exact
// halves in registers: cvt.f16x2.e2m1x2 of the stored bytes times the group's
// scale (2 + 4 significant bits).  K bytes lie as the fragment wants them (a
// thread's dim/4 consecutive elements are its share of every k step); V wants
// two keys in one register, so the nibbles of two keys are interleaved before
// the conversion (4 logic operations for 16 values).
//
// fp32 queries and probabilities are split into two halves (hi + lo, 22 bits,
// after scaling a row by a power of two).  16-bit queries are one half: fp16 as
// they are, bf16 scaled likewise, exact down to 2^-31 of a row's largest and
// within 2^-39 of it below.  Their probabilities are rounded to one half, by at
// most 2^-11 of themselves (their sum is taken before): the output's own half
// unit in fp16 for few keys, less over many, where the errors average; a second
// half would double the products.  Sums, maxima and outputs are fp32; 16-bit
// sums lie in the matrix unit's accumulators, which it cuts (see kPiece).  The running
// maximum is moved only when a logit exceeds it by 2^7 (p <= 2^15 is still a
// half): a warp vote in place of a reduction per tile.
//
// Work is cut evenly whatever the lengths: a unit is 128 keys of one (request,
// kv head, row tile), all units are numbered in order, and each of the
// launch's CTAs takes an equal run of them, found from the lengths on the
// device.  A segment (all units of one row tile) that several CTAs share is
// joined by whichever of them finishes last, in CTA order, so the result does
// not depend on which that is.  Warps take 16 keys each (within one page) and
// keep a ring of cp.async stages; the page of the next tile is fetched one
// step ahead.
//
// What bounds it, 96 requests of 2k-16k keys, 32 heads over 8, dim 128, bf16
// (0.96 GB, 146 us at the card's copy rate): 271 us, 3.5 TB/s.  A warp's 16
// keys x 136 bytes take about 400 instructions, 266 of them the tile's own
// (64 conversions at half rate, 64 scalings, 16 products, the softmax); the
// schedulers issue two of three cycles with 16 warps an SM, which registers
// (128 a thread) and the ring (104 KB a CTA) allow.  With 8 warps an SM and a
// longer ring it took 389 us; with bulk copies by one lane in place of
// cp.async by all, 355 against 325 at the time.  A few short requests (4, up
// to 700 keys) are a chain of latencies, 15 us: lengths, query, page, keys, the
// join of the parts (with at least 4 units a CTA in place of 1: 18 us).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kernels.cuh"
#include "kv4_attention.cuh"
#include "sili_b200.h"

namespace sili {
int set_error(int code, const std::string& msg);
}

namespace {

#define CKV(x)                                                                                          \
    do {                                                                                                \
        const cudaError_t e_ = (x);                                                                     \
        if (e_ != cudaSuccess)                                                                          \
            return sili::set_error(e_ == cudaErrorMemoryAllocation ? SILI_ENOMEM : SILI_ECUDA,          \
                                   std::string(#x) + ": " + cudaGetErrorString(e_));                    \
    } while (0)

using sili::AttendArgs;
using sili::ex2;
using sili::kLift;
using sili::kLn2;
using sili::kLog2e;
using sili::kSlack;
using sili::kTicketBytes;
using sili::mul2;
using sili::pack2;

int bad(const char* who, const char* what) {
    return sili::set_error(SILI_EINVAL, std::string(who) + ": " + what);
}

constexpr int kWarps = 8;
constexpr int kUnit = 16 * kWarps;      // keys of a unit
constexpr int kMaxStages = 4;
// Units of a segment that a warp's 16-bit sums take in at most.  The matrix unit cuts what it adds to an accumulator
// towards zero, 7e-8 a product where V has one sign: 5.8e-4, more than fp16's half unit, after the 8192 products of a
// warp whose CTA walked 1048576 keys.  So a longer run is walked in pieces, whose sums are added in the workspace, rounded
// (7e-5 is left).  In the loop itself the same cost 13 % of a decode batch, by its registers.
constexpr int kPiece = 1024;
constexpr float kNoMaximum = -3e38f;    // below every finite logit, and finite: a masked key's -inf over it is -inf
constexpr int kMaxCtas = 2 * 148;       // two CTAs an SM; one for the wider row tiles

static_assert(kMaxCtas <= sili::kSlotWord, "the counters end before the slots' bits");
constexpr int64_t workspace_bytes() {
    // two partial results a CTA: rows * (dim + 4) floats
    return kTicketBytes + std::max((int64_t)kMaxCtas * 2 * 32 * 132 * 4, sili::kSlotBytes);
}

template <int E, int NT>
struct Layout {
    static constexpr int kDim = 32 * E, kRowBytes = kDim / 2, kRows = 8 * NT;
    static constexpr int kStages = E == 8 && NT == 2 ? 2 : kMaxStages;   // what shared memory holds beside the join space
    static constexpr int kCodes = 16 * kRowBytes, kScales = 16 * E;
    static constexpr int kStage = 2 * (kCodes + kScales);
    static constexpr int kJoinRow = kDim + 4;           // floats; + 4 spreads the rows over the banks
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kJoin = kWarps * kRows * (kJoinRow + 2) * 4;
};
// The Q fragments lie in shared memory where the registers are needed: wide
// row tiles, and fp32's two terms beside a second CTA (128 registers a thread:
// in registers they spill, 160 against 133 us on the fp32 decode batch).
template <typename T, int E, int NT>
constexpr bool q_shared() {
    return NT > 1 || (sizeof(T) == 4 && E < 8);
}
template <typename T, int E, int NT>
constexpr int smem_bytes() {
    using L = Layout<E, NT>;
    constexpr int terms = sizeof(T) == 4 ? 2 : 1;
    return L::kRing + L::kJoin + (q_shared<T, E, NT>() ? NT * 2 * E * terms * 32 * 8 : 0);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src));
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// what is left of (lo, hi) after rounding to the halves h
__device__ __forceinline__ uint32_t rest2(float lo, float hi, uint32_t h) {
    const float2 f = sili::half2_bits_to_float2(h);
    return pack2(lo - f.x, hi - f.y);
}

// One request's share of the work.
struct Req {
    int row0, nq, len;     // first query row, queries, keys
    int64_t pos0;          // position of the first query (negative: it sees nothing)
    int k0, units, tiles;  // first unit of keys, units and row tiles
};

template <int ROWS>
__device__ __forceinline__ Req request(const AttendArgs& a, int r) {
    Req q;
    int64_t s0 = r, s1 = r + 1;
    if (a.starts) { s0 = a.starts[r]; s1 = a.starts[r + 1]; }
    const int64_t past = s1;     // may lie beyond the rows of q: those that are there keep their positions
    s0 = min(max(s0, (int64_t)0), a.tokens);
    s1 = min(max(s1, s0), a.tokens);
    q.row0 = (int)s0;
    q.nq = (int)(s1 - s0);
    const int all = max(a.lens[r], 0);
    q.len = (int)min(min((int64_t)all, (int64_t)a.width * a.page), (int64_t)0x7FFFFF00);
    q.pos0 = all - (past - s0);
    const int64_t from = a.window ? max(q.pos0 - a.window + 1, (int64_t)0) : 0;
    q.k0 = (int)(from / kUnit);
    q.units = max((q.len + kUnit - 1) / kUnit - q.k0, 1);
    const int group = a.heads / a.kv_heads;
    q.tiles = (q.nq * group + ROWS - 1) / ROWS;
    return q;
}
__device__ __forceinline__ int64_t units_of(const AttendArgs& a, const Req& q) {
    return (int64_t)q.units * q.tiles * a.kv_heads;
}

// A position in the numbered units: request, kv head, row tile (a segment)
// and unit of keys.
template <int ROWS>
struct Cursor {
    Req q;
    int r, h, tile, u;

    __device__ __forceinline__ int left() const { return q.k0 + q.units - u; }    // units of the segment from u on
    // the first unit of the next segment (past the last one: never looked at)
    __device__ __forceinline__ void next_segment(const AttendArgs& a) {
        if (++tile == q.tiles) {
            tile = 0;
            if (++h == a.kv_heads) {
                h = 0;
                do {
                    if (++r >= a.requests) return;
                    q = request<ROWS>(a, r);
                } while (q.tiles == 0);
            }
        }
        u = q.k0;
    }
};

// The CTA's run [begin, end) of the units, `c` set to its first; returns the
// number of all units.  One scan of the lengths by the CTA.
template <int ROWS>
__device__ int64_t locate(const AttendArgs& a, Cursor<ROWS>& c, int cta, int ctas, int64_t& begin, int64_t& end) {
    __shared__ int64_t s_part[kWarps], s_hit[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t mine = 0;
    for (int r = tid; r < a.requests; r += kWarps * 32) mine += units_of(a, request<ROWS>(a, r));
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) s_part[warp] = mine;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all += s_part[w];
    ctas = (int)min((int64_t)ctas, all);    // no more CTAs than units: every one of them has some
    if (cta >= ctas) { begin = end = 0; return all; }
    begin = all * cta / ctas;
    end = all * (cta + 1) / ctas;
    int64_t before = 0;
    for (int base = 0; base < a.requests; base += kWarps * 32) {
        const int r = base + tid;
        const int64_t n = r < a.requests ? units_of(a, request<ROWS>(a, r)) : 0;
        int64_t x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t t = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += t;
        }
        __syncthreads();
        if (lane == 31) s_part[warp] = x;
        __syncthreads();
        int64_t total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) x += s_part[w];
            total += s_part[w];
        }
        x += before;
        if (x - n <= begin && begin < x) { s_hit[0] = r; s_hit[1] = begin - (x - n); }
        before += total;
        if (begin < before) break;
    }
    __syncthreads();
    c.r = (int)s_hit[0];
    c.q = request<ROWS>(a, c.r);
    const int64_t seg = s_hit[1] / c.q.units;
    c.u = c.q.k0 + (int)(s_hit[1] - seg * c.q.units);
    c.h = (int)(seg / c.q.tiles);
    c.tile = (int)(seg - (int64_t)c.h * c.q.tiles);
    return all;
}

template <typename T, int E, int NT>
struct Attend {
    using L = Layout<E, NT>;
    static constexpr int kStages = L::kStages;
    static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;
    static constexpr int kDim = L::kDim, kRows = L::kRows, kSteps = kDim / 16;
    static constexpr bool kShared = q_shared<T, E, NT>();
    using Cur = Cursor<kRows>;

    const AttendArgs& a;
    const int lane, warp, g, t;
    uint8_t* ring;         // this warp's stages
    uint32_t ring_at;
    uint32_t held = 0;     // a bit a stage: its tile holds keys
    float* s_cf;           // the row tiles' logit factors (q_shared)
    int step_pages, step_off;   // a unit of keys in table entries and rows
    float* join;
    uint32_t* qs;          // Q fragments in shared memory (kShared)

    // the current segment
    uint32_t qf[kShared ? 1 : kSteps][kTerms][2];
    float cf[NT][2];       // logit = S * cf, in powers of two
    float base[NT][2];     // the running maximum - lift
    float l[NT][2], o[kSteps][NT][4];
    int to[NT][2], from[NT][2];        // the columns' keys [from, to)
    int any_from, any_to, all_from, all_to;   // keys that any of the rows sees, that every row sees

    __device__ __forceinline__ Attend(const AttendArgs& args, uint8_t* smem, float* factors)
        : a(args), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), g(lane >> 2), t(lane & 3) {
        ring = smem + warp * (kStages * L::kStage);
        ring_at = (uint32_t)__cvta_generic_to_shared(ring);
        s_cf = factors;
        step_pages = kUnit / a.page;
        step_off = kUnit - step_pages * a.page;
        join = (float*)(smem + L::kRing);
        qs = (uint32_t*)(smem + L::kRing + L::kJoin);
    }

    // the key of S's row m (the same permutation in both halves of 8): a thread's four P entries are then keys
    // t, 4 + t, 8 + t, 12 + t, whose V rows it reads without bank conflicts
    static __device__ __forceinline__ int key_of(int m) { return (m >> 1) + 4 * (m & 1); }

    // 16-byte chunk c of a key's code row, as stored in a stage
    static __device__ __forceinline__ int k_chunk(int key, int c) { return E == 8 ? c ^ ((key >> 2) & 1) : c; }
    static __device__ __forceinline__ int v_chunk(int key, int c) {
        return E == 8 ? c ^ (2 * (key & 3)) : E == 4 ? c ^ (2 * ((key >> 1) & 1)) : c;
    }

    // What the copies of this warp's tiles need, a tile ahead of them: within a segment a step is an addition to `key0`.
    struct Loader {
        Cur c;
        int key0, left, len;     // the next tile's first key, the segment's tiles from there on, the request's keys
        int page, off;           // its page (-1: none) and place in it
        const int* entry;        // its entry in the table
        const uint8_t *codes, *scales;   // the kv head's first K row of page 0, and this lane's 16 bytes
    };
    __device__ __forceinline__ void look(Loader& d) const {
        d.page = d.key0 < d.len ? __ldg(d.entry) : -1;
    }
    __device__ __forceinline__ void enter(Loader& d) const {
        d.key0 = d.c.u * kUnit + warp * 16;
        d.left = d.c.left();
        d.len = d.c.q.len;
        d.entry = a.table + d.c.r * a.stride + a.column(d.key0, d.off);
        const int64_t rows = (int64_t)d.c.h * a.page;
        d.codes = a.codes + rows * L::kRowBytes + lane * 16;
        d.scales = a.scales + rows * E + (lane % (L::kScales / 16)) * 16;
    }
    __device__ __forceinline__ void step(Loader& d, bool more) const {
        d.key0 += kUnit;
        d.entry += step_pages;
        d.off += step_off;
        if (d.off >= a.page) { d.off -= a.page; ++d.entry; }
        if (--d.left == 0 && more) {
            d.c.next_segment(a);
            enter(d);
        }
        if (more) look(d);
    }

    // starts the copy of the loader's tile into stage s
    __device__ __forceinline__ void issue(const Loader& d, int s) {
        const bool there = (unsigned)d.page < (unsigned)a.n_pages;
        if (there) {
            // (the host has checked that a page's bytes fit 31 bits)
            const uint32_t half = a.half_rows;
            const uint8_t* k = d.codes + (uint64_t)(uint32_t)d.page * (2 * half * L::kRowBytes) + d.off * L::kRowBytes;
            const uint8_t* v = k + half * L::kRowBytes;
            const uint32_t at = ring_at + s * L::kStage;
            constexpr int kPer = L::kRowBytes / 16, kStep = 32 / kPer;     // lanes a key, keys of one copy instruction
            const int key = lane / kPer, c16 = lane % kPer;
            // the chunks' swizzles go by key bits that a step of kStep keys leaves alone
            static_assert(E == 8 || kStep % 4 == 0, "swizzle");
#pragma unroll
            for (int i = 0; i < 16 / kStep; ++i) {
                const int kk = E == 8 ? key + i * kStep : key;
                cp16(at + (key + i * kStep) * L::kRowBytes + k_chunk(kk, c16) * 16, k + i * 512);
                cp16(at + L::kCodes + (key + i * kStep) * L::kRowBytes + v_chunk(kk, c16) * 16, v + i * 512);
            }
            constexpr int kSc = L::kScales / 16;
            if (lane < 2 * kSc) {
                const uint8_t* p = d.scales + (uint64_t)(uint32_t)d.page * (2 * half * E) + d.off * E;
                cp16(at + 2 * L::kCodes + lane * 16, lane >= kSc ? p + half * E : p);
            }
        }
        held = there ? held | 1u << s : held & ~(1u << s);
    }

    __device__ __forceinline__ void begin_segment(const Cur& c) {
        const int h = c.h, group = a.heads / a.kv_heads;
        const int rows = c.q.nq * group, row0 = c.tile * kRows;     // below 2^31: the host has checked tokens * heads
        auto span = [&](int row, int& from_, int& to_) {
            const int64_t pos = c.q.pos0 + row / group;
            to_ = (int)min(pos + 1, (int64_t)c.q.len);
            from_ = a.window ? (int)max(pos - a.window + 1, (int64_t)0) : 0;
        };
        span(row0, any_from, all_to);
        span(min(row0 + kRows, rows) - 1, all_from, any_to);
        if (kShared) __syncthreads();    // the last segment's fragments have been read
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = row0 + n * 8 + g;
            const bool real = row < rows;
            const int64_t tok = c.q.row0 + (real ? row / group : 0);
            const int head = h * group + (real ? row % group : 0);
            const T* src = (const T*)a.q + tok * a.qt + head * a.qh + t * (kDim / 4);
            constexpr int kPart = 8 / sizeof(T) < 4 ? 2 : 4;     // elements of an 8-byte access
            // shared: warp n alone prepares row tile n for all
            if (!kShared || warp == n) {
                float f = 1.f, x[kDim / 4];
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < kDim / 4; i += kPart) {
                    sili::Pack<T, kPart> p;
                    if (real) p = *(const sili::Pack<T, kPart>*)(src + i);
#pragma unroll
                    for (int j = 0; j < kPart; ++j) {
                        x[i + j] = real ? sili::to_f32(p.v[j]) : 0.f;
                        top = max(top, __float_as_uint(x[i + j]) & 0x7FFFFFFFu);
                    }
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // the row's largest into [2^14, 2^15): a half holds it, and 38 binary digits below it
                int e = 0;
                const float sign = a.scale < 0.f ? -1.f : 1.f;
                if (!std::is_same<T, __half>::value && top && top < 0x7F800000u) {
                    e = 14 - max((int)(top >> 23) - 127, -100);
                    f = __int_as_float((127 + e) << 23);
                }
                f *= sign;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const float u = x[4 * i + 2 * p] * f, v = x[4 * i + 2 * p + 1] * f;
                        const uint32_t hi = pack2(u, v);
                        if (!kShared) qf[kShared ? 0 : i][0][p] = hi;
                        else qs[(((n * kSteps + i) * kTerms) * 32 + lane) * 2 + p] = hi;
                        if (kTerms == 2) {
                            const uint32_t lo = rest2(u, v, hi);
                            if (!kShared) qf[kShared ? 0 : i][kTerms - 1][p] = lo;
                            else qs[(((n * kSteps + i) * kTerms + kTerms - 1) * 32 + lane) * 2 + p] = lo;
                        }
                    }
                }
                // undo the scaling (the scale's sign is in q; not 0, which would undo a mask's -inf); the thread's columns are rows 2t and 2t + 1, held by lanes of g = 2t, 2t + 1
                const float back = fmaxf(fabsf(a.scale) * kLog2e * __int_as_float((127 - e) << 23), 0x1p-126f);
                cf[n][0] = __shfl_sync(0xffffffffu, back, 8 * t);
                cf[n][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
                if (kShared) {
                    if (t == 0) s_cf[n * 8 + g] = back;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                span(min(row0 + n * 8 + 2 * t + j, rows - 1), from[n][j], to[n][j]);
                base[n][j] = kNoMaximum;
                l[n][j] = 0.f;
            }
        }
        if (kShared) {
            __syncthreads();
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) cf[n][j] = s_cf[n * 8 + 2 * t + j];
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][n][j] = 0.f;
    }

    __device__ __forceinline__ bool sees(int key, int n, int j) const { return key < to[n][j] && key >= from[n][j]; }

    // Moves the columns' maxima to those of these keys' products x where they are larger; e: the exponents over them.
    __device__ __forceinline__ void raise(const float (&x)[NT][4], float (&e)[NT][4]) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float top = fmaxf(x[n][j], x[n][j + 2]) * cf[n][j];
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                const float fresh = fmaxf(base[n][j], top - kLift);
                const float f = fresh == base[n][j] ? 1.f : ex2(base[n][j] - fresh);
                base[n][j] = fresh;
                l[n][j] *= f;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) { o[i][n][j] *= f; o[i][n][j + 2] *= f; }
                e[n][j] = fmaf(x[n][j], cf[n][j], -fresh);
                e[n][j + 2] = fmaf(x[n][j + 2], cf[n][j], -fresh);
            }
    }

    __device__ __forceinline__ void tile(int key0, int s) {
        if (!(held >> s & 1) || key0 >= any_to || key0 + 16 <= any_from) return;
        const uint8_t* st = ring + s * L::kStage;
        const int ka = key_of(g);
        float x[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[n][j] = 0.f;
        {   // S^T = K Q^T
            constexpr int kWords = kDim / 32;      // words of codes a thread and row
            uint32_t w[2][kWords];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int key = ka + 8 * i;
                const uint8_t* row = st + key * L::kRowBytes;
                if constexpr (E == 2) {
                    const uint2 v = *(const uint2*)(row + t * 8);
                    w[i][0] = v.x; w[i][1] = v.y;
                } else {
#pragma unroll
                    for (int q = 0; q < E / 4; ++q) {
                        const uint4 v = *(const uint4*)(row + k_chunk(key, t * (E / 4) + q) * 16);
                        w[i][4 * q] = v.x; w[i][4 * q + 1] = v.y; w[i][4 * q + 2] = v.z; w[i][4 * q + 3] = v.w;
                    }
                }
            }
            const uint8_t* sc = st + 2 * L::kCodes;
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const int grp = E == 2 ? t >> 1 : E == 4 ? t : 2 * t + j / 4;
                uint32_t f[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t sb = sc[(ka + 8 * i) * E + grp] * 0x00800080u;
                    sili::kv4_decode4(w[i][j], f[i]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) f[i][q] = mul2(f[i][q], sb);
                }
                // (fp32: two steps at a time, small terms first, added outside the matrix unit, which cuts: see below)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int q = kTerms - 1; q >= 0; --q)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint32_t b0, b1;
                            if (!kShared) { b0 = qf[kShared ? 0 : 2 * j + k][q][0]; b1 = qf[kShared ? 0 : 2 * j + k][q][1]; }
                            else {
                                const uint2 b = ((const uint2*)qs)[((n * kSteps + 2 * j + k) * kTerms + q) * 32 + lane];
                                b0 = b.x; b1 = b.y;
                            }
                            mma(kTerms == 1 ? x[n] : sum, f[0][2 * k], f[1][2 * k], f[0][2 * k + 1], f[1][2 * k + 1], b0, b1);
                        }
                    if (kTerms == 2)
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[n][k] += sum[k];
                }
            }
        }
        // exponents over the running maximum
        float e[NT][4];
        if (!(key0 + 16 <= all_to && key0 >= all_from)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!sees(key0 + ka + 8 * (j >> 1), n, j & 1)) x[n][j] = -INFINITY;
        }
        bool above = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                e[n][j] = fmaf(x[n][j], cf[n][j & 1], -base[n][j & 1]);
                above = above || e[n][j] > kLift + kSlack;
            }
        if (__any_sync(0xffffffffu, above)) raise(x, e);
        // P^T fragments
        uint32_t p[NT][kTerms][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[n][j] = ex2(e[n][j]);
                l[n][j & 1] += x[n][j];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t hi = pack2(x[n][2 * i], x[n][2 * i + 1]);
                if (kTerms == 2) p[n][kTerms - 1][i] = transpose8(rest2(x[n][2 * i], x[n][2 * i + 1], hi));
                p[n][0][i] = transpose8(hi);
            }
        }
        {   // O^T += V^T P^T
            constexpr int kWords = kDim / 64;      // words of codes a thread and key
            const uint8_t* vs = st + L::kCodes;
            const uint8_t* sc = st + 2 * L::kCodes + L::kScales;
            const int grp = E == 2 ? g >> 2 : E == 4 ? g >> 1 : g;
            uint32_t w[4][kWords], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 4 * i + t;
                const uint8_t* row = vs + key * L::kRowBytes;
                if constexpr (E == 2) w[i][0] = *(const uint32_t*)(row + g * 4);
                else if constexpr (E == 4) {
                    const uint2 v = *(const uint2*)(row + v_chunk(key, g >> 1) * 16 + (g & 1) * 8);
                    w[i][0] = v.x; w[i][1] = v.y;
                } else {
                    const uint4 v = *(const uint4*)(row + v_chunk(key, g) * 16);
                    w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
                }
                b[i] = sc[key * E + grp];
            }
            // A scale that is not a number reaches only the rows that see its key: such groups are left out of the
            // product (0 * NaN would reach every row) and entered by hand.
            const bool odd = max(max(b[0], b[1]), max(b[2], b[3])) >= 0xF8u;
            if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i] = b[i] >= 0xF8u ? 0u : b[i];
                for (int key = 0; key < 16; ++key) {
                    if (sc[key * E + grp] < 0xF8u) continue;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            if (sees(key0 + key, n, j))
#pragma unroll
                                for (int i = 0; i < kSteps; ++i)
                                    o[i][n][j] = o[i][n][j + 2] = __int_as_float(0x7FC00000);
                }
            }
            const uint32_t s01 = b[0] << 7 | b[1] << 23, s23 = b[2] << 7 | b[3] << 23;
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                constexpr uint32_t kLow = 0x0F0F0F0Fu;
                uint32_t f[4][4];      // keys (t, 4 + t) even / odd elements, then keys (8 + t, 12 + t)
                sili::kv4_decode4((w[0][j] & kLow) | ((w[1][j] << 4) & ~kLow), f[0]);
                sili::kv4_decode4(((w[0][j] >> 4) & kLow) | (w[1][j] & ~kLow), f[1]);
                sili::kv4_decode4((w[2][j] & kLow) | ((w[3][j] << 4) & ~kLow), f[2]);
                sili::kv4_decode4(((w[2][j] >> 4) & kLow) | (w[3][j] & ~kLow), f[3]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t a0 = mul2(f[0][q], s01), a1 = mul2(f[1][q], s01), a2 = mul2(f[2][q], s23),
                                   a3 = mul2(f[3][q], s23);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        if (kTerms == 1) {
                            mma(o[4 * j + q][n], a0, a1, a2, a3, p[n][0][0], p[n][0][1]);
                        } else {
                            // The matrix unit cuts what it adds to its accumulator, always towards zero: over a few
                            // hundred tiles that is 3e-6 of O.  So fp32's tiles are added outside, rounded.
                            float sum[4] = {0.f, 0.f, 0.f, 0.f};
                            mma(sum, a0, a1, a2, a3, p[n][kTerms - 1][0], p[n][kTerms - 1][1]);
                            mma(sum, a0, a1, a2, a3, p[n][0][0], p[n][0][1]);
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[4 * j + q][n][k] += sum[k];
                        }
                }
            }
        }
    }

    // a part of a segment: [row][dim] sums, then the rows' maxima and the sums of their probabilities; those twice, so that
    // the pieces of a run write the one while the other is read
    __device__ __forceinline__ float* partial(int cta, int slot) const {
        return (float*)((uint8_t*)a.workspace + kTicketBytes) + (int64_t)(cta * 2 + slot) * kRows * (kDim + 4);
    }

    // out and lse of one row and four of its values
    __device__ __forceinline__ void store(const Cur& c, int row, int d, const float (&v)[4], float top, float sum) const {
        const int h = c.h, group = a.heads / a.kv_heads;
        const int at = c.tile * kRows + row;
        if (at >= c.q.nq * group) return;
        const int64_t id = (int64_t)(c.q.row0 + at / group) * a.heads + h * group + at % group;
        // sum 0: the row saw nothing; NaN goes through
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        sili::Pack<T, 4> out;
#pragma unroll
        for (int i = 0; i < 4; ++i) out.v[i] = sili::from_f32<T>(v[i] * inv);
        *(sili::Pack<T, 4>*)((T*)a.out + id * kDim + d) = out;
        if (d == 0 && a.lse) a.lse[id] = sum == 0.f ? -INFINITY : kLn2 * (top + log2f(sum));
    }

    // The segment's end in this CTA: joins the warps, then writes the rows, or leaves them to the CTA that comes last.
    // seg0 and seg1 number the segment's first unit and the one past its last.  Of a run in pieces, the first ones (`left`
    // pieces follow) only leave their sums, and the others (`again`) add those before to theirs.
    __device__ __forceinline__ void end_segment(const Cur& c, int64_t seg0, int64_t seg1, int64_t begin, int64_t end,
                                                int64_t all, int* s_last, bool again, int left) {
        constexpr int kThreads = kWarps * 32, kQuads = kDim / 4;
        float* jm = join + kWarps * kRows * L::kJoinRow;       // [warp][row] maxima, then sums
        float* jl = jm + kWarps * kRows;
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float s = l[n][j];
                s += __shfl_xor_sync(0xffffffffu, s, 4);
                s += __shfl_xor_sync(0xffffffffu, s, 8);
                s += __shfl_xor_sync(0xffffffffu, s, 16);
                const int row = warp * kRows + n * 8 + 2 * t + j;
                if (g == 0) { jm[row] = base[n][j]; jl[row] = s; }
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
                    *(float2*)(join + row * L::kJoinRow + g * (kDim / 8) + 2 * i) = make_float2(o[i][n][j], o[i][n][j + 2]);
            }
        __syncthreads();
        const bool whole = seg0 >= begin && seg1 <= end;
        const int64_t ctas = min((int64_t)gridDim.x, all);
        const int cta = blockIdx.x;
        const int lead = whole ? cta : (int)(((seg0 + 1) * ctas - 1) / all);
        // (a whole segment's pieces use the place of the segment that this CTA begins last)
        float* part = partial(cta, cta == lead);
        float* tops = part + kRows * (kDim + 2 * (left & 1));
        for (int i = threadIdx.x; i < kRows * kQuads; i += kThreads) {
            const int row = i / kQuads, d = i % kQuads * 4;
            float top = kNoMaximum, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, jm[w * kRows + row]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float mw = jm[w * kRows + row], f = mw == top ? 1.f : ex2(mw - top);
                const float4 p = *(const float4*)(join + (w * kRows + row) * L::kJoinRow + d);
                sum += jl[w * kRows + row] * f;
                v[0] += p.x * f; v[1] += p.y * f; v[2] += p.z * f; v[3] += p.w * f;
            }
            if (kTerms == 1 && again) {
                const float* before = part + kRows * (kDim + 2 * (~left & 1));
                const float was = __ldcg(before + row), most = fmaxf(was, top);
                const float f = was == most ? 1.f : ex2(was - most), h = top == most ? 1.f : ex2(top - most);
                const float4 p = __ldcg((const float4*)(part + row * kDim + d));
                sum = fmaf(sum, h, __ldcg(before + kRows + row) * f);
                v[0] = fmaf(v[0], h, p.x * f); v[1] = fmaf(v[1], h, p.y * f);
                v[2] = fmaf(v[2], h, p.z * f); v[3] = fmaf(v[3], h, p.w * f);
                top = most;
            }
            if (whole && !left) store(c, row, d, v, top, sum);
            else {
                __stcg((float4*)(part + row * kDim + d), make_float4(v[0], v[1], v[2], v[3]));
                if (d == 0) { __stcg(tops + row, top); __stcg(tops + kRows + row, sum); }
            }
        }
        if (whole || left) return;
        const int last = (int)((seg1 * ctas - 1) / all), n = last - lead + 1;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            int* ticket = (int*)a.workspace + lead;
            const int seen = atomicAdd(ticket, 1);
            if (seen == n - 1) {
                *ticket = 0;       // as the next call wants it
                __threadfence();
            }
            *s_last = seen == n - 1;
        }
        __syncthreads();
        if (!*s_last) return;
        // the weights of the parts, [row][part], in the warps' join space
        for (int row = warp; row < kRows; row += kWarps) {
            float top = kNoMaximum, sum = 0.f;
            for (int i = lane; i < n; i += 32)
                top = fmaxf(top, __ldcg(partial(lead + i, i == 0) + kRows * kDim + row));
#pragma unroll
            for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
            for (int i = lane; i < n; i += 32) {
                const float* p = partial(lead + i, i == 0) + kRows * kDim + row;
                const float mi = __ldcg(p), f = mi == top ? 1.f : ex2(mi - top);
                join[row * kMaxCtas + i] = f;
                sum += __ldcg(p + kRows) * f;
            }
#pragma unroll
            for (int k = 16; k; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
            if (lane == 0) { join[kRows * kMaxCtas + row] = top; join[kRows * kMaxCtas + kRows + row] = sum; }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kRows * kQuads; i += kThreads) {
            const int row = i / kQuads, d = i % kQuads * 4;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
            for (int k = 0; k < n; ++k) {
                const float f = join[row * kMaxCtas + k];
                const float4 p = __ldcg((const float4*)(partial(lead + k, k == 0) + row * kDim + d));
                v[0] += p.x * f; v[1] += p.y * f; v[2] += p.z * f; v[3] += p.w * f;
            }
            store(c, row, d, v, join[kRows * kMaxCtas + row], join[kRows * kMaxCtas + kRows + row]);
        }
    }

    __device__ __forceinline__ void run(Cur c, int64_t begin, int64_t end, int64_t all, int* s_last) {
        const int n = (int)(end - begin);
        Loader d;
        d.c = c;
        enter(d);
        look(d);
#pragma unroll 1
        for (int s = 0; s < kStages - 1; ++s) {
            if (s < n) {
                issue(d, s);
                step(d, s + 1 < n);
            }
            asm volatile("cp.async.commit_group;");
        }
        int stage = 0, done = 0;
        bool again = false;      // the segment's last piece lies behind
        while (done < n) {
            begin_segment(c);
            const int rest = min(c.left(), n - done), here = kTerms == 1 ? min(rest, kPiece) : rest;
            int key0 = c.u * kUnit + warp * 16;
#pragma unroll 1
            for (int i = 0; i < here; ++i, key0 += kUnit) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2));
                __syncwarp();
                const int ahead = done + i + kStages - 1;
                if (ahead < n) {
                    issue(d, stage == 0 ? kStages - 1 : stage - 1);
                    step(d, ahead + 1 < n);
                }
                asm volatile("cp.async.commit_group;");
                tile(key0, stage);
                stage = stage + 1 == kStages ? 0 : stage + 1;
            }
            const int64_t seg0 = begin + done - (c.u - c.q.k0);
            end_segment(c, seg0, seg0 + c.q.units, begin, end, all, s_last, kTerms == 1 && again,
                        kTerms == 1 ? (rest - here + kPiece - 1) / kPiece : 0);
            done += here;
            again = here < rest;
            if (again) c.u += here;
            if (!again && done < n) c.next_segment(a);
        }
    }
};

// rows of q that belong to no request
template <typename T>
__device__ void blank_rows(const AttendArgs& a, int dim) {
    const int64_t from = a.requests ? (a.starts ? min(max((int64_t)a.starts[0], (int64_t)0), a.tokens) : 0) : 0;
    const int64_t to = a.requests ? (a.starts ? min(max((int64_t)a.starts[a.requests], from), a.tokens)
                                              : min((int64_t)a.requests, a.tokens)) : 0;
    const int64_t per = (int64_t)a.heads * dim, skip = to - from, n = (a.tokens - skip) * per;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t x = i < from * per ? i : i + skip * per;
        ((T*)a.out)[x] = sili::from_f32<T>(0.f);
        if (a.lse && x % dim == 0) a.lse[x / dim] = -INFINITY;
    }
}

template <typename T, int E, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 && E < 8 ? 2 : 1) k_attend(const __grid_constant__ AttendArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_factors[8 * 4];
    __shared__ int s_last;
    blank_rows<T>(a, 32 * E);
    Cursor<8 * NT> c;
    int64_t begin, end;
    const int64_t all = locate<8 * NT>(a, c, blockIdx.x, gridDim.x, begin, end);
    if (begin >= end) return;
    Attend<T, E, NT> k(a, smem, s_factors);
    k.run(c, begin, end, all, &s_last);
}

template <typename T, int E, int NT>
int launch(const AttendArgs& a, cudaStream_t s) {
    constexpr int smem = smem_bytes<T, E, NT>();
    static_assert(8 * NT * (32 * E + 4) <= 32 * 132, "the workspace holds the widest row tile");
    static_assert(8 * NT * (kMaxCtas + 2) * 4 <= Layout<E, NT>::kJoin, "the parts' weights fit the join space");
    auto kernel = k_attend<T, E, NT>;
    static std::atomic<uint64_t> set{0};
    CKV(sili::allow_smem(kernel, smem, set));
    kernel<<<NT == 1 && E < 8 ? kMaxCtas : kMaxCtas / 2, kWarps * 32, smem, s>>>(a);
    sili::count_launch();
    CKV(cudaGetLastError());
    return SILI_OK;
}

// Row tiles of 8, 16 or 32 (query, head) rows: the narrowest that holds a
// request's rows, so that decoding wastes no columns and prompts read the
// cache least often (registers hold no wider one: 32 rows x 128, 16 x 256).
template <typename T, int E>
int by_rows(const AttendArgs& a, int64_t rows, cudaStream_t s) {
    if (rows <= 8) return launch<T, E, 1>(a, s);
    if (rows <= 16 || E == 8) return launch<T, E, 2>(a, s);
    return launch<T, E, E == 8 ? 2 : 4>(a, s);
}
template <typename T>
int by_dim(const AttendArgs& a, int dim, int64_t rows, cudaStream_t s) {
    return dim == 64 ? by_rows<T, 2>(a, rows, s) : dim == 128 ? by_rows<T, 4>(a, rows, s) : by_rows<T, 8>(a, rows, s);
}

}  // namespace

extern "C" {

int sili_kv4_attention_status(void* workspace, void* stream) {
    if (!workspace) return bad("kv4_attention_status", "null workspace");
    unsigned word = 0, *at = (unsigned*)workspace + sili::kErrorWord;
    cudaStream_t s = (cudaStream_t)stream;
    CKV(cudaMemcpyAsync(&word, at, sizeof word, cudaMemcpyDeviceToHost, s));
    CKV(cudaStreamSynchronize(s));
    if (!word) return SILI_OK;
    CKV(cudaMemsetAsync(at, 0, sizeof word, s));
    return sili::set_error(SILI_ETIMEOUT, "kv4_attention: a device-side wait gave up; the rows it served are NaN");
}

int sili_kv4_attention_workspace(int64_t* bytes) {
    if (!bytes) return bad("kv4_attention_workspace", "null array");
    *bytes = workspace_bytes();
    return SILI_OK;
}

int sili_kv4_attention_long_prompt(int dtype, int dim, int64_t tokens, int heads, int kv_heads, int most_new, int* yes) {
    const char* who = "kv4_attention_long_prompt";
    if (!yes) return bad(who, "null array");
    if (tokens < 0 || tokens > 0x7fffffffLL || heads < 1 || kv_heads < 1 || heads % kv_heads || most_new < 0)
        return bad(who, "sizes out of range");
    *yes = sili::kv4_prompt_takes(dtype, dim, tokens, heads, kv_heads, most_new);
    return SILI_OK;
}

int sili_kv4_attention(int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens, int heads,
                       int dim, const uint8_t* codes, const uint8_t* scales, int64_t n_pages, int page, int kv_heads,
                       const int* table, int64_t table_stride, int width, const int* lens, int requests,
                       const int* starts, int most_new, float scale, int window, void* out, float* lse, void* workspace,
                       void* stream) {
    const char* who = "kv4_attention";
    if (dtype < SILI_F32 || dtype > SILI_BF16) return bad(who, "unknown element type");
    if (dim != 64 && dim != 128 && dim != 256) return bad(who, "head dimension must be 64, 128 or 256");
    if (page < 16 || page % 16) return bad(who, "page size must be a multiple of 16");
    if (tokens < 0 || tokens > 0x7fffffffLL || heads < 1 || kv_heads < 1 || n_pages < 0 || width < 0 || requests < 0 || window < 0 || most_new < 0)
        return bad(who, "sizes out of range");
    if ((int64_t)kv_heads * page * dim > 0x7fffffffLL || n_pages > 0x7fffffffLL) return bad(who, "sizes out of range");
    if (tokens * heads > 0x7fffff00LL) return bad(who, "sizes out of range");
    if (heads % kv_heads) return bad(who, "the kv heads must divide the query heads");
    if (tokens == 0) return SILI_OK;
    if (!q || !out || !workspace || (requests && !lens) || (requests && width && !table) || (n_pages && (!codes || !scales)))
        return bad(who, "null array");
    if (requests && table_stride < width) return bad(who, "table rows overlap");
    if ((uintptr_t)codes % 16 || (uintptr_t)scales % 16) return bad(who, "codes and scales must be 16-byte aligned");
    const int64_t item = dtype == SILI_F32 ? 4 : 2;
    // (the stride of a single token or head is never used, and may be anything)
    if ((uintptr_t)q % 8 || (tokens > 1 && q_token_stride * item % 8) || (heads > 1 && q_head_stride * item % 8))
        return bad(who, "q rows must be 8-byte aligned");
    if ((uintptr_t)out % 16) return bad(who, "out must be 16-byte aligned");
    AttendArgs a{q, q_token_stride, q_head_stride, tokens, heads, kv_heads, codes, scales, n_pages, page, table,
                 table_stride, width, lens, requests, starts, scale, window, out, lse, workspace,
                 (uint32_t)page / 16, page == 16 ? 0u : (uint32_t)((0x100000000ull + page / 16 - 1) / (page / 16)),
                 (uint32_t)(kv_heads * page)};
    cudaStream_t s = (cudaStream_t)stream;
    if (starts && sili::kv4_prompt_takes(dtype, dim, tokens, heads, kv_heads, most_new))
        return sili::kv4_prompt_launch(dtype, dim, a, s);
    const int64_t rows = (int64_t)std::max(most_new, 1) * (heads / kv_heads);
    return dtype == SILI_F32 ? by_dim<float>(a, dim, rows, s)
         : dtype == SILI_F16 ? by_dim<__half>(a, dim, rows, s) : by_dim<__nv_bfloat16>(a, dim, rows, s);
}

}  // extern "C"
