// What stands between a model's logits and its next tokens: penalties for
// repeated tokens, biases, the temperature and a grammar's mask, written back
// (sili_adjust_logits) or followed by the pick of the largest
// (sili_pick_tokens, which writes no logits).
//
// With x a row's logit of token v, in fp32, each operation rounded:
//   seen(v)  in the request's history or on the row's path: x > 0 ? x / rep : x * rep
//   c(v) > 0 times in the history behind the prompt and on the path: - freq * c, - pres
//   + bias(v);  / temp where temp > 0;  -inf where the mask's bit is not set.
//
// k_touch counts, for each request, the tokens of its history and bias list in
// shared memory, a tile of the vocabulary at a time, and leaves a bit a token
// and a list of those that it touched.  k_stream takes a tile of a row: one
// pass in 16-byte accesses divides and masks what is neither touched nor on
// the row's path (adjusting), or looks for the largest of it before the
// division, which keeps the order (picking); then come the touched tokens, one
// by one, from the list.  k_pick finds a row's largest and its first place: a
// part of the row is read again, since the division may have made neighbours
// equal.  So the logits' bytes are what should bound a large call.  With the
// counts in the streaming CTAs, 32 trees of 32 over 131072 tokens took 252 us
// (a vocabulary's most frequent tokens lie close together, and their CTAs were
// the last by far); with the touched tokens in a launch of their own, which
// fetches them once more, 140.  Now 120: the pass 97, 4.2 TB/s, with the chain
// of loads before a row's (its request, bits, rules, list) and 20 instructions
// an element and warp, a quarter of them the most frequent tokens' rules; without history, drafts and mask it takes 65.  444 rows of
// 131072 adjusted in bf16: 78 us.  A decode step takes what its host side and
// its launches take, 24 us for 16 rows of 32000 adjusted; as one launch without
// scratch space, which took 324 us in place of those 78, it was 18.
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "common.cuh"
#include "kernels.cuh"
#include "kv4.cuh"
#include "sili_b200.h"

namespace sili {
int set_error(int code, const std::string& msg);
}

namespace {

#define CKL(x)                                                                                          \
    do {                                                                                                \
        const cudaError_t e_ = (x);                                                                     \
        if (e_ != cudaSuccess) return sili::set_error(SILI_ECUDA, std::string(#x) + ": " + cudaGetErrorString(e_)); \
    } while (0)

int bad(const char* who, const char* what) {
    return sili::set_error(SILI_EINVAL, std::string(who) + ": " + what);
}

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 8192;                    // tokens that a CTA of k_touch counts
constexpr int kMostDrafts = 256;
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3FFFFFFFu;
constexpr int kMostListed = 1 << 29;    // tokens of a history, or biases: with the path's, their number stays within kCount
// 16-byte accesses of a thread of k_stream, whose CTAs take a tile of a row each
template <typename T> constexpr int kPacksOf = kTile / kThreads * (int)sizeof(T) / 16;

struct LogitArgs {
    const void* x;
    int64_t x_stride;
    void* y;                   // null: pick only
    int64_t y_stride;
    int64_t rows;
    int vocab, requests;
    const int* starts;         // null: row r is request r's
    const int* history;        // [requests, width] or null
    int64_t history_stride;
    int history_width;
    const int* history_lens;
    const int* prompt_lens;    // null: none of it is a prompt's
    const int* drafted;        // [rows] or null
    const int64_t* masks;      // [rows, words]
    int words;
    const float* repetition;   // [requests] each, or null
    const float* presence;
    const float* frequency;
    const float* temperature;
    const int* bias_tokens;    // [requests, biases]
    const float* bias_values;
    int biases;
    const uint32_t* allowed;   // [rows, allowed_stride] or null
    int64_t allowed_stride;
    int* token;                // [rows]
    // scratch
    int4* row_of;              // [rows]: the row's request, or -1, and its first row and the one past its last; null: the row itself
    uint32_t* touched;         // [requests, touched_stride]: a bit a token; null: nothing is
    int64_t touched_stride;
    int2* listed;              // [requests, tiles]: where a tile's touched tokens lie in the list, and their number
    uint2* list;               // [requests, cap]: token, count and marks
    float* list_bias;          // [requests, cap]
    int64_t cap;
    int tiles;
    uint4* parts;              // picking: [rows, chunks, warps]: the order (below) of a warp's largest element that is not
                               // touched; of its largest touched one, after the rules, and that one's token, inverted
};

// x: the request, or -1; y, z: its rows
__device__ __forceinline__ int4 request_of(const LogitArgs& a, int64_t row) {
    return a.row_of ? a.row_of[row] : make_int4(row < a.requests ? (int)row : -1, (int)row, (int)row + 1, 0);
}

// top = x where bit e of `take` is set and x is larger, or not a number
__device__ __forceinline__ void raise(float& top, float x, uint32_t take, int e) {
    asm("{\n\t.reg .pred p;\n\t.reg .b32 t;\n\tand.b32 t, %2, %3;\n\tsetp.ne.u32 p, t, 0;\n\t@p max.NaN.f32 %0, %0, %1;\n\t}"
        : "+f"(top) : "f"(x), "r"(take), "r"(1u << e));
}
// A number's place in the order (NaN above all, -0 as 0), 0 for -inf; and back.
__device__ __forceinline__ uint32_t order_of(float y) {
    const uint32_t u = __float_as_uint(y + 0.f);
    return u == 0xFF800000u ? 0u : y != y ? 0xFFFFFFFFu : (int)u < 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_order(uint32_t u) {
    return u == 0 ? -INFINITY : u == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u)
                  : __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

// Division by one number, many times: with r the rounded reciprocal of t, a quotient within a unit of x / t becomes the
// rounded one by q + r (x - t q) in two fused steps (Markstein, 1990), where nothing on the way leaves the normal range.
struct Divisor {
    float t, r;
    bool on, fast;
    __device__ __forceinline__ void set(float temp) {
        t = temp;
        on = temp > 0.f && temp != 1.f;
        fast = temp >= 0x1p-20f && temp <= 0x1p20f;
        r = fast ? __frcp_rn(temp) : 0.f;
    }
    __device__ __forceinline__ bool takes(float x) const {     // 2^-60 <= |x| < 2^100
        return fast && ((__float_as_uint(x) << 1) - (67u << 24)) < (160u << 24);
    }
    __device__ __forceinline__ float quick(float x) const {
        float q = x * r;
        q = fmaf(fmaf(-t, q, x), r, q);
        return fmaf(fmaf(-t, q, x), r, q);
    }
    __device__ __forceinline__ float over(float x) const { return takes(x) ? quick(x) : x / t; }
    __device__ __forceinline__ float operator()(float x) const { return on ? over(x) : x; }
};

// ── the tokens that a request touches ───────────────────────────────────────
// CTAs past the requests' tiles look up the rows' requests.
__global__ void __launch_bounds__(kThreads) k_touch(const __grid_constant__ LogitArgs a) {
    const int64_t tiles = a.touched ? (int64_t)a.requests * a.tiles : 0;
    if ((int64_t)blockIdx.x >= tiles) {
        const int64_t step = (int64_t)(gridDim.x - tiles) * kThreads;
        for (int64_t row = (int64_t)(blockIdx.x - tiles) * kThreads + threadIdx.x; row < a.rows; row += step) {
            int lo = 0, hi = a.requests;       // the last request with starts[r] <= row
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.starts[mid] <= row) lo = mid; else hi = mid;
            }
            const int s0 = a.requests ? a.starts[lo] : 0, s1 = a.requests ? a.starts[lo + 1] : 0;
            a.row_of[row] = make_int4(s0 <= row && row < s1 ? lo : -1, max(s0, 0), (int)min((int64_t)s1, a.rows), 0);
        }
        return;
    }
    __shared__ uint32_t cnt[kTile];
    __shared__ int s_sum[kWarps], s_below[kWarps], s_twice;
    __shared__ uint32_t s_word[kThreads];
    __shared__ int s_before[kThreads];
    const int r = blockIdx.x / a.tiles, tile = blockIdx.x - r * a.tiles, t0 = tile * kTile, n = min(kTile, a.vocab - t0);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int len = a.history ? min(max(a.history_lens[r], 0), a.history_width) : 0;
    const int prompt = a.history && a.prompt_lens ? a.prompt_lens[r] : 0;
    for (int i = threadIdx.x; i < kTile / 4; i += kThreads) ((uint4*)cnt)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) s_twice = 0;
    __syncthreads();
    // a tile's part of the list begins behind as many places as the history and the biases have tokens before the tile
    int below = 0;
    const int* h = a.history + r * a.history_stride;
    for (int j0 = threadIdx.x; j0 < len; j0 += 8 * kThreads) {
        int v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = j0 + k * kThreads < len ? __ldg(h + j0 + k * kThreads) : -1;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t i = (uint32_t)v[k] - (uint32_t)t0;
            below += v[k] >= 0 && v[k] < t0;
            if (v[k] < 0 || i >= (uint32_t)n) continue;
            if (j0 + k * kThreads < prompt) atomicOr(cnt + i, kSeen); else atomicAdd(cnt + i, 1u);
        }
    }
    if (a.biases) {
        const int* list = a.bias_tokens + (int64_t)r * a.biases;
        for (int j = threadIdx.x; j < a.biases; j += kThreads) {
            const int v = list[j];
            const uint32_t i = (uint32_t)v - (uint32_t)t0;
            below += v >= 0 && v < t0;
            if (i >= (uint32_t)n) continue;
            if (atomicOr(cnt + i, kBiased) & kBiased) s_twice = 1;
        }
    }
    __syncthreads();
    // a word of 32 tokens a thread and turn: a warp's ballots, token by token
    static_assert(kTile == 32 * kThreads, "a word a thread");
    uint32_t word = 0;
    for (int k = 0; k < 32; ++k) {
        const uint32_t bits = __ballot_sync(0xffffffffu, cnt[(warp * 32 + k) * 32 + lane] != 0);
        if (lane == k) word = bits;
    }
    if ((int)threadIdx.x * 32 < n) a.touched[r * a.touched_stride + t0 / 32 + threadIdx.x] = word;
    const uint32_t kept = word;
    int mine = __popc(word), before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += t;
    }
    if (lane == 31) s_sum[warp] = before;
    below = sili::warp_sum(below);
    if (lane == 0) s_below[warp] = below;
    __syncthreads();
    int all = 0;
    below = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s_sum[w];
        all += s_sum[w];
        below += s_below[w];
    }
    if (threadIdx.x == 0) a.listed[r * a.tiles + tile] = make_int2(below, all);
    const int64_t at = r * a.cap + below;
    int e = before - mine;
    for (; word; word &= word - 1, ++e) {
        const int i = (int)threadIdx.x * 32 + __ffs(word) - 1;
        a.list[at + e] = make_uint2(t0 + i, cnt[i]);
    }
    if (!a.biases) return;
    s_word[threadIdx.x] = kept;
    s_before[threadIdx.x] = before - mine;
    __syncthreads();
    const int* list = a.bias_tokens + (int64_t)r * a.biases;
    const float* value = a.bias_values + (int64_t)r * a.biases;
    for (int j = threadIdx.x; j < a.biases; j += kThreads) {
        const int v = list[j];
        const uint32_t i = (uint32_t)v - (uint32_t)t0;
        if (i >= (uint32_t)n) continue;
        float sum = value[j];
        if (s_twice) {
            // a token that is listed again: its first place adds all of them up, in order
            bool first = true;
            for (int k = 0; k < j; ++k) first = first && list[k] != v;
            if (!first) continue;
            for (int k = j + 1; k < a.biases; ++k)
                if (list[k] == v) sum += value[k];
        }
        // its place in the list: the touched tokens before it
        a.list_bias[at + s_before[i >> 5] + __popc(s_word[i >> 5] & ((1u << (i & 31)) - 1u))] = sum;
    }
}

// What is certainly smaller than `top`, and stays so after the division (where a quotient leaves the normal range, any two
// may become the same).
__device__ __forceinline__ float surely_below(const Divisor& by, float top) {
    return by.on && !by.takes(top) ? -INFINITY : top - fabsf(top) * 0x1p-20f;
}

// A row's rules.
struct Rules {
    float freq, pres;
    Divisor rep, by;
    __device__ __forceinline__ Rules(const LogitArgs& a, int r) {
        rep.set(a.repetition ? a.repetition[r] : 1.f);
        freq = a.frequency ? a.frequency[r] : 0.f;
        pres = a.presence ? a.presence[r] : 0.f;
        by.set(a.temperature ? a.temperature[r] : 0.f);
    }
    __device__ __forceinline__ float operator()(float x, uint32_t what, float bias) const {
        // (a count also makes it seen)
        if (what & (kSeen | kCount)) x = x > 0.f ? rep.over(x) : x * rep.t;
        if (what & kCount) {
            x = x - freq * (float)(what & kCount);
            x = x - pres;
        }
        if (what & kBiased) x = x + bias;
        return by(x);
    }
};

// The draft that thread j stands for: its token where the row's path holds it, else -1.
__device__ __forceinline__ int path_token(const LogitArgs& a, const int4& of, int j, uint64_t mask) {
    return (mask >> (j & 63) & 1) && of.y + j < of.z ? a.drafted[of.y + j] : -1;
}
__device__ __forceinline__ uint64_t path_mask(const LogitArgs& a, int64_t row, int j) {
    return a.drafted && j < 64 * a.words ? (uint64_t)a.masks[row * a.words + (j >> 6)] : 0;
}

// element e of a pack, from memory's order of bytes
template <typename T>
__device__ __forceinline__ float element(const sili::Pack<T, 16 / sizeof(T)>& in, int e) {
    const uint4 w = *(const uint4*)&in;
    const int at = e * (int)sizeof(T) / 4;
    const uint32_t u = at == 0 ? w.x : at == 1 ? w.y : at == 2 ? w.z : w.w;
    if (sizeof(T) == 4) return __uint_as_float(u);
    const unsigned short h = (unsigned short)(e & 1 ? u >> 16 : u);
    return sili::to_f32(*(const T*)&h);
}

// Where the 16-byte accesses of a chunk of a row lie: whole ones from the first aligned element on.
template <typename T>
struct Lay {
    static constexpr int kVec = 16 / (int)sizeof(T);
    int t0, n, head, packs;
    __device__ __forceinline__ Lay(const LogitArgs& a, const T* row, int chunk) {
        t0 = chunk * kTile;
        n = min(kTile, a.vocab - t0);
        head = min((int)((16 - (uintptr_t)(row + t0) % 16) % 16 / sizeof(T)), n);
        packs = (n - head) / kVec;
    }
};

// ── the pass over the logits ────────────────────────────────────────────────
// A CTA takes a chunk of one row.  Touched tokens and the row's path are left as they are (adjusting), or aside (picking).
template <typename T, bool WRITE>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 4 : 5) k_stream(const __grid_constant__ LogitArgs a) {
    constexpr int kVec = 16 / (int)sizeof(T), kPacks = kPacksOf<T>, kStep = kThreads * kVec / 32;
    static_assert(kThreads * kVec % 32 == 0, "whole words");
    using P = sili::Pack<T, kVec>;
    constexpr int kWords = kTile / 32;
    // bits of the tile's tokens: those that are allowed; adjusting, those to leave, and picking, those to take
    __shared__ uint32_t s_allow[kWords + 1], s_rest[kWords + 1], s_path[kWords];
    __shared__ int s_tok[kMostDrafts], s_n;        // the path's tokens that lie in the tile
    const int64_t row = blockIdx.x / a.tiles;
    const int chunk = blockIdx.x - (int)row * a.tiles, tid = threadIdx.x;
    const T* x = (const T*)a.x + row * a.x_stride;
    T* y = WRITE ? (T*)a.y + row * a.y_stride : nullptr;
    Lay<T> lay(a, x, chunk);
    if (WRITE && ((uintptr_t)y - (uintptr_t)x) % 16) { lay.head = lay.n; lay.packs = 0; }
    const int t0 = lay.t0, n = lay.n, head = lay.head, packs = lay.packs;
    x += t0;
    y += t0;
    const int first = head + tid * kVec;
    P in[kPacks];
#pragma unroll
    for (int k = 0; k < kPacks; ++k)
        if (tid + k * kThreads < packs) in[k] = *(const P*)(x + first + k * kThreads * kVec);
    const int4 of = request_of(a, row);
    const uint64_t mask = path_mask(a, row, tid);
    const int r = of.x;
    if (r < 0) {
        // of no request: as it is
        if (WRITE && (const void*)x != (void*)y)
            for (int i = tid; i < n; i += kThreads) y[i] = x[i];
        return;
    }
    const uint32_t* allow = a.allowed ? a.allowed + row * a.allowed_stride + (t0 >> 5) : nullptr;
    const uint32_t* touched = a.touched ? a.touched + r * a.touched_stride + (t0 >> 5) : nullptr;
    const bool bits = a.allowed || a.touched || a.drafted;
    const int2 listed = touched ? a.listed[r * a.tiles + chunk] : make_int2(0, 0);
    const Rules rule(a, r);
    const Divisor& by = rule.by;
    bool path = false;
    if (bits) {
        uint32_t i = 0xFFFFFFFFu;
        if (a.drafted) {
            const int v = path_token(a, of, tid, mask);
            if (v >= 0) i = (uint32_t)v - (uint32_t)t0;
        }
        uint32_t word[2][kWords / kThreads];
#pragma unroll
        for (int k = 0; k < kWords / kThreads; ++k) {
            const int w = tid + k * kThreads;
            word[0][k] = allow && w * 32 < n ? __ldg(allow + w) : 0xFFFFFFFFu;
            word[1][k] = touched && w * 32 < n ? touched[w] : 0u;
        }
#pragma unroll
        for (int k = 0; k < kWords / kThreads; ++k) {
            const int w = tid + k * kThreads;
            s_allow[w] = word[0][k];
            s_rest[w] = WRITE ? word[1][k] : word[0][k] & ~word[1][k];
        }
        path = __syncthreads_or(i < (uint32_t)n);
        if (path) {
            for (int w = tid; w < kWords; w += kThreads) s_path[w] = 0;
            if (tid == 0) s_n = 0;
            __syncthreads();
            if (i < (uint32_t)n) {
                atomicOr(s_path + (i >> 5), 1u << (i & 31));
                s_tok[atomicAdd(&s_n, 1)] = (int)i;
                if (WRITE) atomicOr(s_rest + (i >> 5), 1u << (i & 31)); else atomicAnd(s_rest + (i >> 5), ~(1u << (i & 31)));
            }
            __syncthreads();
        }
    }
    // this thread's first touched token, on its way during the pass
    const int64_t list_at = r * a.cap + listed.x;
    uint2 next = make_uint2((uint32_t)t0, 0);
    float next_bias = 0.f;
    if (tid < listed.y) {
        next = a.list[list_at + tid];
        if (a.biases) next_bias = a.list_bias[list_at + tid];
    }
    // a pack's bits lie in one word or two, whose places move by a constant from pack to pack
    const int shift = first & 31, at0 = first >> 5, more = ((first + kVec - 1) >> 5) - at0;
    auto bits_of = [&](const uint32_t* words, int k) {
        return __funnelshift_r(words[at0 + k * kStep], words[at0 + k * kStep + more], shift);
    };
    float most = -INFINITY;
    // elements before and behind the whole accesses
    for (int i = tid; i < n - packs * kVec; i += kThreads) {
        const int j = i < head ? i : i + packs * kVec, w = j >> 5;
        if (WRITE) {
            const bool left = bits && (s_rest[w] >> (j & 31) & 1), may = !bits || (s_allow[w] >> (j & 31) & 1);
            y[j] = left ? x[j] : sili::from_f32<T>(may ? by(sili::to_f32(x[j])) : -INFINITY);
        } else raise(most, sili::to_f32(x[j]), bits ? s_rest[w] >> (j & 31) : 1u, 0);
    }
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
        if (tid + k * kThreads >= packs) break;
        const uint32_t take = bits ? bits_of(WRITE ? s_allow : s_rest, k) : 0xFFFFFFFFu;
        if (WRITE) {
            const uint32_t rest = bits ? bits_of(s_rest, k) : 0u;
            P out;
            float v[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) v[e] = sili::to_f32(in[k].v[e]);
            if (by.on) {
                bool quick = by.fast;
#pragma unroll
                for (int e = 0; e < kVec; ++e) quick = quick && by.takes(v[e]);
                if (quick)
#pragma unroll
                    for (int e = 0; e < kVec; ++e) v[e] = by.quick(v[e]);
                else
#pragma unroll 1
                    for (int e = 0; e < kVec; ++e) {
                        const float u = element<T>(in[k], e) / by.t;
#pragma unroll
                        for (int f = 0; f < kVec; ++f) v[f] = f == e ? u : v[f];
                    }
            }
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                out.v[e] = sili::from_f32<T>(take >> e & 1 ? v[e] : -INFINITY);
                if (rest >> e & 1) out.v[e] = in[k].v[e];
            }
            *(P*)(y + first + k * kThreads * kVec) = out;
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) raise(most, sili::to_f32(in[k].v[e]), take, e);
        }
    }
    const uint32_t all = WRITE ? 0u : __reduce_max_sync(0xffffffffu, order_of(most));
    uint32_t high = 0, low = 0;    // picking: the largest touched one and its token, inverted
    if (touched || path) {
        if (WRITE) __syncthreads();        // (what is touched has been written as it was, with what lies beside it)
        // picking, where the penalties raise no logit: one below the warp's largest other stays there
        const bool lowers = !WRITE && rule.rep.t >= 1.f && rule.freq >= 0.f && rule.pres >= 0.f;
        const float near = WRITE ? 0.f : surely_below(by, of_order(all));
        auto times = [&](int i) {          // on the path
            uint32_t c = 0;
            if (path && (s_path[i >> 5] >> (i & 31) & 1))
                for (int k = 0; k < s_n; ++k) c += s_tok[k] == i;
            return c;
        };
        auto one = [&](int i, T raw, uint32_t what, float bias) {
            const float v = sili::to_f32(raw);
            if (!WRITE && lowers && !(what & kBiased) && v < near) return;
            const bool may = s_allow[i >> 5] >> (i & 31) & 1;
            const float z = may ? rule(v, what + times(i), bias) : -INFINITY;
            if (WRITE) y[i] = sili::from_f32<T>(z);
            else {
                const uint32_t u = order_of(z);
                if (u > high) { high = u; low = ~(uint32_t)(t0 + i); }
                else if (u == high) low = max(low, ~(uint32_t)(t0 + i));
            }
        };
        if (tid < listed.y) one((int)next.x - t0, x[(int)next.x - t0], next.y, next_bias);
        constexpr int kBatch = 4;      // in flight: no load is used before all of them have been asked for
        for (int e0 = tid + kThreads; e0 < listed.y; e0 += kBatch * kThreads) {
            uint2 it[kBatch];
            float bias[kBatch];
            T v[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (e0 + b * kThreads < listed.y) {
                    it[b] = a.list[list_at + e0 + b * kThreads];
                    bias[b] = a.biases ? a.list_bias[list_at + e0 + b * kThreads] : 0.f;
                }
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (e0 + b * kThreads < listed.y) v[b] = x[(int)it[b].x - t0];
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (e0 + b * kThreads < listed.y) one((int)it[b].x - t0, v[b], it[b].y, bias[b]);
        }
        // the path's tokens that are on no list, at the first of their places
        if (path && tid < s_n) {
            const int i = s_tok[tid];
            bool is = !touched || !(touched[i >> 5] >> (i & 31) & 1);
            for (int k = 0; k < tid; ++k) is = is && s_tok[k] != i;
            if (is) one(i, x[i], 0u, 0.f);
        }
        if (!WRITE) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, high);
            low = __reduce_max_sync(0xffffffffu, high == top ? low : 0u);
            high = top;
        }
    }
    if (!WRITE && (tid & 31) == 0) a.parts[((int64_t)row * a.tiles + chunk) * kWarps + (tid >> 5)] = make_uint4(all, high, low, 0);
}

// ── the pick ────────────────────────────────────────────────────────────────
// A row a CTA: the largest of its parts, and the first place of it.
constexpr int kPickThreads = 128, kMostHeld = 64;

template <typename T>
__global__ void __launch_bounds__(kPickThreads) k_pick(const __grid_constant__ LogitArgs a) {
    __shared__ uint32_t s_red[2][kPickThreads / 32];
    __shared__ int s_hold[kMostHeld], s_held;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int4 of = request_of(a, row);
    const int r = of.x;
    if (r < 0) {
        if (tid == 0) a.token[row] = -1;
        return;
    }
    if (tid == 0) s_held = 0;
    Divisor by;
    by.set(a.temperature ? a.temperature[r] : 0.f);
    auto reduce = [&](uint32_t u, int which) {
        u = __reduce_max_sync(0xffffffffu, u);
        if (lane == 0) s_red[which][warp] = u;
        __syncthreads();
        uint32_t top = 0;
#pragma unroll
        for (int w = 0; w < kPickThreads / 32; ++w) top = max(top, s_red[which][w]);
        return top;
    };
    const uint4* parts = a.parts + row * a.tiles * kWarps;
    const int n_parts = a.tiles * kWarps;
    uint32_t other = 0, high = 0, low = 0;
    for (int i = tid; i < n_parts; i += kPickThreads) {
        const uint4 p = parts[i];
        other = max(other, p.x);
        if (p.y > high) { high = p.y; low = p.z; }
        else if (p.y == high) low = max(low, p.z);
    }
    other = order_of(by(of_order(other)));
    const uint32_t all = reduce(max(other, high), 0);
    if (high != all) low = 0;
    if (all && __syncthreads_or(other == all)) {
        // the parts that hold it are read again: after the division, elements next to the largest may be as large
        const T* x = (const T*)a.x + row * a.x_stride;
        const uint32_t* allow = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
        const uint32_t* touched = a.touched ? a.touched + r * a.touched_stride : nullptr;
        auto candidate = [&](int v, float value) {
            if (order_of(by(value)) != all || (touched && (touched[v >> 5] >> (v & 31) & 1))) return;
            if (allow && !(__ldg(allow + (v >> 5)) >> (v & 31) & 1)) return;
            if (a.drafted)
                for (int w = 0; w < a.words; ++w)
                    for (uint64_t left = path_mask(a, row, 64 * w); left; left &= left - 1)
                        if (path_token(a, of, 64 * w + __ffsll((long long)left) - 1, left) == v) return;
            low = max(low, ~(uint32_t)v);
        };
        for (int i = tid; i < n_parts; i += kPickThreads)
            if (order_of(by(of_order(parts[i].x))) == all) {
                const int k = atomicAdd(&s_held, 1);
                if (k < kMostHeld) s_hold[k] = i;
            }
        __syncthreads();
        // (more of them than there is room for, as where a row is one value: all parts are looked at)
        const int held = s_held > kMostHeld ? n_parts : s_held;
        using P = sili::Pack<T, 16 / sizeof(T)>;
        constexpr int kVec = 16 / (int)sizeof(T), kPacks = kPacksOf<T>;
        for (int k = 0; k < held; ++k) {
            const int i = s_held > kMostHeld ? k : s_hold[k];
            const float top = of_order(parts[i].x), near = surely_below(by, top);
            if (s_held > kMostHeld && order_of(by(top)) != all) continue;
            // the warp's whole accesses, and the single elements that were its own
            const int chunk = i / kWarps, w = i - chunk * kWarps;
            const Lay<T> lay(a, x, chunk);
#pragma unroll
            for (int b = 0; b < kPacks; b += kPickThreads / 32) {
                const int p = w * 32 + lane + (b + warp) * kThreads, at = lay.t0 + lay.head + p * kVec;
                if (p >= lay.packs) continue;
                const P in = *(const P*)(x + at);
                uint32_t some = 0;
#pragma unroll
                for (int e = 0; e < kVec; ++e) some |= !(sili::to_f32(in.v[e]) < near) ? 1u << e : 0u;
                for (; some; some &= some - 1) candidate(at + __ffs(some) - 1, element<T>(in, __ffs(some) - 1));
            }
            if (warp == 0)
                for (int e = w * 32 + lane; e < lay.n - lay.packs * kVec; e += kThreads) {
                    const int j = lay.t0 + (e < lay.head ? e : e + lay.packs * kVec);
                    candidate(j, sili::to_f32(x[j]));
                }
        }
    }
    low = reduce(low, 1);
    if (tid == 0) a.token[row] = all ? (int)~low : -1;
}

// ── the entries ─────────────────────────────────────────────────────────────
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

// The parts of the scratch space, one after the other from `base` on; returns its bytes.
int64_t lay_out(LogitArgs& a, bool counts, bool pick, uint8_t* base) {
    int64_t at = 0;
    auto part = [&](int64_t bytes) { const int64_t here = at; at += round16(bytes); return base + here; };
    a.tiles = (a.vocab + kTile - 1) / kTile;
    a.cap = (int64_t)a.history_width + a.biases;
    a.touched_stride = (int64_t)a.tiles * (kTile / 32) + 1;
    a.row_of = a.starts ? (int4*)part(a.rows * 16) : nullptr;
    a.touched = nullptr;
    if (counts) {
        a.touched = (uint32_t*)part(a.requests * a.touched_stride * 4);
        a.listed = (int2*)part((int64_t)a.requests * a.tiles * 8);
        a.list = (uint2*)part(a.requests * a.cap * 8);
        a.list_bias = (float*)part(a.biases ? a.requests * a.cap * 4 : 0);
    }
    a.parts = pick ? (uint4*)part(a.rows * a.tiles * kWarps * 16) : nullptr;
    return at;
}

template <typename T, bool WRITE>
int launch(const LogitArgs& a, cudaStream_t s) {
    if (a.row_of || a.touched) {
        const int64_t tiles = a.touched ? (int64_t)a.requests * a.tiles : 0;
        const int64_t finders = a.row_of ? std::min<int64_t>((a.rows + kThreads - 1) / kThreads, 148) : 0;
        k_touch<<<(unsigned)(tiles + finders), kThreads, 0, s>>>(a);
        sili::count_launch();
    }
    k_stream<T, WRITE><<<(unsigned)(a.rows * a.tiles), kThreads, 0, s>>>(a);
    sili::count_launch();
    if (!WRITE) {
        k_pick<T><<<(unsigned)a.rows, kPickThreads, 0, s>>>(a);
        sili::count_launch();
    }
    CKL(cudaGetLastError());
    return SILI_OK;
}
template <bool WRITE>
int by_type(int dtype, const LogitArgs& a, cudaStream_t s) {
    return dtype == SILI_F32 ? launch<float, WRITE>(a, s)
         : dtype == SILI_F16 ? launch<__half, WRITE>(a, s) : launch<__nv_bfloat16, WRITE>(a, s);
}

// Everything but where the result goes.
int prepare(const char* who, int dtype, const void* logits, int64_t stride, int64_t rows, int vocab, int requests,
            const sili_logit_rules* rules, bool pick, void* scratch, LogitArgs& a, int64_t* bytes) {
    if (!rules) return bad(who, "null array");
    const sili_logit_rules& q = *rules;
    if (dtype < SILI_F32 || dtype > SILI_BF16) return bad(who, "unknown element type");
    if (rows < 0 || rows > 0x7fffffffLL || vocab < 1 || requests < 0 || q.history_width < 0 || q.biases < 0 || q.words < 0 ||
        q.words > 4)
        return bad(who, "sizes out of range");
    // (an array of no columns may have no address)
    if (q.history_width && (q.history != nullptr) != (q.history_lens != nullptr))
        return bad(who, "history and its lengths come together");
    if (q.history_width > kMostListed || q.biases > kMostListed) return bad(who, "history or biases too long");
    if (q.history && requests > 1 && q.history_stride < 0) return bad(who, "sizes out of range");
    if ((q.drafted != nullptr) != (q.masks != nullptr) || (q.drafted && (!q.starts || q.words < 1)))
        return bad(who, "drafted tokens, masks and starts come together");
    if (q.biases && requests && (!q.bias_tokens || !q.bias_values)) return bad(who, "null array");
    if (q.allowed && q.allowed_stride < (vocab + 31) / 32 && rows > 1) return bad(who, "mask rows overlap");
    if (!q.starts && requests != rows) return bad(who, "without starts there is one row a request");
    a = LogitArgs{};
    a.x = logits;
    a.x_stride = stride;
    a.rows = rows;
    a.vocab = vocab;
    a.requests = requests;
    a.starts = q.starts;
    a.history = q.history_width ? q.history : nullptr;
    a.history_stride = q.history_stride;
    a.history_width = a.history ? q.history_width : 0;
    a.history_lens = q.history_lens;
    a.prompt_lens = q.prompt_lens;
    a.drafted = q.drafted;
    a.masks = q.masks;
    a.words = q.words;
    a.repetition = q.repetition;
    a.presence = q.presence;
    a.frequency = q.frequency;
    a.temperature = q.temperature;
    a.bias_tokens = q.bias_tokens;
    a.bias_values = q.bias_values;
    a.biases = q.biases;
    a.allowed = q.allowed;
    a.allowed_stride = q.allowed_stride;
    const int64_t need = lay_out(a, (a.history || a.biases) && requests, pick, (uint8_t*)scratch);
    if (rows * a.tiles > 0x7fffffffLL || (int64_t)requests * a.tiles > 0x7fff0000LL) return bad(who, "sizes out of range");
    if (bytes) { *bytes = need; return SILI_OK; }
    if (rows == 0) return SILI_OK;
    if (!logits || (need && !scratch)) return bad(who, "null array");
    if (rows > 1 && stride < vocab) return bad(who, "rows overlap");
    if ((uintptr_t)logits % (dtype == SILI_F32 ? 4 : 2)) return bad(who, "logits must be aligned to their type");
    if ((uintptr_t)scratch % 16) return bad(who, "scratch must be 16-byte aligned");
    return SILI_OK;
}

}  // namespace

extern "C" {

int sili_logits_scratch(int dtype, int64_t rows, int vocab, int requests, const sili_logit_rules* rules, int pick,
                        int64_t* bytes) {
    if (!bytes) return bad("logits_scratch", "null array");
    LogitArgs a;
    return prepare("logits_scratch", dtype, nullptr, vocab, rows, vocab, requests, rules, pick != 0, nullptr, a, bytes);
}

int sili_adjust_logits(int dtype, const void* logits, int64_t stride, int64_t rows, int vocab, int requests,
                       const sili_logit_rules* rules, void* out, int64_t out_stride, void* scratch, void* stream) {
    const char* who = "adjust_logits";
    LogitArgs a;
    if (const int e = prepare(who, dtype, logits, stride, rows, vocab, requests, rules, false, scratch, a, nullptr)) return e;
    if (rows == 0) return SILI_OK;
    if (!out) return bad(who, "null array");
    if (rows > 1 && out_stride < vocab) return bad(who, "rows overlap");
    if ((uintptr_t)out % (dtype == SILI_F32 ? 4 : 2)) return bad(who, "out must be aligned to its type");
    a.y = out;
    a.y_stride = out_stride;
    return by_type<true>(dtype, a, (cudaStream_t)stream);
}

int sili_pick_tokens(int dtype, const void* logits, int64_t stride, int64_t rows, int vocab, int requests,
                     const sili_logit_rules* rules, int* token, void* scratch, void* stream) {
    const char* who = "pick_tokens";
    LogitArgs a;
    if (const int e = prepare(who, dtype, logits, stride, rows, vocab, requests, rules, true, scratch, a, nullptr)) return e;
    if (rows == 0) return SILI_OK;
    if (!token) return bad(who, "null array");
    a.token = token;
    return by_type<false>(dtype, a, (cudaStream_t)stream);
}

}  // extern "C"
