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
// A CTA takes a tile of the vocabulary and a few consecutive rows.  The
// tokens of a request's history that lie in the tile are counted in shared
// memory, once for the rows that share it; a row's path (the drafted tokens
// that its mask names) is counted on top and taken off again, where any of it
// lies in the tile.  The tokens so touched are also listed, each once: they
// are taken one by one, and the rest of a row is one pass over registers that
// only divides by the temperature and masks.  A pick compares the rest before
// the division, which keeps the order; what it may make equal is told apart
// for the few elements next to the largest.
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "common.cuh"
#include "kernels.cuh"
#include "kv4_attention.cuh"
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
constexpr int kEach = 16;                      // elements of a row that a thread holds in registers
constexpr int kTile = kThreads * kEach;        // tokens of a tile
constexpr int kGroup = 8;                      // rows of a CTA at most
static_assert(kGroup <= kThreads / 32, "a warp a row picks");
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3FFFFFFFu;

struct LogitArgs {
    const void* x;
    int64_t x_stride;
    void* y;                   // null: pick only
    int64_t y_stride;
    int64_t rows;
    int vocab, requests;
    const int* starts;         // null: row r is request r's
    const int* history;        // [requests, width]
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
    unsigned long long* best;  // [rows, tiles]: a tile's largest
    int* token;                // [rows]
    int tiles, group;          // tiles, rows of a CTA
};

// A larger value, then a lower token, has the larger key; NaN is above all numbers (the first one is picked) and -inf below
// every key (0).
__device__ __forceinline__ unsigned long long key_of(float y, int token) {
    uint32_t u = __float_as_uint(y + 0.f);     // -0 as 0
    if (u == 0xFF800000u) return 0;
    u = y != y ? 0xFFFFFFFFu : (int)u < 0 ? ~u : u | 0x80000000u;
    return (unsigned long long)u << 32 | (0xFFFFFFFFu - (uint32_t)token);
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
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

struct Shared {
    uint32_t cnt[kTile];                       // a token's count and marks
    uint32_t touched[kTile / 32 + 1];          // a bit a token whose count is not 0
    uint16_t list[kTile];                      // those tokens
    uint16_t draft[256];                       // the request's drafted tokens, 0xFFFF: not in the tile
    unsigned long long masks[kGroup][4];
    unsigned long long key[kGroup][kThreads / 32];     // picking: a warp's largest key of touched and single elements,
    uint32_t y[kGroup][kThreads / 32];                 // and the upper half of that of the others
    int listed, has_path[kGroup], twice;
    float value[1];                            // [kTile] biases, then (writing) [kTile] the listed tokens' results
};

template <typename T, bool WRITE>
struct Logits {
    static constexpr int kVec = 16 / sizeof(T), kPacks = kEach / kVec;
    using P = sili::Pack<T, kVec>;
    const LogitArgs& a;
    Shared& s;
    float *bias, *result;
    int t0, n;            // the tile's first token, its tokens
    const uint32_t* allow;
    float freq, pres;
    Divisor rep, by;

    __device__ __forceinline__ uint32_t note(uint32_t i, uint32_t what) const {
        const uint32_t was = what & kCount ? atomicAdd(s.cnt + i, what) : atomicOr(s.cnt + i, what);
        const uint32_t bit = 1u << (i & 31);
        if (!was && !(atomicOr(s.touched + (i >> 5), bit) & bit)) s.list[atomicAdd(&s.listed, 1)] = (uint16_t)i;
        return was;
    }
    // the tokens of the request's history and bias list that lie in the tile, and which of rows [row, last) have a path there
    __device__ void count_request(int r, int64_t row, int64_t last, int64_t row0, int64_t row1) {
        for (int i = threadIdx.x; i < kTile; i += kThreads) s.cnt[i] = 0;
        for (int i = threadIdx.x; i <= kTile / 32; i += kThreads) s.touched[i] = 0;
        if (threadIdx.x == 0) s.listed = s.twice = 0;
        if (a.drafted) {
            const uint32_t v = row0 + threadIdx.x < row1 && (int)threadIdx.x < 64 * a.words
                                   ? (uint32_t)a.drafted[row0 + threadIdx.x] - (uint32_t)t0 : 0xFFFFFFFFu;
            s.draft[threadIdx.x] = v < (uint32_t)n ? (uint16_t)v : (uint16_t)0xFFFFu;
            const int64_t k = row + threadIdx.x / 4;
            const int w = threadIdx.x & 3;
            if (threadIdx.x < 4 * kGroup) {
                s.masks[threadIdx.x / 4][w] = k < last && w < a.words ? (unsigned long long)a.masks[k * a.words + w] : 0;
                s.has_path[threadIdx.x / 4] = 0;
            }
        }
        __syncthreads();
        if (a.drafted && s.draft[threadIdx.x] != 0xFFFFu)
#pragma unroll
            for (int k = 0; k < kGroup; ++k)
                if (s.masks[k][threadIdx.x >> 6] >> (threadIdx.x & 63) & 1) s.has_path[k] = 1;
        if (a.history) {
            const int* h = a.history + r * a.history_stride;
            const int len = min(max(a.history_lens[r], 0), a.history_width);
            const int prompt = a.prompt_lens ? a.prompt_lens[r] : 0;
#pragma unroll 4
            for (int j = threadIdx.x; j < len; j += kThreads) {
                const uint32_t i = (uint32_t)__ldg(h + j) - (uint32_t)t0;
                if (i < (uint32_t)n) note(i, j < prompt ? kSeen : 1u);
            }
        }
        if (a.biases) {
            const int* list = a.bias_tokens + (int64_t)r * a.biases;
            const float* value = a.bias_values + (int64_t)r * a.biases;
            for (int j = threadIdx.x; j < a.biases; j += kThreads) {
                const uint32_t i = (uint32_t)list[j] - (uint32_t)t0;
                if (i >= (uint32_t)n) continue;
                bias[i] = value[j];
                if (note(i, kBiased) & kBiased) s.twice = 1;
            }
            __syncthreads();
            if (s.twice)
                // a token is listed again: its first place adds all of them up, in order
                for (int j = threadIdx.x; j < a.biases; j += kThreads) {
                    const int v = list[j];
                    const uint32_t i = (uint32_t)v - (uint32_t)t0;
                    if (i >= (uint32_t)n) continue;
                    bool first = true;
                    for (int k = 0; k < j; ++k) first = first && list[k] != v;
                    if (!first) continue;
                    float sum = value[j];
                    for (int k = j + 1; k < a.biases; ++k)
                        if (list[k] == v) sum += value[k];
                    bias[i] = sum;
                }
        }
        __syncthreads();
    }
    // the path of the CTA's row k on top of the counts, or off them again (the list is then cut to what it was)
    __device__ void count_path(int k, bool off, int listed) const {
        const uint32_t i = s.draft[threadIdx.x];
        if (i != 0xFFFFu && (s.masks[k][threadIdx.x >> 6] >> (threadIdx.x & 63) & 1)) {
            if (!off) note(i, 1u);
            else if (atomicSub(s.cnt + i, 1u) == 1u) atomicAnd(s.touched + (i >> 5), ~(1u << (i & 31)));
        }
        if (off && threadIdx.x == 0) s.listed = listed;
        __syncthreads();
    }

    __device__ __forceinline__ float ruled(float x, uint32_t what, int i) const {
        // (a count also makes it seen)
        if (what & (kSeen | kCount)) x = x > 0.f ? rep.over(x) : x * rep.t;
        if (what & kCount) {
            x = x - freq * (float)(what & kCount);
            x = x - pres;
        }
        if (what & kBiased) x = x + bias[i];
        return by(x);
    }
    __device__ __forceinline__ bool may(int i) const {
        const int v = t0 + i;
        return !allow || (__ldg(allow + (v >> 5)) >> (v & 31) & 1);
    }
    __device__ __forceinline__ float single(T x, int i) const {
        return may(i) ? ruled(sili::to_f32(x), s.cnt[i], i) : -INFINITY;
    }

    // one row of the tile, the CTA's row k of the request
    __device__ void row(const T* x, T* y, int at) const {
        unsigned long long top = 0;
        // whole 16 bytes from the first aligned element on
        const int lead = (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T));
        const int head = !WRITE || (uintptr_t)y % 16 == (uintptr_t)x % 16 ? min(lead, n) : n;
        const int packs = (n - head) / kVec, tail = head + packs * kVec;
        P in[kPacks];
        uint32_t words[kPacks][2];
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            const int p = threadIdx.x + k * kThreads;
            words[k][0] = words[k][1] = 0xFFFFFFFFu;
            if (p < packs) {
                in[k] = *(const P*)(x + head + p * kVec);
                if (allow) {
                    const int v = t0 + head + p * kVec;
                    words[k][0] = __ldg(allow + (v >> 5));
                    words[k][1] = __ldg(allow + ((v + kVec - 1) >> 5));
                }
            }
        }
        const int listed = s.listed;
        for (int e = threadIdx.x; e < listed; e += kThreads) {
            const int i = s.list[e];
            const float v = single(x[i], i);
            if (WRITE) result[e] = v; else top = max(top, key_of(v, t0 + i));
        }
        if (WRITE && listed) __syncthreads();     // (y may be x)
        for (int i = threadIdx.x; i < n - packs * kVec; i += kThreads) {
            const int j = i < head ? i : i - head + tail;
            const float v = single(x[j], j);
            if (WRITE) y[j] = sili::from_f32<T>(v); else top = max(top, key_of(v, t0 + j));
        }
        float most = -INFINITY;
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            const int p = threadIdx.x + k * kThreads;
            if (p >= packs) break;
            const int i = head + p * kVec;
            uint32_t take = __funnelshift_r(words[k][0], words[k][1], (t0 + i) & 31);
            if (WRITE) {
                P out;
                bool quick = by.fast;
                float v[kVec];
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    v[e] = sili::to_f32(in[k].v[e]);
                    quick = quick && by.takes(v[e]);
                }
                if (by.on) {
                    if (quick)
#pragma unroll
                        for (int e = 0; e < kVec; ++e) v[e] = by.quick(v[e]);
                    else
#pragma unroll
                        for (int e = 0; e < kVec; ++e) v[e] = v[e] / by.t;
                }
#pragma unroll
                for (int e = 0; e < kVec; ++e) out.v[e] = sili::from_f32<T>(take >> e & 1 ? v[e] : -INFINITY);
                *(P*)(y + i) = out;
            } else {
                take &= ~__funnelshift_r(s.touched[i >> 5], s.touched[(i >> 5) + 1], i & 31);
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    most = max_nan(most, take >> e & 1 ? sili::to_f32(in[k].v[e]) : -INFINITY);
            }
        }
        if (WRITE) {
            if (listed) {
                __syncthreads();
                for (int e = threadIdx.x; e < listed; e += kThreads) y[s.list[e]] = sili::from_f32<T>(result[e]);
            }
        } else {
            const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(top >> 32));
            const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(top >> 32) == high ? (uint32_t)top : 0u);
            const uint32_t most_y = __reduce_max_sync(0xffffffffu, (uint32_t)(key_of(by(most), 0) >> 32));
            if ((threadIdx.x & 31) == 0) {
                s.key[at][threadIdx.x >> 5] = (unsigned long long)high << 32 | low;
                s.y[at][threadIdx.x >> 5] = most_y;
            }
        }
    }

    // picking: the row's first token of the largest value, by one warp.  The parts of the row whose largest it is are read
    // again: after the division, elements next to it may be as large.
    __device__ void settle(int64_t row, int at) const {
        const int lane = threadIdx.x & 31, part = lane % (kThreads / 32);
        const unsigned long long key = s.key[at][part];
        const uint32_t y = s.y[at][part], high = (uint32_t)(key >> 32);
        const uint32_t all = max(__reduce_max_sync(0xffffffffu, y), __reduce_max_sync(0xffffffffu, high));
        unsigned parts = __ballot_sync(0xffffffffu, all && y == all) & ((1u << kThreads / 32) - 1u);
        uint32_t low = high == all ? (uint32_t)key : 0u;
        const T* x = (const T*)a.x + row * a.x_stride + t0;
        const uint32_t* may = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
        const int head = min((int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T)), n), packs = (n - head) / kVec;
        for (; parts; parts &= parts - 1) {
#pragma unroll 1
            for (int k = 0; k < kPacks; ++k) {
                const int p = (__ffs(parts) - 1) * 32 + lane + k * kThreads;
                if (p >= packs) break;
                const int i0 = head + p * kVec;
                const P in = *(const P*)(x + i0);
#pragma unroll 1
                for (int e = 0; e < kVec; ++e) {
                    const int i = i0 + e, v = t0 + i;
                    const unsigned long long here = key_of(by(pick_of(in, e)), v);
                    if ((uint32_t)(here >> 32) != all || (s.touched[i >> 5] >> (i & 31) & 1)) continue;
                    if (may && !(__ldg(may + (v >> 5)) >> (v & 31) & 1)) continue;
                    bool on_path = false;     // (the counts are those without the path)
                    if (a.drafted && s.has_path[at])
                        for (int j = 0; j < 64 * a.words; ++j)
                            on_path = on_path || (s.draft[j] == i && (s.masks[at][j >> 6] >> (j & 63) & 1));
                    if (!on_path) low = max(low, (uint32_t)here);
                }
            }
        }
        low = __reduce_max_sync(0xffffffffu, low);
        if (lane == 0) a.best[row * a.tiles + blockIdx.x % a.tiles] = all ? (unsigned long long)all << 32 | low : 0;
    }
    // element e of a pack, from memory's order of bytes
    static __device__ __forceinline__ float pick_of(const P& in, int e) {
        const uint4 w = *(const uint4*)&in;
        const int at = e * (int)sizeof(T) / 4;
        const uint32_t u = at == 0 ? w.x : at == 1 ? w.y : at == 2 ? w.z : w.w;
        if (sizeof(T) == 4) return __uint_as_float(u);
        const unsigned short h = (unsigned short)(e & 1 ? u >> 16 : u);
        return sili::to_f32(*(const T*)&h);
    }
};

template <typename T, bool WRITE>
__global__ void __launch_bounds__(kThreads) k_logits(const __grid_constant__ LogitArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& s = *(Shared*)smem;
    Logits<T, WRITE> k{a, s, s.value, s.value + (a.biases ? kTile : 0)};
    const int tile = blockIdx.x % a.tiles;
    k.t0 = tile * kTile;
    k.n = min(kTile, a.vocab - k.t0);
    const int64_t first = (int64_t)(blockIdx.x / a.tiles) * a.group, last = min(first + a.group, a.rows);
    int64_t begin = first, row0 = 0, row1 = -1;      // the current request's rows, the first of them here
    int r = -1;
    for (int64_t row = first; row < last; ++row) {
        if (row >= row1) {
            // the request that holds the row, if any
            begin = row;
            if (!a.starts) {
                r = row < a.requests ? (int)row : -1;
                row0 = row;
                row1 = row + 1;
            } else {
                int lo = 0, hi = a.requests;       // the last request with starts[r] <= row
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (a.starts[mid] <= row) lo = mid; else hi = mid;
                }
                r = a.requests ? lo : -1;
                if (r >= 0) {
                    row0 = max(a.starts[r], 0);
                    row1 = min((int64_t)a.starts[r + 1], a.rows);
                    if (row < row0 || row >= row1) r = -1;
                }
                if (r < 0) { row0 = row; row1 = row + 1; }
            }
            if (r >= 0) {
                __syncthreads();     // the last request's counts have been read
                k.count_request(r, row, min(last, row1), row0, row1);
                k.rep.set(a.repetition ? a.repetition[r] : 1.f);
                k.freq = a.frequency ? a.frequency[r] : 0.f;
                k.pres = a.presence ? a.presence[r] : 0.f;
                k.by.set(a.temperature ? a.temperature[r] : 0.f);
            }
        }
        const T* x = (const T*)a.x + row * a.x_stride + k.t0;
        T* y = WRITE ? (T*)a.y + row * a.y_stride + k.t0 : nullptr;
        if (r < 0) {
            // of no request: as it is
            if (WRITE)
                for (int i = threadIdx.x; i < k.n; i += kThreads) y[i] = x[i];
        } else {
            k.allow = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
            const bool path = a.drafted && s.has_path[row - begin];
            const int listed = s.listed;
            if (path) {
                __syncthreads();
                k.count_path((int)(row - begin), false, 0);
            }
            k.row(x, y, (int)(row - begin));
            if (path) {
                __syncthreads();
                k.count_path((int)(row - begin), true, listed);
            }
        }
        if (!WRITE && (r < 0 || row + 1 == last || row + 1 >= row1)) {
            // the end of the request's rows here
            __syncthreads();
            const int64_t at = begin + (threadIdx.x >> 5);
            if (r < 0) {
                if (threadIdx.x == 0) a.best[row * a.tiles + tile] = 0;
            } else if (at <= row) k.settle(at, (int)(at - begin));
        }
    }
}

// the largest of a row's tiles, a warp a row
__global__ void __launch_bounds__(128) k_picked(const unsigned long long* best, int64_t rows, int tiles, int* token) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= rows) return;
    unsigned long long top = 0;
    for (int i = threadIdx.x & 31; i < tiles; i += 32) top = max(top, best[row * tiles + i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) token[row] = top ? (int)(0xFFFFFFFFu - (uint32_t)top) : -1;
}

template <typename T, bool WRITE>
int launch(LogitArgs& a, cudaStream_t s) {
    const int smem = (int)sizeof(Shared) + ((a.biases ? kTile : 0) + (WRITE ? kTile : 0)) * 4;
    auto kernel = k_logits<T, WRITE>;
    static std::atomic<uint64_t> set{0};
    if (smem > 48 * 1024) CKL(sili::allow_smem(kernel, (int)sizeof(Shared) + 2 * kTile * 4, set));
    kernel<<<(unsigned)((a.rows + a.group - 1) / a.group * a.tiles), kThreads, smem, s>>>(a);
    sili::count_launch();
    CKL(cudaGetLastError());
    return SILI_OK;
}
template <bool WRITE>
int by_type(int dtype, LogitArgs& a, cudaStream_t s) {
    return dtype == SILI_F32 ? launch<float, WRITE>(a, s)
         : dtype == SILI_F16 ? launch<__half, WRITE>(a, s) : launch<__nv_bfloat16, WRITE>(a, s);
}

int check(const char* who, int dtype, int64_t rows, int vocab, int requests, int history_width, int words, int biases) {
    if (dtype < SILI_F32 || dtype > SILI_BF16) return bad(who, "unknown element type");
    if (rows < 0 || rows > 0x7fffffffLL || vocab < 1 || requests < 0 || history_width < 0 || biases < 0 || words < 0 || words > 4)
        return bad(who, "sizes out of range");
    return SILI_OK;
}

// Everything but where the result goes.
int prepare(const char* who, int dtype, const void* logits, int64_t stride, int64_t rows, int vocab, int requests,
            const sili_logit_rules* rules, LogitArgs& a) {
    if (!rules) return bad(who, "null array");
    const sili_logit_rules& q = *rules;
    if (const int e = check(who, dtype, rows, vocab, requests, q.history_width, q.words, q.biases)) return e;
    if (!logits && rows) return bad(who, "null array");
    if (rows > 1 && stride < vocab) return bad(who, "rows overlap");
    if ((q.history != nullptr) != (q.history_lens != nullptr)) return bad(who, "history and its lengths come together");
    if (q.history && requests > 1 && q.history_stride < 0) return bad(who, "sizes out of range");
    if ((q.drafted != nullptr) != (q.masks != nullptr) || (q.drafted && (!q.starts || q.words < 1)))
        return bad(who, "drafted tokens, masks and starts come together");
    if (q.biases && (!q.bias_tokens || !q.bias_values)) return bad(who, "null array");
    if (q.allowed && q.allowed_stride < (vocab + 31) / 32 && rows > 1) return bad(who, "mask rows overlap");
    if (!q.starts && requests != rows) return bad(who, "without starts there is one row a request");
    const int64_t item = dtype == SILI_F32 ? 4 : 2;
    if ((uintptr_t)logits % item) return bad(who, "logits must be aligned to their type");
    a = LogitArgs{logits, stride, nullptr, 0, rows, vocab, requests, q.starts, q.history_width ? q.history : nullptr,
                  q.history_stride, q.history_width, q.history_lens, q.prompt_lens, q.drafted, q.masks, q.words,
                  q.repetition, q.presence, q.frequency, q.temperature, q.bias_tokens, q.bias_values, q.biases, q.allowed,
                  q.allowed_stride, nullptr, nullptr, (vocab + kTile - 1) / kTile, 0};
    // rows that share a request's counts, as far as the mean goes
    const int64_t mean = requests ? (rows + requests - 1) / requests : rows;
    a.group = (int)std::min<int64_t>(kGroup, std::max<int64_t>(1, mean));
    if ((rows + a.group - 1) / a.group * a.tiles > 0x7fffffffLL) return bad(who, "sizes out of range");
    return SILI_OK;
}

}  // namespace

extern "C" {

int sili_adjust_logits(int dtype, const void* logits, int64_t stride, int64_t rows, int vocab, int requests,
                       const sili_logit_rules* rules, void* out, int64_t out_stride, void* stream) {
    const char* who = "adjust_logits";
    LogitArgs a;
    if (const int e = prepare(who, dtype, logits, stride, rows, vocab, requests, rules, a)) return e;
    if (rows == 0) return SILI_OK;
    if (!out) return bad(who, "null array");
    if (rows > 1 && out_stride < vocab) return bad(who, "rows overlap");
    if ((uintptr_t)out % (dtype == SILI_F32 ? 4 : 2)) return bad(who, "out must be aligned to its type");
    a.y = out;
    a.y_stride = out_stride;
    return by_type<true>(dtype, a, (cudaStream_t)stream);
}

int sili_pick_tokens_scratch(int64_t rows, int vocab, int64_t* bytes) {
    if (!bytes) return bad("pick_tokens_scratch", "null array");
    if (rows < 0 || rows > 0x7fffffffLL || vocab < 1) return bad("pick_tokens_scratch", "sizes out of range");
    *bytes = rows * ((vocab + kTile - 1) / kTile) * 8;
    return SILI_OK;
}

int sili_pick_tokens(int dtype, const void* logits, int64_t stride, int64_t rows, int vocab, int requests,
                     const sili_logit_rules* rules, int* token, void* scratch, void* stream) {
    const char* who = "pick_tokens";
    LogitArgs a;
    if (const int e = prepare(who, dtype, logits, stride, rows, vocab, requests, rules, a)) return e;
    if (rows == 0) return SILI_OK;
    if (!token || !scratch) return bad(who, "null array");
    if ((uintptr_t)scratch % 8) return bad(who, "scratch must be 8-byte aligned");
    a.best = (unsigned long long*)scratch;
    a.token = token;
    cudaStream_t s = (cudaStream_t)stream;
    if (const int e = by_type<false>(dtype, a, s)) return e;
    k_picked<<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(a.best, rows, a.tiles, token);
    sili::count_launch();
    CKL(cudaGetLastError());
    return SILI_OK;
}

}  // extern "C"
