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
// that its mask names) is counted on top and taken off again.  A bit a token
// tells which need the penalties at all: the rest is one pass over the row
// with 16-byte accesses, so the logits' bytes are what bounds it.
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
    int tile, tiles, group;    // tokens of a tile, tiles, rows of a CTA
};

// A larger value, then a lower token, has the larger key; NaN is above all numbers (the first one is picked) and -inf below
// every key (0).
__device__ __forceinline__ unsigned long long key_of(float y, int token) {
    uint32_t u = __float_as_uint(y + 0.f);     // -0 as 0
    if (u == 0xFF800000u) return 0;
    u = y != y ? 0xFFFFFFFFu : (int)u < 0 ? ~u : u | 0x80000000u;
    return (unsigned long long)u << 32 | (0xFFFFFFFFu - (uint32_t)token);
}

struct Rules {
    float rep, freq, pres, temp;
};

template <typename T, bool WRITE>
struct Logits {
    static constexpr int kVec = 16 / sizeof(T);
    using P = sili::Pack<T, kVec>;
    const LogitArgs& a;
    uint32_t* cnt;        // [tile]
    uint32_t* touched;    // [tile / 32 + 1]: a bit a token whose count is not 0
    float* bias;          // [tile], where kBiased says so
    int t0, n;            // the tile's first token, its tokens
    const uint32_t* allow;
    Rules w;

    __device__ __forceinline__ void note(uint32_t i, uint32_t what) const {
        if (what & kCount) atomicAdd(cnt + i, what); else atomicOr(cnt + i, what);
        atomicOr(touched + (i >> 5), 1u << (i & 31));
    }
    // the tokens of the request's history and bias list that lie in the tile
    __device__ void count_request(int r) {
        for (int i = threadIdx.x; i < n; i += kThreads) cnt[i] = 0;
        for (int i = threadIdx.x; i <= a.tile / 32; i += kThreads) touched[i] = 0;
        __syncthreads();
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
                const int v = list[j];
                const uint32_t i = (uint32_t)v - (uint32_t)t0;
                if (i >= (uint32_t)n) continue;
                // a token that is listed again: the first place adds them up, in order
                bool first = true;
                for (int k = 0; k < j; ++k) first = first && list[k] != v;
                if (!first) continue;
                float sum = value[j];
                for (int k = j + 1; k < a.biases; ++k)
                    if (list[k] == v) sum += value[k];
                bias[i] = sum;
                note(i, kBiased);
            }
        }
        __syncthreads();
    }
    // the row's path on top of the counts, or off them again
    __device__ void count_path(int64_t row, int64_t row0, int64_t row1, bool off) {
        if (!a.drafted) return;
        for (int j = threadIdx.x; j < 64 * a.words; j += kThreads) {
            if (!((uint64_t)a.masks[row * a.words + (j >> 6)] >> (j & 63) & 1) || row0 + j >= row1) continue;
            const uint32_t i = (uint32_t)a.drafted[row0 + j] - (uint32_t)t0;
            if (i >= (uint32_t)n) continue;
            if (!off) note(i, 1u);
            else if (atomicSub(cnt + i, 1u) == 1u) atomicAnd(touched + (i >> 5), ~(1u << (i & 31)));
        }
        __syncthreads();
    }

    __device__ __forceinline__ float ruled(float x, uint32_t what, int i) const {
        if (what) {
            // (a count also makes it seen)
            if (what & (kSeen | kCount)) x = x > 0.f ? x / w.rep : x * w.rep;
            if (what & kCount) {
                x = x - w.freq * (float)(what & kCount);
                x = x - w.pres;
            }
            if (what & kBiased) x = x + bias[i];
        }
        return w.temp > 0.f ? x / w.temp : x;
    }
    // bits [i, i + 8) of the tile's tokens, of which there is one word more than the tile needs
    static __device__ __forceinline__ uint32_t bits8(const uint32_t* words, int i) {
        return __funnelshift_r(words[i >> 5], words[(i >> 5) + 1], i & 31) & 0xFFu;
    }
    __device__ __forceinline__ bool may(int i) const {
        const int v = t0 + i;
        return !allow || (__ldg(allow + (v >> 5)) >> (v & 31) & 1);
    }
    __device__ __forceinline__ unsigned long long single(const T* x, T* y, int i) const {
        const float v = may(i) ? ruled(sili::to_f32(x[i]), cnt[i], i) : -INFINITY;
        if (WRITE) y[i] = sili::from_f32<T>(v);
        return WRITE ? 0 : key_of(v, t0 + i);
    }

    // one row of the tile; returns this thread's largest key
    __device__ unsigned long long row(const T* x, T* y) const {
        unsigned long long top = 0;
        // whole 16 bytes from the first aligned element on
        const int lead = (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T));
        const bool vectors = (uintptr_t)x % sizeof(T) == 0 && (!WRITE || (uintptr_t)y % 16 == (uintptr_t)x % 16);
        const int head = vectors ? min(lead, n) : n, packs = (n - head) / kVec, tail = head + packs * kVec;
        for (int i = threadIdx.x; i < head; i += kThreads) top = max(top, single(x, y, i));
        for (int i = tail + threadIdx.x; i < n; i += kThreads) top = max(top, single(x, y, i));
        for (int p0 = threadIdx.x; p0 < packs; p0 += 4 * kThreads) {
            P in[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (p0 + k * kThreads < packs) in[k] = *(const P*)(x + head + (p0 + k * kThreads) * kVec);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (p0 + k * kThreads >= packs) break;
                const int i = head + (p0 + k * kThreads) * kVec;
                const uint32_t some = bits8(touched, i);
                P out;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const float v = may(i + e) ? ruled(sili::to_f32(in[k].v[e]), some >> e & 1 ? cnt[i + e] : 0u, i + e) : -INFINITY;
                    if (WRITE) out.v[e] = sili::from_f32<T>(v);
                    else top = max(top, key_of(v, t0 + i + e));
                }
                if (WRITE) *(P*)(y + i) = out;
            }
        }
        return top;
    }
};

template <typename T, bool WRITE>
__global__ void __launch_bounds__(kThreads) k_logits(const __grid_constant__ LogitArgs a) {
    extern __shared__ uint32_t smem[];
    __shared__ unsigned long long s_top[kThreads / 32];
    Logits<T, WRITE> k{a};
    k.cnt = smem;
    k.touched = smem + a.tile;
    k.bias = (float*)(smem + a.tile + a.tile / 32 + 2);
    k.t0 = blockIdx.x * a.tile;
    k.n = min(a.tile, a.vocab - k.t0);
    const int64_t first = (int64_t)blockIdx.y * a.group, last = min(first + a.group, a.rows);
    int64_t row0 = 0, row1 = -1;      // the current request's rows
    int r = -1;
    for (int64_t row = first; row < last; ++row) {
        if (row >= row1) {
            // the request that holds the row, if any
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
                k.count_request(r);
                k.w.rep = a.repetition ? a.repetition[r] : 1.f;
                k.w.freq = a.frequency ? a.frequency[r] : 0.f;
                k.w.pres = a.presence ? a.presence[r] : 0.f;
                k.w.temp = a.temperature ? a.temperature[r] : 0.f;
            }
        }
        const T* x = (const T*)a.x + row * a.x_stride + k.t0;
        T* y = WRITE ? (T*)a.y + row * a.y_stride + k.t0 : nullptr;
        unsigned long long top = 0;
        if (r < 0) {
            // of no request: as it is
            if (WRITE)
                for (int i = threadIdx.x; i < k.n; i += kThreads) y[i] = x[i];
        } else {
            k.allow = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
            k.count_path(row, row0, row1, false);
            top = k.row(x, y);
            if (a.drafted) {
                __syncthreads();
                k.count_path(row, row0, row1, true);
            }
        }
        if (!WRITE) {
#pragma unroll
            for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            __syncthreads();
            if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
            __syncthreads();
            if (threadIdx.x == 0) {
#pragma unroll
                for (int i = 1; i < kThreads / 32; ++i) top = max(top, s_top[i]);
                a.best[row * a.tiles + blockIdx.x] = top;
            }
        }
        if (row + 1 >= row1) __syncthreads();     // the next request's counts come over these
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

// Tokens of a tile, and rows of a CTA.
constexpr int kTile = 8192;
int tile_of(int vocab) { return std::min(kTile, (vocab + 31) / 32 * 32); }

template <typename T, bool WRITE>
int launch(LogitArgs& a, cudaStream_t s) {
    const int smem = (a.tile + a.tile / 32 + 2 + (a.biases ? a.tile : 0)) * 4;
    auto kernel = k_logits<T, WRITE>;
    if (smem > 48 * 1024) CKL(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    kernel<<<dim3(a.tiles, (unsigned)((a.rows + a.group - 1) / a.group)), kThreads, smem, s>>>(a);
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
                  q.allowed_stride, nullptr, nullptr, tile_of(vocab), 0, 0};
    a.tiles = (vocab + a.tile - 1) / a.tile;
    // rows that share a request's counts, as far as the mean goes
    const int64_t mean = requests ? (rows + requests - 1) / requests : rows;
    a.group = (int)std::min<int64_t>(8, std::max<int64_t>(1, mean));
    if ((rows + a.group - 1) / a.group > 65535) a.group = (int)((rows + 65534) / 65535);
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
    *bytes = rows * ((vocab + tile_of(vocab) - 1) / tile_of(vocab)) * 8;
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
