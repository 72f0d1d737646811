// Decoding with drafted tokens, around the attention: the plan of a step's
// trees and what becomes of the tokens that were accepted.
//
// A request's drafted tokens are rows starts[r] .. starts[r + 1) of a step, a
// row's parent before it.  All of it is integer work on little data: bound by
// launches and the latency of a few loads, except that the accepted rows' keys
// and values move in every layer's cache.  Calls take what their host side does:
// 11 us for the plan of 192 requests of up to 250 drafts, 26 for the end of a
// small step, 44 for one of 96 requests in 12 layers (whose 24 arrays are
// checked).  Two take longer: an accepted way is walked a row at a time (64 rows
// 32 us, 256 rows 109; 27 and 91 without masks), and the rows of no request are
// one CTA's beside the requests' (24000 of them: the plan 21 us; 4000: 11).
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

#define CKD(x)                                                                                          \
    do {                                                                                                \
        const cudaError_t e_ = (x);                                                                     \
        if (e_ != cudaSuccess) return sili::set_error(SILI_ECUDA, std::string(#x) + ": " + cudaGetErrorString(e_)); \
    } while (0)

int bad(const char* who, const char* what) {
    return sili::set_error(SILI_EINVAL, std::string(who) + ": " + what);
}

// A request's rows, and the position of the token behind its committed ones.
struct Rows {
    int64_t row0;
    int n;
    int64_t base;
};
__device__ __forceinline__ Rows rows_of(const int* starts, const int* lens, int64_t tokens, int r) {
    Rows q;
    const int64_t s0 = min(max((int64_t)starts[r], (int64_t)0), tokens);
    const int64_t past = starts[r + 1], s1 = min(max(past, s0), tokens);     // (rows that the step lacks keep their places)
    q.row0 = s0;
    q.n = (int)(s1 - s0);
    q.base = max(lens[r], 0) - max(past - s0, (int64_t)0);
    return q;
}
// The rows of no request: [0, from) and [to, tokens).  Calls f for each, spread over the launch's last CTAs.
template <typename F>
__device__ __forceinline__ void other_rows(const int* starts, int requests, int64_t tokens, int cta, int ctas, F f) {
    const int64_t from = requests ? min(max((int64_t)starts[0], (int64_t)0), tokens) : 0;
    const int64_t to = requests ? min(max((int64_t)starts[requests], from), tokens) : 0;
    for (int64_t i = (int64_t)cta * blockDim.x + threadIdx.x; i < tokens - (to - from); i += (int64_t)ctas * blockDim.x)
        f(i < from ? i : i + (to - from));
}

// ── the plan of a step's trees ──────────────────────────────────────────────
// Row i sees its ancestors and itself.  A CTA holds one request's rows: every
// row's set of ancestors and the first one that is not yet in it, and log2(n)
// times takes in the set of that one (path doubling: the set is then twice as
// deep).  A row whose parent is not an earlier row (or -1) is none, and so are
// its descendants: an empty mask, position -1.
constexpr int kMostWords = 4;

struct PlanArgs {
    const int* parents;
    const int* starts;
    const int* lens;
    int requests;
    int64_t tokens;
    int words, window;
    int64_t* masks;
    int* positions;
};

__global__ void k_draft_tree(PlanArgs a) {
    __shared__ unsigned long long s_set[kMostWords][64 * kMostWords];
    __shared__ int s_next[64 * kMostWords];     // -1: complete, -2: none
    const int r = blockIdx.x, i = threadIdx.x, most = 64 * a.words;
    if (r >= a.requests) {
        other_rows(a.starts, a.requests, a.tokens, r - a.requests, gridDim.x - a.requests, [&](int64_t row) {
            for (int w = 0; w < a.words; ++w) a.masks[row * a.words + w] = 0;
            a.positions[row] = -1;
        });
        return;
    }
    const Rows q = rows_of(a.starts, a.lens, a.tokens, r);
    const int n = min(q.n, most);
    unsigned long long set[kMostWords];
    int next = -2;
    if (i < n) {
        const int p = a.parents[q.row0 + i];
        next = p >= -1 && p < i ? p : -2;
    }
#pragma unroll
    for (int w = 0; w < kMostWords; ++w) {
        set[w] = i < n && i >> 6 == w ? 1ull << (i & 63) : 0;
        s_set[w][i] = set[w];
    }
    s_next[i] = next;
    __syncthreads();
    for (int reach = 1; reach < n; reach *= 2) {
        if (next >= 0) {
            const int at = next;
            next = s_next[at];
#pragma unroll
            for (int w = 0; w < kMostWords; ++w) set[w] |= s_set[w][at];
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kMostWords; ++w) s_set[w][i] = set[w];
        s_next[i] = next;
        __syncthreads();
    }
    if (i < n) {
        int depth = 0;
#pragma unroll
        for (int w = 0; w < kMostWords; ++w) {
            if (next == -2) set[w] = 0;
            depth += __popcll(set[w]);
        }
        a.positions[q.row0 + i] = depth ? (int)(q.base + depth - 1) : -1;
        // a window keeps the nearest ancestors: those with the highest places
        int over = a.window ? depth - a.window : 0;
#pragma unroll
        for (int w = 0; w < kMostWords; ++w) {
            for (; over > 0 && set[w]; --over) set[w] &= set[w] - 1;
            if (w < a.words) a.masks[(q.row0 + i) * a.words + w] = (int64_t)set[w];
        }
    }
    for (int64_t k = (int64_t)most + i; k < q.n; k += blockDim.x) {     // more rows than the masks have bits
        for (int w = 0; w < a.words; ++w) a.masks[(q.row0 + k) * a.words + w] = 0;
        a.positions[q.row0 + k] = -1;
    }
}

// ── the end of a step ───────────────────────────────────────────────────────
// k_accept, a warp a request: from row 0 down to the first child whose token is
// the row's pick.  k_keep: the accepted rows' codes and scale bytes move up
// behind the committed tokens, a CTA a request and layer; one more CTA gives
// the pages back that hold none of a request's tokens any more.
constexpr int kCachesOfLaunch = 64;

struct SettleArgs {
    const int* drafted;
    const int* parents;
    const int64_t* masks;      // [tokens, words] or null: rows without a bit, or past the masks' bits, are none
    int words;
    const void* picked;
    int picked64;
    const int* starts;
    const int* lens;
    int requests;
    int64_t tokens;
    int* path;
    int* kept;
    int* token;
    int* lens_out;
    const int* table;
    int64_t stride;
    int width;
    int* ring;
    int ring_size;
    const int64_t* pool;
    int64_t* pool_out;
    int page;
    int64_t n_pages;
    int kv_heads, dim;
};
struct Caches {
    uint8_t* codes[kCachesOfLaunch];
    uint8_t* scales[kCachesOfLaunch];
};

__global__ void __launch_bounds__(128) k_accept(SettleArgs a) {
    const int ctas = (a.requests + 3) / 4, lane = threadIdx.x & 31;
    if ((int)blockIdx.x >= ctas) {
        other_rows(a.starts, a.requests, a.tokens, blockIdx.x - ctas, gridDim.x - ctas, [&](int64_t row) { a.path[row] = -1; });
        return;
    }
    const int r = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (r >= a.requests) return;
    const Rows q = rows_of(a.starts, a.lens, a.tokens, r);
    auto pick = [&](int i) {
        return a.picked64 ? ((const int64_t*)a.picked)[q.row0 + i] : (int64_t)((const int*)a.picked)[q.row0 + i];
    };
    auto there = [&](int i) {
        if (!a.masks) return true;
        int64_t any = 0;
#pragma unroll
        for (int w = 0; w < kMostWords; ++w) any |= w < a.words ? a.masks[(q.row0 + i) * a.words + w] : 0;
        return any != 0 && i < 64 * a.words;
    };
    int node = q.n > 0 && a.parents[q.row0] == -1 && there(0) ? 0 : -1, kept = 0;
    int64_t want = -1;
    while (node >= 0) {
        if (lane == 0) a.path[q.row0 + kept] = node;
        ++kept;
        want = pick(node);
        int child = -1;
        if (want >= 0)
            for (int at = (node + 1) & ~31; at < q.n; at += 32) {
                const int i = at + lane;
                const bool in = i > node && i < q.n;       // (all of a row's loads are asked for at once: a step waits for one)
                const int up = in ? a.parents[q.row0 + i] : -2;
                const int64_t own = in ? a.drafted[q.row0 + i] : -2;
                const bool is = in & there(in ? i : 0) & (up == node) & (own == want);
                const unsigned hit = __ballot_sync(0xffffffffu, is);
                if (hit) { child = at + __ffs(hit) - 1; break; }
            }
        node = child;
    }
    for (int i = kept + lane; i < q.n; i += 32) a.path[q.row0 + i] = -1;
    if (lane == 0) {
        a.kept[r] = kept;
        a.token[r] = (int)want;
        a.lens_out[r] = (int)max(q.base + kept, (int64_t)0);
    }
}

// The pages past ceil(lens_out / page) of each request, up to those that its lens took, go to the ring in request order.
// The table keeps its entries (nothing reads those past a request's tokens), so a call with the same inputs writes the
// same again.
__device__ void trim_pages(const SettleArgs& a) {
    __shared__ int64_t s_sum[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x / 32;
    const int64_t given = a.pool[1];
    int64_t carry = 0;
    for (int base = 0; base < a.requests; base += blockDim.x) {
        const int r = base + tid;
        int from = 0, to = 0, n = 0;
        const int* row = a.table;
        if (r < a.requests) {
            row += r * a.stride;
            from = (int)min(((int64_t)a.lens_out[r] + a.page - 1) / a.page, (int64_t)a.width);
            to = (int)min(((int64_t)max(a.lens[r], 0) + a.page - 1) / a.page, (int64_t)a.width);
            for (int c = from; c < to; ++c) n += row[c] >= 0;
        }
        int64_t x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t t = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += t;
        }
        if (lane == 31) s_sum[warp] = x;
        __syncthreads();
        int64_t all = 0;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) x += s_sum[w];
            all += s_sum[w];
        }
        int64_t at = given + carry + x - n;
        for (int c = from; c < to; ++c)
            if (row[c] >= 0) {
                a.ring[((at % a.ring_size) + a.ring_size) % a.ring_size] = row[c];
                ++at;
            }
        carry += all;
        __syncthreads();
    }
    if (tid == 0) {
        a.pool_out[0] = a.pool[0];
        a.pool_out[1] = given + carry;
    }
}

// A thread owns 16 bytes of codes (or a scale group's bytes) of one kv head's K or V and moves them row by row: a row
// goes to a place before it, rows ascend, so in order nothing is written before it has been read.  Eight rows are read
// before the first of them is written.
template <typename V>
__device__ __forceinline__ void move_rows(uint8_t* base, int64_t row_bytes, const int64_t* from, const int64_t* to, int n) {
    for (int j = 0; j < n; j += 8) {
        V v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (j + k < n && from[j + k] >= 0) v[k] = *(const V*)(base + from[j + k] * row_bytes);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (j + k < n && to[j + k] >= 0) *(V*)(base + to[j + k] * row_bytes) = v[k];
    }
}

constexpr int kKeepRows = 128, kKeepThreads = 256;
enum { kTrimsNot, kTrimsToo, kTrimsAlone };

__global__ void __launch_bounds__(kKeepThreads) k_keep(SettleArgs a, const __grid_constant__ Caches caches, int trims) {
    if ((int)blockIdx.x == a.requests || trims == kTrimsAlone) {
        if (trims != kTrimsNot && blockIdx.y == 0) trim_pages(a);
        return;
    }
    __shared__ int64_t s_from[kKeepRows], s_to[kKeepRows];     // rows of the first kv head's K; -1: not moved
    const int r = blockIdx.x;
    const Rows q = rows_of(a.starts, a.lens, a.tokens, r);
    const int kept = min(a.kept[r], q.n);
    uint8_t* codes = caches.codes[blockIdx.y];
    uint8_t* scales = caches.scales[blockIdx.y];
    const int E = a.dim / 32, chunks = a.dim / 32;             // 16-byte chunks of a row's codes, bytes of its scales
    const int units = 2 * a.kv_heads * chunks, heads2 = 2 * a.kv_heads;
    for (int j0 = 0; j0 < kept; j0 += kKeepRows) {
        const int n = min(kept - j0, kKeepRows);
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += kKeepThreads) {
            const int i = a.path[q.row0 + j0 + j];
            int64_t at[2] = {-1, -1};
            if (i > j0 + j && i < q.n) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int64_t pos = q.base + (k ? j0 + j : i), c = pos >= 0 ? pos / a.page : -1;
                    const int pg = c >= 0 && c < a.width ? a.table[r * a.stride + c] : -1;
                    if (pg >= 0 && pg < a.n_pages) at[k] = sili::kv4_row(pg, 0, 0, a.kv_heads, a.page) + (pos - c * a.page);
                }
            }
            const bool both = at[0] >= 0 && at[1] >= 0;
            s_from[j] = both ? at[0] : -1;
            s_to[j] = both ? at[1] : -1;
        }
        __syncthreads();
        for (int u = threadIdx.x; u < units + heads2; u += kKeepThreads) {
            if (u < units) {
                const int head = u / chunks, c = u - head * chunks;
                move_rows<uint4>(codes + (int64_t)head * a.page * (a.dim / 2) + c * 16, a.dim / 2, s_from, s_to, n);
            } else {
                uint8_t* base = scales + (int64_t)(u - units) * a.page * E;
                if (E == 2) move_rows<uint16_t>(base, 2, s_from, s_to, n);
                else if (E == 4) move_rows<uint32_t>(base, 4, s_from, s_to, n);
                else move_rows<uint2>(base, 8, s_from, s_to, n);
            }
        }
    }
}

}  // namespace

extern "C" {

int sili_draft_tree(const int* parents, const int* starts, const int* lens, int requests, int64_t tokens, int words,
                    int window, int64_t* masks, int* positions, void* stream) {
    const char* who = "draft_tree";
    if (requests < 0 || tokens < 0 || tokens > 0x7fffffffLL || window < 0) return bad(who, "sizes out of range");
    if (words < 1 || words > kMostWords) return bad(who, "masks must have 1 to 4 words a row");
    if (tokens == 0) return SILI_OK;
    if (!parents || !masks || !positions || (requests && (!starts || !lens))) return bad(who, "null array");
    PlanArgs a{parents, starts, lens, requests, tokens, words, window, masks, positions};
    // one CTA a request, and for the rows of none one more, or as many as they fill where there are no requests
    const int64_t extra = requests ? 1 : std::min<int64_t>((tokens + 255) / 256, 148);
    if (requests + extra > 0x7fffffffLL) return bad(who, "sizes out of range");
    k_draft_tree<<<(unsigned)(requests + extra), 64 * words, 0, (cudaStream_t)stream>>>(a);
    sili::count_launch();
    CKD(cudaGetLastError());
    return SILI_OK;
}

int sili_settle_masked_drafts(const int* drafted, const int* parents, const int64_t* masks, int words, const void* picked,
                              int picked64, const int* starts, const int* lens, int requests, int64_t tokens, int* path,
                              int* kept, int* token, int* lens_out, const int* table, int64_t table_stride, int width,
                              int* ring, int ring_size, const int64_t* pool, int64_t* pool_out, int n_caches,
                              void* const* codes, void* const* scales, int64_t n_pages, int page, int kv_heads, int dim,
                              void* stream) {
    const char* who = "settle_drafts";
    if (masks && (words < 1 || words > kMostWords)) return bad(who, "masks must have 1 to 4 words a row");
    if (requests < 0 || tokens < 0 || tokens > 0x7fffffffLL || width < 0 || ring_size < 1 || n_caches < 0 || n_pages < 0 ||
        page < 1 || kv_heads < 1)
        return bad(who, "sizes out of range");
    if (dim != 64 && dim != 128 && dim != 256) return bad(who, "head dimension must be 64, 128 or 256");
    if ((int64_t)kv_heads * page * dim > 0x7fffffffLL || n_pages > 0x7fffffffLL || requests > 0x7ffffff0)
        return bad(who, "sizes out of range");
    if (!ring || !pool || !pool_out || (n_caches && (!codes || !scales)) ||
        (tokens && (!drafted || !parents || !picked || !path)) ||
        (requests && (!starts || !lens || !kept || !token || !lens_out || (width && !table))))
        return bad(who, "null array");
    if (requests && table_stride < width) return bad(who, "table rows overlap");
    for (int i = 0; i < n_caches && n_pages; ++i) {
        if (!codes[i] || !scales[i]) return bad(who, "null array");
        if ((uintptr_t)codes[i] % 16 || (uintptr_t)scales[i] % 16) return bad(who, "codes and scales must be 16-byte aligned");
    }
    SettleArgs a{drafted, parents, masks, words, picked, picked64, starts, lens, requests, tokens, path, kept, token, lens_out, table,
                 table_stride, width, ring, ring_size, pool, pool_out, page, n_pages, kv_heads, dim};
    cudaStream_t s = (cudaStream_t)stream;
    k_accept<<<(unsigned)((requests + 3) / 4 + 1), 128, 0, s>>>(a);
    const int layers = n_pages ? n_caches : 0;
    for (int l0 = 0; l0 == 0 || l0 < layers; l0 += kCachesOfLaunch) {
        Caches c{};
        const int n = std::min(layers - l0, kCachesOfLaunch);
        for (int i = 0; i < n; ++i) { c.codes[i] = (uint8_t*)codes[l0 + i]; c.scales[i] = (uint8_t*)scales[l0 + i]; }
        if (n > 0) k_keep<<<dim3(requests + 1, n), kKeepThreads, 0, s>>>(a, c, l0 == 0 ? kTrimsToo : kTrimsNot);
        else k_keep<<<1, kKeepThreads, 0, s>>>(a, c, kTrimsAlone);
        sili::count_launch();
    }
    sili::count_launch();
    CKD(cudaGetLastError());
    return SILI_OK;
}

int sili_settle_drafts(const int* drafted, const int* parents, const void* picked, int picked64, const int* starts,
                       const int* lens, int requests, int64_t tokens, int* path, int* kept, int* token, int* lens_out,
                       const int* table, int64_t table_stride, int width, int* ring, int ring_size, const int64_t* pool,
                       int64_t* pool_out, int n_caches, void* const* codes, void* const* scales, int64_t n_pages, int page,
                       int kv_heads, int dim, void* stream) {
    return sili_settle_masked_drafts(drafted, parents, nullptr, 0, picked, picked64, starts, lens, requests, tokens, path, kept,
                                     token, lens_out, table, table_stride, width, ring, ring_size, pool, pool_out, n_caches,
                                     codes, scales, n_pages, page, kv_heads, dim, stream);
}

}  // extern "C"
