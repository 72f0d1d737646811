// Attention over the 4-bit paged cache: one warp per (query token, head),
// keys one by one, an online softmax in fp32.
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

#define CKV(x)                                                                                          \
    do {                                                                                                \
        const cudaError_t e_ = (x);                                                                     \
        if (e_ != cudaSuccess)                                                                          \
            return sili::set_error(e_ == cudaErrorMemoryAllocation ? SILI_ENOMEM : SILI_ECUDA,          \
                                   std::string(#x) + ": " + cudaGetErrorString(e_));                    \
    } while (0)

int bad(const char* who, const char* what) {
    return sili::set_error(SILI_EINVAL, std::string(who) + ": " + what);
}

struct AttendArgs {
    const void* q;
    int64_t qt, qh;        // q strides of tokens and heads, in elements
    int64_t tokens;
    int heads, kv_heads;
    const uint8_t* codes;
    const uint8_t* scales;
    int64_t n_pages;
    int page;
    const int* table;
    int64_t stride;
    int width;
    const int* lens;
    int requests;
    const int* starts;     // null: request r's one token is row r
    float scale;
    int window;
    void* out;             // [tokens, heads, dim]
    float* lse;            // [tokens, heads] or null
};

template <typename T, int E>
__global__ void __launch_bounds__(128) k_attend_simple(AttendArgs a) {
    constexpr int kDim = 32 * E;
    const int lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (id >= a.tokens * a.heads) return;
    const int64_t t = id / a.heads;
    const int h = (int)(id - t * a.heads), g = h / (a.heads / a.kv_heads);
    int r = -1, ahead = 0;   // the token's request and how many of its tokens follow
    if (a.starts) {
        for (int i = 0; i < a.requests; ++i)
            if (a.starts[i] <= t && t < a.starts[i + 1]) { r = i; ahead = (int)(a.starts[i + 1] - 1 - t); break; }
    } else if (t < a.requests) {
        r = (int)t;
    }
    float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        q[i] = sili::to_f32(((const T*)a.q)[t * a.qt + h * a.qh + lane * E + i]) * a.scale;
        o[i] = 0.f;
    }
    if (r >= 0) {
        const int64_t len = min((int64_t)max(a.lens[r], 0), (int64_t)a.width * a.page);
        const int64_t pos = (int64_t)a.lens[r] - 1 - ahead;
        const int64_t end = min(len, pos + 1), from = a.window ? max(pos - a.window + 1, (int64_t)0) : 0;
        for (int64_t j = from; j < end; ++j) {
            const int64_t c = j / a.page;
            const int pg = a.table[r * a.stride + c];
            if (pg < 0 || pg >= a.n_pages) continue;
            float kv[2][E];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int64_t at = sili::kv4_row(pg, w, g, a.kv_heads, a.page) + (j - c * a.page);
                const uint8_t* p = a.codes + at * (kDim / 2) + lane * (E / 2);
                const float sc = sili::kv4_scale(a.scales[at * E + lane / (32 / E)]);
#pragma unroll
                for (int i = 0; i < E / 2; ++i) {
                    kv[w][2 * i] = sili::fp4_decode(p[i] & 15u) * sc;
                    kv[w][2 * i + 1] = sili::fp4_decode(p[i] >> 4) * sc;
                }
            }
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) s = fmaf(q[i], kv[0][i], s);
            s = sili::warp_sum(s);
            const float mn = fmaxf(m, s), f = m == mn ? 1.f : expf(m - mn), p = expf(s - mn);
            l = l * f + p;
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = fmaf(p, kv[1][i], o[i] * f);
            m = mn;
        }
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
        ((T*)a.out)[id * kDim + lane * E + i] = sili::from_f32<T>(l > 0.f ? o[i] / l : (l == 0.f ? 0.f : l));
    if (lane == 0 && a.lse) a.lse[id] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace

extern "C" {

int sili_kv4_attention_workspace(int64_t* bytes) {
    if (!bytes) return bad("kv4_attention_workspace", "null array");
    *bytes = 0;
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
    if (tokens < 0 || heads < 1 || kv_heads < 1 || n_pages < 0 || width < 0 || requests < 0 || window < 0 || most_new < 0)
        return bad(who, "sizes out of range");
    if (heads % kv_heads) return bad(who, "the kv heads must divide the query heads");
    if (tokens == 0) return SILI_OK;
    if (!q || !out || (requests && !lens) || (requests && width && !table) || (n_pages && (!codes || !scales)))
        return bad(who, "null array");
    if (requests && table_stride < width) return bad(who, "table rows overlap");
    if ((uintptr_t)codes % 16 || (uintptr_t)scales % 4) return bad(who, "codes must be 16-byte, scales 4-byte aligned");
    const int64_t item = dtype == SILI_F32 ? 4 : 2;
    if ((uintptr_t)q % 8 || (uintptr_t)out % 16 || q_token_stride * item % 8 || q_head_stride * item % 8)
        return bad(who, "q rows must be 8-byte aligned");
    AttendArgs a{q, q_token_stride, q_head_stride, tokens, heads, kv_heads, codes, scales, n_pages, page, table,
                 table_stride, width, lens, requests, starts, scale, window, out, lse};
    cudaStream_t s = (cudaStream_t)stream;
    (void)workspace;
    const int64_t ctas = (tokens * heads + 3) / 4;
    if (ctas > 0x7fffffffLL) return bad(who, "sizes out of range");
    auto go = [&](auto kernel) {
        kernel<<<(unsigned)ctas, 128, 0, s>>>(a);
        sili::count_launch();
    };
    if (dtype == SILI_F32) {
        if (dim == 64) go(k_attend_simple<float, 2>); else if (dim == 128) go(k_attend_simple<float, 4>); else go(k_attend_simple<float, 8>);
    } else if (dtype == SILI_F16) {
        if (dim == 64) go(k_attend_simple<__half, 2>); else if (dim == 128) go(k_attend_simple<__half, 4>); else go(k_attend_simple<__half, 8>);
    } else {
        if (dim == 64) go(k_attend_simple<__nv_bfloat16, 2>);
        else if (dim == 128) go(k_attend_simple<__nv_bfloat16, 4>); else go(k_attend_simple<__nv_bfloat16, 8>);
    }
    CKV(cudaGetLastError());
    return SILI_OK;
}

}  // extern "C"
