// What a decode or prompt step of a folded stack does around its
// projections: block tables and slot maps from request lengths, rotary
// positions, and the 4-bit key/value cache's append and read-back.
//
//   page tables   integer bookkeeping; bound by launch and L2 latency
//   rotary        streams q and k once; bound by HBM
//   append/read   stream k and v (and q) once; bound by HBM
//
// The attention over the cache is in kv4_attention.cu.
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

using sili::Pack;

#define CKS(x)                                                                                          \
    do {                                                                                                \
        const cudaError_t e_ = (x);                                                                     \
        if (e_ != cudaSuccess)                                                                          \
            return sili::set_error(e_ == cudaErrorMemoryAllocation ? SILI_ENOMEM : SILI_ECUDA,          \
                                   std::string(#x) + ": " + cudaGetErrorString(e_));                    \
    } while (0)

int bad(const char* who, const char* what) {
    return sili::set_error(SILI_EINVAL, std::string(who) + ": " + what);
}

// ── page tables ─────────────────────────────────────────────────────────────
// Request r holds cached[r] tokens and brings fresh[r] more.  Its pages are
// table[r][0 .. ceil(cached / page)); the pages that the new tokens open come
// from the ring of free pages in request order.  With
//   want[r]  = pages opened by r,  first[r] = sum of want before r,
//   starts[r] = sum of fresh before r
// every output is a lookup: token i belongs to the last r with starts[r] <= i
// (binary search), stands at cached[r] + i - starts[r], and the page of
// column c is table[r][c] where c was there before, else
// ring[(taken + first[r] + c - have[r]) mod size].  No lookup reads what the
// launch writes, so CTAs need no order among themselves.  The data is little
// (0.9 MB for 1531 requests and 68k tokens): a call is its launch and a few L2
// latencies, 19 us with the host's side at 64 and at 1531 requests alike.
struct TableArgs {
    const int* cached;
    const int* fresh;
    int n;
    int* table;
    int64_t stride;
    int width;
    const int* ring;
    int ring_size;
    const int64_t* pool;   // [2] pages taken from, pages given to the ring, ever
    int page;
    int64_t most;
    int* starts;
    int* lens;
    int64_t* slots;
    int* positions;
    int64_t* pool_out;
    int64_t* status;       // [3] pages that lacked, tokens beyond `most`, pages beyond the table's width
};

constexpr int kTableThreads = 256;
// Up to this many requests every CTA scans the lengths itself into shared
// memory (one launch); above, one CTA scans into global memory first.
constexpr int kTableSharedMost = 4096;

struct ReqPages {
    int64_t fresh, have, want, beyond;
};
__device__ __forceinline__ ReqPages pages_of(const TableArgs& a, int r) {
    ReqPages p;
    const int64_t c = max(a.cached[r], 0);
    p.fresh = max(a.fresh[r], 0);
    const int64_t need = (c + p.fresh + a.page - 1) / a.page;
    p.have = min((c + a.page - 1) / a.page, (int64_t)a.width);
    p.want = min(need, (int64_t)a.width) - p.have;
    p.beyond = need - min(need, (int64_t)a.width);
    return p;
}

// Exclusive scan of (fresh, want) over all requests by one CTA; fills
// starts[0..n] and first[0..n], returns the pages beyond the table's width
// (valid in every thread).
template <int THREADS>
__device__ int64_t scan_requests(const TableArgs& a, int* starts, int* first) {
    __shared__ int64_t s_sum[3][THREADS / 32];
    __shared__ int64_t s_carry[3];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < 3) s_carry[tid] = 0;
    __syncthreads();
    for (int base = 0; base < a.n; base += THREADS) {
        const int r = base + tid;
        int64_t v[3] = {0, 0, 0};
        if (r < a.n) {
            const ReqPages p = pages_of(a, r);
            v[0] = p.fresh; v[1] = p.want; v[2] = p.beyond;
        }
        int64_t x[3] = {v[0], v[1], v[2]};
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const int64_t t = __shfl_up_sync(0xffffffffu, x[k], o);
                if (lane >= o) x[k] += t;
            }
        }
        if (lane == 31)
            for (int k = 0; k < 3; ++k) s_sum[k][warp] = x[k];
        __syncthreads();
        int64_t before[3] = {s_carry[0], s_carry[1], s_carry[2]};
        for (int w = 0; w < warp; ++w)
            for (int k = 0; k < 3; ++k) before[k] += s_sum[k][w];
        if (r < a.n) {
            starts[r] = (int)(before[0] + x[0] - v[0]);
            first[r] = (int)(before[1] + x[1] - v[1]);
        }
        __syncthreads();
        if (tid == THREADS - 1)
            for (int k = 0; k < 3; ++k) s_carry[k] = before[k] + x[k];
        __syncthreads();
    }
    if (tid == 0) {
        starts[a.n] = (int)s_carry[0];
        first[a.n] = (int)s_carry[1];
    }
    __syncthreads();
    return s_carry[2];
}

// the last r in [0, n) with start[r] <= i (start[0] = 0 <= i)
__device__ __forceinline__ int find_request(const int* start, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ void fill_tables(const TableArgs& a, const int* starts, const int* first) {
    const int64_t step = (int64_t)gridDim.x * blockDim.x, at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t taken = a.pool[0];
    const int left = (int)max((int64_t)0, min(a.pool[1] - taken, (int64_t)a.ring_size));
    const int head = a.ring_size ? (int)(((taken % a.ring_size) + a.ring_size) % a.ring_size) : 0;
    auto ring_page = [&](int64_t j) {
        if (j >= left) return -1;
        int64_t x = head + j;
        if (x >= a.ring_size) x -= a.ring_size;
        return a.ring[x];
    };
    const int total = starts[a.n], opened = first[a.n];
    for (int64_t i = at; i < a.most; i += step) {
        int64_t slot = -1;
        int pos = -1;
        if (i < total) {
            const int r = find_request(starts, a.n, (int)i);
            const ReqPages p = pages_of(a, r);
            const int64_t x = (int64_t)max(a.cached[r], 0) + i - starts[r], c = x / a.page;
            pos = (int)x;
            if (c < a.width) {
                const int pg = c < p.have ? a.table[r * a.stride + c] : ring_page(first[r] + c - p.have);
                if (pg >= 0) slot = (int64_t)pg * a.page + (x - c * a.page);
            }
        }
        a.slots[i] = slot;
        a.positions[i] = pos;
    }
    for (int64_t j = at; j < opened; j += step) {
        // the last r with first[r] <= j opened page j (requests that open none share their successor's value)
        const int r = find_request(first, a.n, (int)j);
        const ReqPages p = pages_of(a, r);
        a.table[r * a.stride + p.have + (j - first[r])] = ring_page(j);
    }
}

__device__ void write_totals(const TableArgs& a, const int* starts, const int* first, int64_t beyond) {
    for (int r = threadIdx.x; r < a.n; r += blockDim.x)
        a.lens[r] = (int)((int64_t)max(a.cached[r], 0) + max(a.fresh[r], 0));
    if (threadIdx.x == 0) {
        const int64_t left = max((int64_t)0, min(a.pool[1] - a.pool[0], (int64_t)a.ring_size));
        const int64_t got = min((int64_t)first[a.n], left);
        a.pool_out[0] = a.pool[0] + got;
        a.pool_out[1] = a.pool[1];
        a.status[0] = first[a.n] - got;
        a.status[1] = max((int64_t)starts[a.n] - a.most, (int64_t)0);
        a.status[2] = beyond;
    }
}

__global__ void __launch_bounds__(kTableThreads) k_page_tables(TableArgs a) {
    extern __shared__ int s_scan[];   // starts [n + 1], first [n + 1]
    int* starts = s_scan;
    int* first = s_scan + a.n + 1;
    const int64_t beyond = scan_requests<kTableThreads>(a, starts, first);
    if (blockIdx.x == 0) {
        for (int r = threadIdx.x; r <= a.n; r += blockDim.x) a.starts[r] = starts[r];
        write_totals(a, starts, first, beyond);
    }
    fill_tables(a, starts, first);
}

__global__ void __launch_bounds__(1024) k_page_scan(TableArgs a, int* first) {
    const int64_t beyond = scan_requests<1024>(a, a.starts, first);
    write_totals(a, a.starts, first, beyond);
}
__global__ void __launch_bounds__(kTableThreads) k_page_fill(TableArgs a, const int* first) {
    fill_tables(a, a.starts, first);
}

// Pages of finished requests go back to the ring in request order.  One CTA,
// a warp per request; entries of -1 (pages that lacked) are not given back.
struct ReleaseArgs {
    const uint8_t* finished;
    int n;
    int* lens;
    int* table;
    int64_t stride;
    int width;
    int* ring;
    int ring_size;
    const int64_t* pool;
    int page;
    int64_t* pool_out;
    int* counts;           // [n] scratch
};
__global__ void __launch_bounds__(1024) k_release_pages(ReleaseArgs a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ int64_t s_total;
    auto cols = [&](int r) {
        const int64_t l = max(a.lens[r], 0);
        return (int)min((l + a.page - 1) / a.page, (int64_t)a.width);
    };
    for (int r = warp; r < a.n; r += 32) {
        int c = 0;
        if (a.finished[r])
            for (int j = lane; j < cols(r); j += 32) c += a.table[r * a.stride + j] >= 0;
        c = sili::warp_sum(c);
        if (lane == 0) a.counts[r] = c;
    }
    __syncthreads();
    if (warp == 0) {   // exclusive scan of the counts, in place
        int64_t carry = 0;
        for (int base = 0; base < a.n; base += 32) {
            const int r = base + lane;
            const uint32_t v = r < a.n ? (uint32_t)a.counts[r] : 0u;
            const uint32_t inc = sili::warp_inclusive_scan(v);
            if (r < a.n) a.counts[r] = (int)(carry + inc - v);
            carry += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) s_total = carry;
    }
    __syncthreads();
    const int64_t given = a.pool[1];
    for (int r = warp; r < a.n; r += 32) {
        if (!a.finished[r]) continue;
        int64_t at = given + a.counts[r];
        const int n = cols(r);
        for (int base = 0; base < n; base += 32) {
            const int j = base + lane;
            const int pg = j < n ? a.table[r * a.stride + j] : -1;
            const unsigned has = __ballot_sync(0xffffffffu, pg >= 0);
            if (pg >= 0) {
                const int64_t x = at + __popc(has & ((1u << lane) - 1u));
                a.ring[((x % a.ring_size) + a.ring_size) % a.ring_size] = pg;
            }
            if (j < n) a.table[r * a.stride + j] = -1;
            at += __popc(has);
        }
        __syncwarp();
        if (lane == 0) a.lens[r] = 0;
    }
    if (threadIdx.x == 0) {
        a.pool_out[0] = a.pool[0];
        a.pool_out[1] = given + s_total;
    }
}

// ── rotary positions ────────────────────────────────────────────────────────
// Pair (a, b) of a head becomes (a c - b s, b c + a s) with c, s the cosine
// and sine of the token's angle for that pair; the inverse rotation (its
// transpose: the gradient) takes -s.  Products are rounded one by one (no
// fused multiply-add), so the append's rotated K is the same bits.
struct RotaryArgs {
    const void* x[2];      // q, k
    void* y[2];
    int64_t xt[2], xh[2], yt[2], yh[2];   // strides of tokens and heads, in elements
    int heads[2];
    int64_t tokens;
    int dim, rot;
    const float* cos;
    const float* sin;
    int64_t n_positions;
    const void* positions;
    int pos64, interleaved;
    float sign;
};

__device__ __forceinline__ int64_t load_position(const void* p, int pos64, int64_t t) {
    return pos64 ? ((const int64_t*)p)[t] : (int64_t)((const int*)p)[t];
}

// V elements an access.  One unit of a head row is V pairs (half layout: V
// elements at i and V at i + rot/2), V/2 pairs (interleaved: V adjacent
// elements) or V elements that pass through; a thread keeps its unit and so
// its cosines while it walks the heads.  Each value is read and written once.
// 8191 tokens of 32 + 8 heads x 128 in fp32, forward and gradient: 131 us,
// 5.1 TB/s, bound by HBM (whole heads turned, 16001 tokens: 6.1 TB/s).  In
// bf16 4.2 TB/s, not HBM's bound: y may be x, so a thread's next loads wait
// behind its stores.  The fp32 form is held to 32 registers: with 8 CTAs an SM in
// place of 5 it took 131 us for 148; the 16-bit one keeps its registers (80
// us against 113 with 8).  Few tokens are spread over several CTAs each, a
// call of 64 tokens is its launch (19 us with the host's side).
template <typename T, int V>
__global__ void __launch_bounds__(V == 1 ? 1024 : 256, V == 1 || sizeof(T) == 2 ? 1 : 8) k_rotary(RotaryArgs a, int units, int rot_units, int rows) {
    using P = Pack<T, V>;
    const int u = threadIdx.x % units, row = threadIdx.x / units;
    if (row >= rows) return;
    const int64_t t = blockIdx.x;
    const int64_t pos = load_position(a.positions, a.pos64, t);
    const bool pad = pos < 0, past = pos >= a.n_positions;
    const float blank = pad ? 0.f : __int_as_float(0x7FC00000);
    const int half = a.rot / 2, heads = a.heads[0] + a.heads[1];
    const bool turns = u < rot_units;
    float c[V], s[V];
    if (turns && !pad && !past) {
        const int n = a.interleaved ? max(V / 2, 1) : V;
        const float* pc = a.cos + pos * half + (int64_t)u * n;
        const float* ps = a.sin + pos * half + (int64_t)u * n;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) { c[i] = __ldg(pc + i); s[i] = __ldg(ps + i) * a.sign; }
    }
    // element offsets of the unit's two parts
    int e0, e1 = -1;
    if (turns) {
        if (a.interleaved) { e0 = V > 1 ? u * V : 2 * u; if (V == 1) e1 = e0 + 1; }
        else { e0 = u * V; e1 = e0 + half; }
    } else {
        e0 = a.rot + (u - rot_units) * V;
    }
#pragma unroll 4
    for (int h = blockIdx.y * rows + row; h < heads; h += rows * gridDim.y) {
        const int w = h >= a.heads[0], hh = w ? h - a.heads[0] : h;
        const T* x = (const T*)a.x[w] + t * a.xt[w] + hh * a.xh[w];
        T* y = (T*)a.y[w] + t * a.yt[w] + hh * a.yh[w];
        P p0 = *(const P*)(x + e0), p1;
        if (e1 >= 0) p1 = *(const P*)(x + e1);
        if (pad || past) {
#pragma unroll
            for (int i = 0; i < V; ++i) p0.v[i] = p1.v[i] = sili::from_f32<T>(blank);
        } else if (e1 >= 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float f = sili::to_f32(p0.v[i]), g = sili::to_f32(p1.v[i]);
                p0.v[i] = sili::from_f32<T>(__fsub_rn(__fmul_rn(f, c[i]), __fmul_rn(g, s[i])));
                p1.v[i] = sili::from_f32<T>(__fadd_rn(__fmul_rn(g, c[i]), __fmul_rn(f, s[i])));
            }
        } else if (turns) {
#pragma unroll
            for (int i = 0; i + 1 < V; i += 2) {
                const float f = sili::to_f32(p0.v[i]), g = sili::to_f32(p0.v[i + 1]);
                p0.v[i] = sili::from_f32<T>(__fsub_rn(__fmul_rn(f, c[i / 2]), __fmul_rn(g, s[i / 2])));
                p0.v[i + 1] = sili::from_f32<T>(__fadd_rn(__fmul_rn(g, c[i / 2]), __fmul_rn(f, s[i / 2])));
            }
        }
        *(P*)(y + e0) = p0;
        if (e1 >= 0) *(P*)(y + e1) = p1;
    }
}

template <typename T, int V>
void launch_rotary(const RotaryArgs& a, cudaStream_t s) {
    const int rot_units = a.interleaved ? (V > 1 ? a.rot / V : a.rot / 2) : a.rot / 2 / V;
    const int units = rot_units + (a.dim - a.rot) / V;
    const int heads = a.heads[0] + a.heads[1];
    // as many heads side by side as 256 threads hold, evened out over the passes that all heads then take
    const int fit = std::max(1, std::min(heads, 256 / units)), passes = (heads + fit - 1) / fit;
    const int rows = (heads + passes - 1) / passes, threads = (rows * units + 31) / 32 * 32;
    // few tokens: more CTAs a token, so that every SM has some (one head a thread at the extreme)
    const int split = (int)std::max<int64_t>(1, std::min<int64_t>(passes, 592 / std::max<int64_t>(a.tokens, 1)));
    k_rotary<T, V><<<dim3((unsigned)a.tokens, split), threads, 0, s>>>(a, units, rot_units, rows);
    sili::count_launch();
}

template <typename T>
int run_rotary(const RotaryArgs& a, cudaStream_t s) {
    // 16-byte accesses where every row, part and stride allows them, else element by element
    constexpr int V = 16 / sizeof(T);
    bool wide = (a.interleaved ? a.rot % V == 0 : a.rot / 2 % V == 0) && (a.dim - a.rot) % V == 0;
    for (int w = 0; w < 2; ++w) {
        if (!a.heads[w]) continue;
        wide = wide && (uintptr_t)a.x[w] % 16 == 0 && (uintptr_t)a.y[w] % 16 == 0;
        for (int64_t st : {a.xt[w], a.xh[w], a.yt[w], a.yh[w]}) wide = wide && st % V == 0;
    }
    if (wide) launch_rotary<T, V>(a, s);
    else launch_rotary<T, 1>(a, s);
    return SILI_OK;
}

__global__ void k_rotary_table(double* inv, int half, int64_t n, float gain, float* cos_out, float* sin_out) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n * half; i += (int64_t)gridDim.x * blockDim.x) {
        double sv, cv;
        sincos((double)(i / half) * inv[i % half], &sv, &cv);
        cos_out[i] = (float)(cv * gain);
        sin_out[i] = (float)(sv * gain);
    }
}

// ── the cache: append and read ──────────────────────────────────────────────
struct AppendArgs {
    RotaryArgs r;          // x: q, k; y[0]: rotated q (heads[0] may be 0); rot 0: no rotation
    const void* v;
    int64_t vt, vh;
    uint8_t* codes;
    uint8_t* scales;
    int64_t n_slots;       // pages * page
    int page;
    const int64_t* slots;
};

// page and place of a slot; in 32 bits where the cache has no more slots
__device__ __forceinline__ int64_t split_slot(int64_t slot, int64_t n_slots, int page, int& off) {
    if (n_slots <= 0x7fffffff) {
        const uint32_t pg = (uint32_t)slot / (uint32_t)page;
        off = (int)((uint32_t)slot - pg * (uint32_t)page);
        return pg;
    }
    const int64_t pg = slot / page;
    off = (int)(slot - pg * page);
    return pg;
}

constexpr int kAppendThreads = 128;

// Eight consecutive elements a lane, dim / 8 lanes a head row (1, 2 or 4 rows
// a warp), so a group of 32 is four lanes: its maximum is two shuffles and its
// codes leave as four bytes a lane, whole rows together.  In half layout the
// rotation's partner element is rot/2 away, the same element of another lane
// (rot % 16 == 0), and comes by shuffle.  A CTA's warps share one token and
// walk its q, k and v rows with the token's cosines in registers.  Bound by
// instructions (the codes: three comparisons a value) before HBM: 16384
// tokens of 32 + 2 x 8 heads x 128 in bf16 take 111 us (8 CTAs an SM: 64
// registers; 127 us with 5), 3.1 TB/s, and the read-back below 24 us.
template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads, 8) k_kv4_append(const __grid_constant__ AppendArgs a) {
    constexpr int kLanes = D / 8, kRows = 32 / kLanes;     // lanes a row, rows a warp
    constexpr int kWarps = kAppendThreads / 32;
    constexpr int kWord = sizeof(T) == 2 ? 4 : 8;          // 32-bit words of a lane's elements
    const RotaryArgs& r = a.r;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % kLanes;
    const int64_t t = blockIdx.x;
    const int nq = r.heads[0], nk = r.heads[1];
    const int half = r.rot / 2, e = sub * 8;
    const bool turns = e < r.rot;
    const T* const qs = (const T*)r.x[0] + t * r.xt[0] + e;
    T* const qo = (T*)r.y[0] + t * r.yt[0] + e;
    const T* const ks = (const T*)r.x[1] + t * r.xt[1] + e;
    const T* const vs = (const T*)a.v + t * a.vt + e;
    const int first = (blockIdx.y * kWarps + warp) * kRows + lane / kLanes, step = kWarps * kRows * gridDim.y;
    using In = union { uint32_t u[kWord]; Pack<T, 8> p; uint4 v[kWord / 4]; };
    auto fetch = [&](const T* src, bool active) {
        In in;
#pragma unroll
        for (int i = 0; i < kWord / 4; ++i) in.v[i] = active ? ((const uint4*)src)[i] : make_uint4(0, 0, 0, 0);
        return in;
    };
    constexpr int kBatch = sizeof(T) == 2 ? 4 : 2;     // q rows whose loads are in flight together
    In batch[kBatch];
    auto fetch_q = [&](int h0) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) batch[k] = fetch(qs + (h0 + k * step) * r.xh[0], h0 + k * step < nq);
    };
    // before the position and the table's row, which wait for one another
    fetch_q(first);
    const int64_t slot = a.slots[t];
    const int64_t pos = r.rot ? load_position(r.positions, r.pos64, t) : 0;
    const bool pad = pos < 0, past = r.rot && pos >= r.n_positions;
    const float blank = pad ? 0.f : __int_as_float(0x7FC00000);
    float c[8], s[8];
    if (turns && !pad && !past) {
        if (r.interleaved) {
            const float4 u = __ldg((const float4*)(r.cos + pos * half + e / 2));
            const float4 v = __ldg((const float4*)(r.sin + pos * half + e / 2));
            c[0] = c[1] = u.x; c[2] = c[3] = u.y; c[4] = c[5] = u.z; c[6] = c[7] = u.w;
            s[0] = s[1] = v.x; s[2] = s[3] = v.y; s[4] = s[5] = v.z; s[6] = s[7] = v.w;
        } else {
            // the second half's sine with the sign that its sum takes
            const int j = e < half ? e : e - half;
            const float sign = e < half ? -1.f : 1.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 u = __ldg((const float4*)(r.cos + pos * half + j) + i);
                const float4 v = __ldg((const float4*)(r.sin + pos * half + j) + i);
                c[4 * i] = u.x; c[4 * i + 1] = u.y; c[4 * i + 2] = u.z; c[4 * i + 3] = u.w;
                s[4 * i] = sign * v.x; s[4 * i + 1] = sign * v.y; s[4 * i + 2] = sign * v.z; s[4 * i + 3] = sign * v.w;
            }
        }
    }
    const int partner = (lane - sub) + ((e < half ? e + half : e - half) / 8 & (kLanes - 1));
    const bool stored = slot >= 0 && slot < a.n_slots;
    int off;
    const int64_t pg = split_slot(stored ? slot : 0, a.n_slots, a.page, off);
    const int64_t row_at = pg * (2 * (int64_t)nk * a.page) + off;     // K's row of kv head 0
    // the row's eight values, turned where `turn` says so (every lane of the warp comes here together)
    auto turned = [&](const In& in, bool turn, float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = sili::to_f32(in.p.v[i]);
        if (!r.rot) return;
        if (r.interleaved) {
            if (turns && turn) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float f = x[i], g = x[i + 1];
                    x[i] = __fsub_rn(__fmul_rn(f, c[i]), __fmul_rn(g, s[i]));
                    x[i + 1] = __fadd_rn(__fmul_rn(g, c[i]), __fmul_rn(f, s[i]));
                }
            }
        } else {
            In other;
#pragma unroll
            for (int i = 0; i < kWord; ++i) other.u[i] = __shfl_sync(0xffffffffu, in.u[i], partner);
            if (turns && turn) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(sili::to_f32(other.p.v[i]), s[i]));
            }
        }
        if ((pad || past) && turn) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = blank;
        }
    };
    float x[8];
    for (int h0 = first; h0 - lane / kLanes < nq;) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int h = h0 + k * step;
            if (h - lane / kLanes >= nq) break;        // (the same for the whole warp)
            turned(batch[k], true, x);
            Pack<T, 8> o;
#pragma unroll
            for (int i = 0; i < 8; ++i) o.v[i] = sili::from_f32<T>(x[i]);
            if (h < nq) *(Pack<T, 8>*)(qo + h * r.yh[0]) = o;
        }
        h0 += kBatch * step;
        if (h0 - lane / kLanes < nq) fetch_q(h0);
    }
    if (!stored) return;
#pragma unroll 2
    for (int row = first; row - lane / kLanes < 2 * nk; row += step) {      // K's rows, then V's
        const bool is_v = row >= nk, active = row < 2 * nk;
        const int h = is_v ? row - nk : row;
        turned(fetch(is_v ? vs + h * a.vh : ks + h * r.xh[1], active), !is_v, x);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const uint32_t b = sili::kv4_scale_byte(m);
        const sili::Kv4Thresholds th(sili::kv4_scale(b));
        uint32_t packed = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) packed |= th.code(x[i]) << (4 * i);
        if (active) {
            const int64_t at = row_at + (int64_t)row * a.page;       // V's rows follow K's nk heads
            *(uint32_t*)(a.codes + at * (D / 2) + sub * 4) = packed;
            if (sub % 4 == 0) a.scales[at * (D / 32) + sub / 4] = (uint8_t)b;
        }
    }
}

struct ReadArgs {
    const uint8_t* codes;
    const uint8_t* scales;
    int64_t n_slots;
    int page, kv_heads;
    const int64_t* slots;
    int64_t tokens;
    void* k;
    void* v;
};

// 8 elements (4 bytes of codes) of K and of V a thread: one 16- or 32-byte
// write each.  A CTA takes whole tokens, so a token's units divide by 32-bit
// shifts only.
template <typename T>
__global__ void __launch_bounds__(256) k_kv4_read(ReadArgs a, int dim, int tokens_per_cta) {
    const int per = dim / 8, all = a.kv_heads * per;
    const int64_t t = (int64_t)blockIdx.x * tokens_per_cta + threadIdx.x / (unsigned)all;
    if (threadIdx.x >= (unsigned)(all * tokens_per_cta) || t >= a.tokens) return;
    const int64_t slot = a.slots[t];
    const bool stored = slot >= 0 && slot < a.n_slots;
    int off;
    const int64_t pg = split_slot(stored ? slot : 0, a.n_slots, a.page, off);
    const int64_t half = (int64_t)a.kv_heads * a.page, row0 = pg * (2 * half) + off;
    for (int u = threadIdx.x % (unsigned)all; u < all; u += 256) {
        const int h = u / per, unit = u - h * per;
        const int64_t at = row0 + (int64_t)h * a.page, to = (t * a.kv_heads + h) * dim + unit * 8;
        uint32_t code[2] = {0, 0}, sc[2] = {0, 0};
        if (stored) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                code[w] = __ldg((const uint32_t*)(a.codes + (at + w * half) * (dim / 2) + unit * 4));
                sc[w] = __ldg(a.scales + (at + w * half) * (dim / 32) + unit / 4);
            }
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t f[4];
            sili::kv4_decode4(code[w], f);
            const float scale = sili::kv4_scale(sc[w]);
            Pack<T, 8> o;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float2 v2 = sili::half2_bits_to_float2(f[q]);
                o.v[2 * q] = sili::from_f32<T>(v2.x * scale);
                o.v[2 * q + 1] = sili::from_f32<T>(v2.y * scale);
            }
            *(Pack<T, 8>*)((T*)(w ? a.v : a.k) + to) = o;
        }
    }
}

int check_rotary(const char* who, int dtype, int64_t tokens, int dim, int rot, const void* positions,
                 const float* cos, const float* sin, int64_t n_positions) {
    if (dtype < SILI_F32 || dtype > SILI_BF16) return bad(who, "unknown element type");
    if (tokens < 0 || tokens > 0x7fffffffLL || dim < 1) return bad(who, "sizes out of range");
    if (rot < 2 || rot % 2 || rot > dim) return bad(who, "the rotated part must be even, at least 2 and at most the head");
    if (n_positions < 1 || !cos || !sin) return bad(who, "no cosine / sine table");
    if (tokens && !positions) return bad(who, "null positions");
    return SILI_OK;
}

}  // namespace

extern "C" {

int sili_page_tables(const int* cached, const int* fresh, int n_requests, int* table, int64_t table_stride, int width,
                     const int* ring, int ring_size, const int64_t* pool, int page, int64_t max_tokens, int* starts,
                     int* lens, int64_t* slots, int* positions, int64_t* pool_out, int64_t* status, int* scratch,
                     void* stream) {
    const char* who = "page_tables";
    if (n_requests < 0 || width < 0 || ring_size < 0 || page < 1 || max_tokens < 0 || max_tokens > 0x7fffffffLL)
        return bad(who, "sizes out of range");
    if (!pool || !starts || !pool_out || !status || (n_requests && (!cached || !fresh || !lens)) ||
        (n_requests && width && !table) || (ring_size && !ring) || (max_tokens && (!slots || !positions)))
        return bad(who, "null array");
    if (n_requests && table_stride < width) return bad(who, "table rows overlap");
    cudaStream_t s = (cudaStream_t)stream;
    TableArgs a{cached, fresh, n_requests, table, table_stride, width, ring, ring_size, pool, page, max_tokens,
                starts, lens, slots, positions, pool_out, status};
    const int64_t items = std::max<int64_t>(max_tokens, n_requests);
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(148, (items + 511) / 512));
    if (n_requests <= kTableSharedMost) {
        k_page_tables<<<grid, kTableThreads, (size_t)(n_requests + 1) * 8, s>>>(a);
        sili::count_launch();
    } else {
        if (!scratch) return bad(who, "null scratch (needed above 4096 requests)");
        k_page_scan<<<1, 1024, 0, s>>>(a, scratch);
        k_page_fill<<<grid * 4, kTableThreads, 0, s>>>(a, scratch);
        sili::count_launch(2);
    }
    CKS(cudaGetLastError());
    return SILI_OK;
}

int sili_release_pages(const uint8_t* finished, int n_requests, int* lens, int* table, int64_t table_stride, int width,
                       int* ring, int ring_size, const int64_t* pool, int page, int64_t* pool_out, int* scratch,
                       void* stream) {
    const char* who = "release_pages";
    if (n_requests < 0 || width < 0 || ring_size < 1 || page < 1) return bad(who, "sizes out of range");
    if (!ring || !pool || !pool_out || (n_requests && (!finished || !lens || !scratch)) ||
        (n_requests && width && !table))
        return bad(who, "null array");
    if (n_requests && table_stride < width) return bad(who, "table rows overlap");
    ReleaseArgs a{finished, n_requests, lens, table, table_stride, width, ring, ring_size, pool, page, pool_out, scratch};
    k_release_pages<<<1, 1024, 0, (cudaStream_t)stream>>>(a);
    sili::count_launch();
    CKS(cudaGetLastError());
    return SILI_OK;
}

int sili_rotary_table(const double* inv_freq, int rot, int64_t n_positions, float gain, float* cos_out, float* sin_out,
                      void* stream) {
    if (rot < 2 || rot % 2 || n_positions < 1 || !inv_freq || !cos_out || !sin_out)
        return bad("rotary_table", "bad arguments");
    cudaStream_t s = (cudaStream_t)stream;
    const int half = rot / 2;
    double* dev = nullptr;
    CKS(cudaMallocAsync((void**)&dev, (size_t)half * 8, s));
    cudaError_t e = cudaMemcpyAsync(dev, inv_freq, (size_t)half * 8, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) {
        const int64_t n = n_positions * half;
        k_rotary_table<<<(unsigned)std::min<int64_t>((n + 255) / 256, 148 * 16), 256, 0, s>>>(dev, half, n_positions, gain,
                                                                                            cos_out, sin_out);
        sili::count_launch();
        e = cudaGetLastError();
    }
    cudaFreeAsync(dev, s);
    CKS(e);
    return SILI_OK;
}

int sili_rotary(int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                int64_t qo_token_stride, int64_t qo_head_stride, int q_heads, const void* k, int64_t k_token_stride,
                int64_t k_head_stride, void* k_out, int64_t ko_token_stride, int64_t ko_head_stride, int k_heads,
                int64_t tokens, int dim, int rot, const float* cos, const float* sin, int64_t n_positions,
                const void* positions, int pos64, int interleaved, int inverse, void* stream) {
    const char* who = "rotary";
    int rc = check_rotary(who, dtype, tokens, dim, rot, positions, cos, sin, n_positions);
    if (rc) return rc;
    if (q_heads < 0 || k_heads < 0) return bad(who, "sizes out of range");
    if (tokens == 0 || q_heads + k_heads == 0) return SILI_OK;
    if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return bad(who, "null array");
    if (dim > 1024) return bad(who, "head dimension above 1024");
    RotaryArgs a{{q, k}, {q_out, k_out}, {q_token_stride, k_token_stride}, {q_head_stride, k_head_stride},
                 {qo_token_stride, ko_token_stride}, {qo_head_stride, ko_head_stride}, {q_heads, k_heads}, tokens, dim,
                 rot, cos, sin, n_positions, positions, pos64, interleaved, inverse ? -1.f : 1.f};
    cudaStream_t s = (cudaStream_t)stream;
    rc = dtype == SILI_F32 ? run_rotary<float>(a, s)
       : dtype == SILI_F16 ? run_rotary<__half>(a, s) : run_rotary<__nv_bfloat16>(a, s);
    if (rc) return rc;
    CKS(cudaGetLastError());
    return SILI_OK;
}

int sili_kv4_append(int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                    int64_t qo_token_stride, int64_t qo_head_stride, int q_heads, const void* k, int64_t k_token_stride,
                    int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride, int kv_heads,
                    int64_t tokens, int dim, int rot, const float* cos, const float* sin, int64_t n_positions,
                    const void* positions, int pos64, int interleaved, uint8_t* codes, uint8_t* scales, int64_t n_pages,
                    int page, const int64_t* slots, void* stream) {
    const char* who = "kv4_append";
    if (rot) {
        const int rc = check_rotary(who, dtype, tokens, dim, rot, positions, cos, sin, n_positions);
        if (rc) return rc;
        if (rot % 16) return bad(who, "the rotated part must be a multiple of 16");
        if ((uintptr_t)cos % 16 || (uintptr_t)sin % 16) return bad(who, "the table must be 16-byte aligned");
    }
    if (dtype < SILI_F32 || dtype > SILI_BF16) return bad(who, "unknown element type");
    if (dim != 64 && dim != 128 && dim != 256) return bad(who, "head dimension must be 64, 128 or 256");
    if (tokens < 0 || tokens > 0x7fffffffLL || q_heads < 0 || kv_heads < 1 || n_pages < 0 || page < 1)
        return bad(who, "sizes out of range");
    if (q_heads && !rot) return bad(who, "q is only taken along to be rotated");
    if (tokens == 0) return SILI_OK;
    if (!k || !v || !slots || (q_heads && (!q || !q_out)) || (n_pages && (!codes || !scales))) return bad(who, "null array");
    const int64_t item = dtype == SILI_F32 ? 4 : 2;
    // (the stride of a single token or head is never used, and may be anything)
    auto aligned = [&](const void* p, int64_t ts, int64_t hs, int heads) {
        return (uintptr_t)p % 16 == 0 && (tokens == 1 || ts * item % 16 == 0) && (heads == 1 || hs * item % 16 == 0);
    };
    if (!aligned(k, k_token_stride, k_head_stride, kv_heads) || !aligned(v, v_token_stride, v_head_stride, kv_heads) ||
        (q_heads && (!aligned(q, q_token_stride, q_head_stride, q_heads) ||
                     !aligned(q_out, qo_token_stride, qo_head_stride, q_heads))))
        return bad(who, "rows must start on 16 bytes");
    if ((uintptr_t)codes % 16) return bad(who, "codes must be 16-byte aligned");
    AppendArgs a{{{q, k}, {q_out, nullptr}, {q_token_stride, k_token_stride}, {q_head_stride, k_head_stride},
                  {qo_token_stride, 0}, {qo_head_stride, 0}, {q_heads, kv_heads}, tokens, dim, rot, cos, sin, n_positions,
                  positions, pos64, interleaved, 1.f},
                 v, v_token_stride, v_head_stride, codes, scales, n_pages * page, page, slots};
    cudaStream_t s = (cudaStream_t)stream;
    const int per = kAppendThreads / 32 * (256 / dim);       // rows a pass of a CTA
    const int passes = (std::max(q_heads, 2 * kv_heads) + per - 1) / per;
    const dim3 grid((unsigned)tokens, (unsigned)std::max<int64_t>(1, std::min<int64_t>(passes, 592 / tokens)));
    auto go = [&](auto kernel) {
        kernel<<<grid, kAppendThreads, 0, s>>>(a);
        sili::count_launch();
    };
    if (dtype == SILI_F32) {
        if (dim == 64) go(k_kv4_append<float, 64>); else if (dim == 128) go(k_kv4_append<float, 128>); else go(k_kv4_append<float, 256>);
    } else if (dtype == SILI_F16) {
        if (dim == 64) go(k_kv4_append<__half, 64>);
        else if (dim == 128) go(k_kv4_append<__half, 128>); else go(k_kv4_append<__half, 256>);
    } else {
        if (dim == 64) go(k_kv4_append<__nv_bfloat16, 64>);
        else if (dim == 128) go(k_kv4_append<__nv_bfloat16, 128>); else go(k_kv4_append<__nv_bfloat16, 256>);
    }
    CKS(cudaGetLastError());
    return SILI_OK;
}

int sili_kv4_read(int dtype, const uint8_t* codes, const uint8_t* scales, int64_t n_pages, int page, int kv_heads, int dim,
                  const int64_t* slots, int64_t tokens, void* k_out, void* v_out, void* stream) {
    const char* who = "kv4_read";
    if (dtype < SILI_F32 || dtype > SILI_BF16) return bad(who, "unknown element type");
    if (dim != 64 && dim != 128 && dim != 256) return bad(who, "head dimension must be 64, 128 or 256");
    if (tokens < 0 || kv_heads < 1 || n_pages < 0 || page < 1) return bad(who, "sizes out of range");
    if (tokens == 0) return SILI_OK;
    if (!slots || !k_out || !v_out || (n_pages && (!codes || !scales))) return bad(who, "null array");
    if ((uintptr_t)k_out % 32 || (uintptr_t)v_out % 32 || (uintptr_t)codes % 16) return bad(who, "outputs must be 32-byte, codes 16-byte aligned");
    ReadArgs a{codes, scales, n_pages * page, page, kv_heads, slots, tokens, k_out, v_out};
    const int tpc = std::max(1, 256 / (kv_heads * (dim / 8)));
    if ((tokens + tpc - 1) / tpc > 0x7fffffffLL) return bad(who, "sizes out of range");
    const unsigned grid = (unsigned)((tokens + tpc - 1) / tpc);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == SILI_F32) k_kv4_read<float><<<grid, 256, 0, s>>>(a, dim, tpc);
    else if (dtype == SILI_F16) k_kv4_read<__half><<<grid, 256, 0, s>>>(a, dim, tpc);
    else k_kv4_read<__nv_bfloat16><<<grid, 256, 0, s>>>(a, dim, tpc);
    sili::count_launch();
    CKS(cudaGetLastError());
    return SILI_OK;
}

}  // extern "C"
