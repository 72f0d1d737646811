// What the two attention kernels over the 4-bit cache share.
#pragma once

#include <atomic>
#include <string>

#include "kv4.cuh"

namespace sili {

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
    void* workspace;
    uint32_t page16;       // page / 16
    uint32_t page_magic;   // ceil(2^32 / page16); 0 where page16 is 1
    uint32_t half_rows;    // token rows of K, and of V, in a page: kv_heads * page
    int polls, output_polls;   // of a wait before it gives up, and of a row tile's last one (kv4_prompt.cu sets them)
    const int64_t* masks;      // [tokens, words]: the drafted keys that a row sees; null where there are no drafts
    int words;

    // the table column of a key and the key's place in its page: one high product in place of a division, corrected by
    // one where the product is one too large (magic exceeds 2^32 / page16 by less than one)
    __device__ __forceinline__ int column(int key, int& off) const {
        const uint32_t run = (uint32_t)key >> 4;
        uint32_t col = page_magic ? __umulhi(run, page_magic) : run;
        int left = (int)(run - col * page16);
        if (left < 0) { --col; left += (int)page16; }
        off = left * 16 + (key & 15);
        return (int)col;
    }
};

// The workspace: a counter a CTA, the taken slots' bits, an error word; then the partial results of the one kernel, or
// the other's slots.
constexpr int kTicketBytes = 4096;
constexpr int kErrorWord = kTicketBytes / 4 - 1;
// A slot: the sums of a CTA's 256 rows that have left tensor memory (kv4_prompt.cu), and the maxima they stand over.  As
// many as CTAs can be resident, one an SM.
constexpr int kSlotWord = 512, kSlotWords = 5, kSlotRows = 256, kSlotDim = 128;
constexpr int64_t kSlotFloats = kSlotRows * (kSlotDim + 1), kSlotBytes = kSlotWords * 32 * kSlotFloats * 4;

// p = 2^(x - m + 8): room below (a half's subnormals start at 2^-32 of the largest) and above (x may exceed m by 7)
constexpr float kLift = 8.f, kSlack = 7.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    uint32_t c;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    return c;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Lets a kernel have `bytes` of dynamic shared memory on the current device; `set` remembers the devices (a bit each)
// on which it has, which the attribute belongs to.
template <typename K>
inline cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t>& set) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bit && (set.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) set.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

constexpr int kUnit = 128;              // keys of a unit of the work that is cut evenly over the CTAs

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
template <int ROWS, int kWarps>
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

// Long 16-bit prompts (kv4_prompt.cu): whether this call is one, and the launch.
bool kv4_prompt_takes(int dtype, int dim, int64_t tokens, int heads, int kv_heads, int64_t most_new);
int kv4_prompt_launch(int dtype, int dim, const AttendArgs& a, cudaStream_t s);

// The process's limits of a wait, into the arguments (kv4_prompt.cu).
void kv4_polls(AttendArgs& a);
// Trees with many 16-bit rows a request (kv4_tree.cu).
bool kv4_tree_takes(int dtype, int dim, int64_t rows);
int64_t kv4_tree_workspace(int dim, int64_t rows);
int kv4_tree_launch(int dtype, int dim, const AttendArgs& a, int64_t rows, cudaStream_t s);

}  // namespace sili
