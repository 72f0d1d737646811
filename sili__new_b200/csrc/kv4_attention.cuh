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

// Long 16-bit prompts (kv4_prompt.cu): whether this call is one, and the launch.
bool kv4_prompt_takes(int dtype, int dim, int64_t tokens, int heads, int kv_heads, int64_t most_new);
int kv4_prompt_launch(int dtype, int dim, const AttendArgs& a, cudaStream_t s);

}  // namespace sili
