// 4-bit keys and values of 128 keys at a time into stages of shared memory, as
// the tensor-memory kernels over the cache take them: K as it lies, V
// transposed by interleaving the nibbles of two keys, halves, with the
// 128-byte swizzle.
#pragma once

#include "kv4_attention.cuh"
#include "kv4_mma.cuh"

namespace sili {
namespace mma {

constexpr int kKeys = 128;            // keys a stage of shared memory

// Eight warps (threads kSoftmax .. kSoftmax + 255): stages [w.j0, w.last) of request w.r's and kv head w.h's keys, n0 and
// on of the kernel's, into two buffers in turn.  S holds the buffers k, v, their barriers kv_full and kv_free, and of each
// which keys' pages exist (there) and which V scales are no numbers (odd_keys; odd: the last stage that had any, plus one).
// False: a wait gave up.
template <int D, typename S, typename W>
__device__ __forceinline__ bool dequantise_stages(const AttendArgs& a, S& s, const W& w, int kSoftmax, int n0) {
    constexpr int E = D / 32;
    const int tid = threadIdx.x - kSoftmax, dw = tid >> 5, lane = tid & 31;
    // K: 16 keys a warp, E lanes a key, 16 bytes (one group of 32) each
    constexpr int kPer = 32 / E, kLoads = 16 / kPer;       // keys of one load instruction, loads
    const int kq = lane % E, kkey = dw * 16;
    // V: 8 keys x 8 elements a thread; lane & 7 numbers the keys, so a store instruction fills whole rows
    const int half = dw & 1, c = lane & 7, db = (dw >> 1) * 4 + (lane >> 3), vkey = half * 64 + c * 8;
    const bool has_v = db < D / 8;
    const int vg = db >> 2;
    uint4 rk[kLoads], sv[E / 2];
    uint32_t sk[kLoads], rv[8];
    int pk, pv, next_pk, next_pv;
    auto page_of = [&](int key) {
        // whole runs of 16 keys (they share a page and a bit of `there`), of which the last may reach past the end
        int off;
        return (key & ~15) < w.len ? __ldg(a.table + w.r * a.stride + a.column(key, off)) : -1;
    };
    auto pages = [&](int j) {
        next_pk = page_of(j * kKeys + kkey);
        next_pv = page_of(j * kKeys + vkey);
    };
    const int64_t head_rows = (int64_t)w.h * a.page, v_rows = (int64_t)a.kv_heads * a.page;
    auto row_of = [&](int pg, int key) {
        int off;
        a.column(key, off);
        return (int64_t)pg * (2 * v_rows) + head_rows + off;
    };
    // (what a missing page leaves in K is masked in S; its V scales are zeroed, for 0 * NaN is none)
    auto load_k = [&](int j) {
        const bool there = pk >= 0 && pk < a.n_pages;
        if (there) {
            const int64_t row = row_of(pk, j * kKeys + kkey) + lane / E;
            const uint8_t* codes = a.codes + row * (D / 2) + kq * 16;
            const uint8_t* scales = a.scales + row * E + kq;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                rk[i] = __ldg((const uint4*)(codes + i * kPer * (D / 2)));
                sk[i] = __ldg(scales + i * kPer * E);
            }
        }
        return there;
    };
    auto load_v = [&](int j) {
        if (has_v && pv >= 0 && pv < a.n_pages) {
            const int64_t row = row_of(pv, j * kKeys + vkey) + v_rows;
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
    const uint32_t pick = E == 4 ? (uint32_t)(vg | (4 + vg) << 8) : (uint32_t)(vg | (2 + vg) << 8);      // selector nibbles 0 and 2
    auto pair_of = [&](int p) {
        if constexpr (E == 4) {
            const uint4 v = sv[p >> 1 & (E / 2 - 1)];
            return __byte_perm(p & 1 ? v.z : v.x, p & 1 ? v.w : v.y, pick) & 0x00FF00FFu;
        } else {
            const uint32_t v = p == 0 ? sv[0].x : p == 1 ? sv[0].y : p == 2 ? sv[0].z : sv[0].w;
            return __byte_perm(v, 0, pick) & 0x00FF00FFu;
        }
    };
    pages(w.j0);
    pk = next_pk; pv = next_pv;
    bool there = load_k(w.j0);
    load_v(w.j0);
    if (w.j0 + 1 < w.last) pages(w.j0 + 1);
    for (int j = w.j0; j < w.last; ++j) {
        const int n = n0 + j - w.j0, st = n & 1;
        const bool more = j + 1 < w.last;
        if (n >= 2 && !bar_wait(&s.kv_free[st], ((n >> 1) - 1) & 1, &s.dead, a.polls)) return false;
        // K: rows are keys
        if (lane == 0) s.there[st][dw] = there;
        {
            uint8_t* block = s.k[st] + (kq >> 1) * (kKeys * 128);
            // lanes of the second block go through their four chunks two further on: eight lanes, eight banks' worth
            const bool far = E == 4 && (kq & 2);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int key = kkey + lane / E + i * kPer;
                const uint32_t sc = sk[i] * 0x00800080u;
                const uint32_t wd[4] = {far ? rk[i].z : rk[i].x, far ? rk[i].w : rk[i].y, far ? rk[i].x : rk[i].z,
                                        far ? rk[i].y : rk[i].w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t f[4];
                    sili::kv4_decode4(wd[q], f);
                    const int ch = (kq & 1) * 4 + (far ? q ^ 2 : q);
                    *(uint4*)(block + chunk_at(key, ch)) =
                        make_uint4(mul2(f[0], sc), mul2(f[1], sc), mul2(f[2], sc), mul2(f[3], sc));
                }
            }
        }
        if (more) {
            pk = next_pk;
            there = load_k(j + 1);
        }
        // V: rows are elements; scales that are no numbers are left out and noted
        if (has_v) {
            uint32_t pairs[4], odd_any = 0, bits = 0;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                pairs[p] = pair_of(p);
                odd_any |= pairs[p] + 0x00080008u;      // carries into bit 8 of a byte of at least 0xF8
            }
            if (odd_any & 0x01000100u) {
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    if ((pairs[p] & 0xFFu) >= 0xF8u) { bits |= 1u << (2 * p); pairs[p] &= 0xFFFF0000u; }
                    if ((pairs[p] >> 16) >= 0xF8u) { bits |= 2u << (2 * p); pairs[p] &= 0xFFFFu; }
                }
                *(volatile int*)&s.odd[st] = n + 1;
            }
            if ((db & 3) == 0) s.odd_keys[st][half * 8 + c][vg] = (uint8_t)bits;
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
                *(uint4*)(block + chunk_at(d, c)) = make_uint4(even[0][b], even[1][b], even[2][b], even[3][b]);
                *(uint4*)(block + chunk_at(d + 1, c)) = make_uint4(odd[0][b], odd[1][b], odd[2][b], odd[3][b]);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        bar_arrive(&s.kv_full[st]);
        if (more) {
            pv = next_pv;
            load_v(j + 1);
            if (j + 2 < w.last) pages(j + 2);
        }
    }
    return true;
}

}  // namespace mma
}  // namespace sili
