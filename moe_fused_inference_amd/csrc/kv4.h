// kv4.h -- the MXFP4 KV cache of the kv4 entry points (kv4.hip, attn_kv4.hip):
// its layout, the place of a position in it, and the host's checks.
//
// A head row (one position's keys or values of one kv head) is D/2 bytes of
// E2M1 nibbles and D/32 E8M0 codes, the library's MXFP4 row.  A page holds
// `page` positions of every head, head by head, so that what one workgroup
// streams (one head's positions) lies together: kq, vq (n_pages, Hkv, page,
// D/2), ks, vs (n_pages, Hkv, page, D/32).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx_host.h"

namespace kv4 {

constexpr int kTile = 16;   // positions of an MFMA tile; pages hold whole tiles
constexpr int kMaxPos = 1 << 30;   // positions of a sequence

struct Cache {
    uint8_t* kq;
    uint8_t* ks;
    uint8_t* vq;
    uint8_t* vs;
    const int32_t* pages;   // (B, max_pages) or null: sequence b is page b
    int n_pages, page, max_pages, lg, Hkv, max_pos;   // lg: log2(page) with a table
};

// The head row of position pos (0 <= pos < max_pos) of sequence b, or -1
// where the table names no page of the pool.
__device__ __forceinline__ int64_t head_row(const Cache& c, int b, int g, int pos) {
    int pid = b, r = pos;
    if (c.pages) {
        pid = c.pages[(int64_t)b * c.max_pages + (pos >> c.lg)];
        if ((uint32_t)pid >= (uint32_t)c.n_pages) return -1;
        r = pos & (c.page - 1);
    }
    return ((int64_t)pid * c.Hkv + g) * c.page + r;
}

// The same of the two tiles of a unit, those of positions pos and pos + kTile (0 on), for the kernels that hold rows in 32
// bits, which make_cache makes enough of: kNoRow where there is none, or not `wanted`.  Both entries of the table at once:
// a unit's rows are one memory latency.
constexpr uint32_t kNoRow = 0xFFFFFFFFu;
__device__ __forceinline__ void unit_rows(const Cache& c, int b, int g, int64_t pos, bool wanted, uint32_t (&row)[2]) {
    const bool there[2] = {wanted && pos < c.max_pos, wanted && pos + kTile < c.max_pos};
    const int at[2] = {there[0] ? (int)pos : 0, there[1] ? (int)pos + kTile : 0};
    uint32_t pid[2] = {(uint32_t)b, (uint32_t)b}, r[2] = {(uint32_t)at[0], (uint32_t)at[1]};
    bool ok[2] = {there[0], there[1]};
    if (c.pages) {
        const int32_t* const table = c.pages + (int64_t)b * c.max_pages;
        pid[0] = table[at[0] >> c.lg];
        pid[1] = table[at[1] >> c.lg];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            ok[t] = ok[t] && pid[t] < (uint32_t)c.n_pages;
            r[t] = at[t] & (c.page - 1);
        }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) row[t] = ok[t] ? (pid[t] * (uint32_t)c.Hkv + (uint32_t)g) * (uint32_t)c.page + r[t] : kNoRow;
}

// 2^(code - 127) for the packed conversions, which read the exponent field: 0
// stands for 2^-127 there and 255 for NaN, as in E8M0.
__device__ __forceinline__ float scale_of(uint32_t code) { return __uint_as_float(code << 23); }

// The two nibbles of byte SEL of w as bf16 (exact; past bf16's range infinite).
template <int SEL>
__device__ __forceinline__ uint32_t pair_bf16(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
__device__ __forceinline__ uint4 eight_bf16(uint32_t w, float scale) {
    return make_uint4(pair_bf16<0>(w, scale), pair_bf16<1>(w, scale), pair_bf16<2>(w, scale), pair_bf16<3>(w, scale));
}

// The nibbles of w whose values under scale code `code` bf16 does not hold (infinite, or NaN): a 1 for each.
// 4 and 6 times 2^126, 2 and more times 2^127, and all of code 255.
__device__ __forceinline__ uint32_t not_finite(uint32_t w, uint32_t code) {
    const uint32_t bits = code == 255 ? ~0u : code == 254 ? w >> 2 : code == 253 ? w >> 2 & w >> 1 : 0u;
    return bits & 0x11111111u;
}
constexpr uint32_t kLargeScale = 253u << 23;   // of scale_of's exponent field: values that are not finite may be there

// The cache arguments of an entry point as a Cache; MXFP4_EINVAL with a message if they cannot be one.
inline int make_cache(Cache& c, const char* what, const uint8_t* kq, const uint8_t* ks, const uint8_t* vq, const uint8_t* vs,
                      const int32_t* pages, int n_pages, int page, int max_pages, int B, int Hkv, int D) {
    MXH_REQUIRE(kq && ks && vq && vs, "%s: null cache pointer", what);
    MXH_REQUIRE((((uintptr_t)kq | (uintptr_t)ks | (uintptr_t)vq | (uintptr_t)vs) & 15) == 0,
                "%s: cache tensors must be 16-byte aligned", what);
    MXH_REQUIRE(D == 64 || D == 128, "%s: head_dim D=%d (64 or 128)", what, D);
    MXH_REQUIRE(B > 0 && B <= 65535 && Hkv > 0 && Hkv <= 65535, "%s: B=%d Hkv=%d", what, B, Hkv);
    MXH_REQUIRE(n_pages > 0 && page > 0 && page % kTile == 0, "%s: page=%d must be a multiple of %d, n_pages=%d > 0", what,
                page, kTile, n_pages);
    int lg = 0;
    int64_t max_pos = page;
    if (pages) {
        MXH_REQUIRE((page & (page - 1)) == 0, "%s: page=%d must be a power of two with a page table", what, page);
        MXH_REQUIRE(max_pages > 0, "%s: max_pages=%d", what, max_pages);
        while ((1 << lg) < page) ++lg;
        max_pos = (int64_t)max_pages * page;
    } else {
        MXH_REQUIRE(n_pages >= B, "%s: %d sequences without a page table need as many pages, got %d", what, B, n_pages);
    }
    MXH_REQUIRE(max_pos <= kMaxPos, "%s: more than 2^30 positions a sequence", what);
    MXH_REQUIRE((int64_t)n_pages * page <= ((1ll << 32) - 2) / Hkv, "%s: a cache of 2^32 - 1 head rows or more", what);
    c = Cache{const_cast<uint8_t*>(kq), const_cast<uint8_t*>(ks), const_cast<uint8_t*>(vq), const_cast<uint8_t*>(vs),
              pages, n_pages, page, max_pages, lg, Hkv, (int)max_pos};
    return MXFP4_OK;
}

}  // namespace kv4
