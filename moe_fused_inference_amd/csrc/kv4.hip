// kv4.hip -- the MXFP4 KV cache's write and read-back (layout: kv4.h).
//
//   kv4_write_kernel    k, v rows (bf16, fp16 or fp32) -> MXFP4 at positions
//                       dpos[b] + m: per 32-block the library's quantizer
//                       (quant_rows.h), eight values a lane, a block a quad; or at
//                       the places of a list (slots), a token each.
//   qk_rope_kv4_kernel  the decode step's form: q / k head RMSNorm and RoPE of
//                       the fp32 projections (head_rope.h), q out as bf16, k
//                       and bf16(v) to the cache.
//   kv4_read_kernel     rows of a context as bf16, fp16 or fp32, eight values a
//                       lane by the hardware's packed conversion.
//
// All are bound by memory, or at a few tokens by the launch.  The place of a
// row (page table, head) is found per lane: a table entry is one load that the
// row's lanes share.
#include "head_rope.h"
#include "kv4.h"
#include "mx_device.h"
#include "mx_host.h"
#include "quant_rows.h"

namespace {

using kv4::Cache;

// The positions of the call: token m of sequence b at at[b] + m (at null: m).
// Row -1 if that lies outside the cache or on no page.
__device__ __forceinline__ int64_t row_of(const Cache& c, const int32_t* at, int b, int m, int g) {
    const int64_t pos = (int64_t)(at ? at[b] : 0) + m;
    if (pos < 0 || pos >= c.max_pos) return -1;
    return kv4::head_row(c, b, g, (int)pos);
}

// The row of head g at a place of the pool, page * (rows of a page) + row, or -1.
__device__ __forceinline__ int64_t row_of_slot(const Cache& c, int64_t slot, int g) {
    if (slot < 0 || slot >= (int64_t)c.n_pages * c.page) return -1;       // (what is left has 32 bits)
    const uint32_t pid = (uint32_t)slot / (uint32_t)c.page;
    return ((int64_t)pid * c.Hkv + g) * c.page + ((uint32_t)slot - pid * (uint32_t)c.page);
}

// Thread: eight consecutive values of a head row of k and of v; LU = log2(D / 8).
// SLOTS: the tokens' places, and M = 1; else dpos.
template <int SRC, int LU, bool SLOTS>
__global__ __launch_bounds__(256) void kv4_write_kernel(const void* __restrict__ k, const void* __restrict__ v,
                                                        int64_t ldk, int64_t ldv, int vec, Cache c,
                                                        const int32_t* __restrict__ dpos, const int64_t* __restrict__ slots, int M,
                                                        int64_t heads) {
    constexpr int D = 8 << LU;
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t th = idx >> LU;             // token * Hkv + head
    if (th >= heads) return;                  // whole quads: heads << LU is a multiple of 8
    const int u = (int)idx & ((1 << LU) - 1);
    const int tok = (int)((uint32_t)th / (uint32_t)c.Hkv), g = (int)th - tok * c.Hkv;
    const int b = SLOTS ? 0 : (int)((uint32_t)tok / (uint32_t)M), m = tok - b * M;
    float kv[8], vv[8];
    mxq::load8<SRC>(k, (int64_t)tok * ldk + g * D, 8 * u, D, vec & 1, kv);
    mxq::load8<SRC>(v, (int64_t)tok * ldv + g * D, 8 * u, D, vec & 2, vv);
    int64_t row;
    if constexpr (SLOTS) row = row_of_slot(c, slots[tok], g);
    else row = row_of(c, dpos, b, m, g);
    uint32_t kc, vc;
    const uint32_t kp = mxq::quantize8<SRC, 0>(kv, kc), vp = mxq::quantize8<SRC, 0>(vv, vc);
    if (row < 0) return;
    *reinterpret_cast<uint32_t*>(c.kq + row * (D / 2) + 4 * u) = kp;
    *reinterpret_cast<uint32_t*>(c.vq + row * (D / 2) + 4 * u) = vp;
    if ((u & 3) == 0) {
        c.ks[row * (D / 32) + (u >> 2)] = (uint8_t)kc;
        c.vs[row * (D / 32) + (u >> 2)] = (uint8_t)vc;
    }
}

// Eight values of one nibble word as DST, 16 (32) bytes at p.
template <int DST>
__device__ __forceinline__ void store8(void* p, int64_t at, uint32_t w, float s) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef float f4 __attribute__((ext_vector_type(4)));
    if constexpr (DST == MXFP4_DT_BF16) {
        const uint4 e = kv4::eight_bf16(w, s);
        __builtin_nontemporal_store((u4{e.x, e.y, e.z, e.w}), reinterpret_cast<u4*>(static_cast<uint16_t*>(p) + at));
    } else {
        const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
        const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
        if constexpr (DST == MXFP4_DT_F32) {
            float* o = static_cast<float*>(p) + at;
            __builtin_nontemporal_store((f4{a[0], a[1], b[0], b[1]}), reinterpret_cast<f4*>(o));
            __builtin_nontemporal_store((f4{d[0], d[1], e[0], e[1]}), reinterpret_cast<f4*>(o + 4));
        } else {
            typedef _Float16 h8 __attribute__((ext_vector_type(8)));
            __builtin_nontemporal_store((h8{(_Float16)a[0], (_Float16)a[1], (_Float16)b[0], (_Float16)b[1], (_Float16)d[0],
                                            (_Float16)d[1], (_Float16)e[0], (_Float16)e[1]}),
                                        reinterpret_cast<h8*>(static_cast<_Float16*>(p) + at));
        }
    }
}

template <int DST, int LU>
__global__ __launch_bounds__(256) void kv4_read_kernel(Cache c, const int32_t* __restrict__ start, void* __restrict__ k,
                                                       void* __restrict__ v, int n, int64_t heads) {
    constexpr int D = 8 << LU;
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t th = idx >> LU;
    if (th >= heads) return;
    const int u = (int)idx & ((1 << LU) - 1);
    const int tok = (int)((uint32_t)th / (uint32_t)c.Hkv), g = (int)th - tok * c.Hkv;
    const int b = (int)((uint32_t)tok / (uint32_t)n), m = tok - b * n;
    const int64_t row = row_of(c, start, b, m, g);
    uint32_t kw = 0, vw = 0, kc = 127, vc = 127;   // zeros where there is no row
    if (row >= 0) {
        kw = *reinterpret_cast<const uint32_t*>(c.kq + row * (D / 2) + 4 * u);
        vw = *reinterpret_cast<const uint32_t*>(c.vq + row * (D / 2) + 4 * u);
        kc = c.ks[row * (D / 32) + (u >> 2)];
        vc = c.vs[row * (D / 32) + (u >> 2)];
    }
    store8<DST>(k, idx * 8, kw, kv4::scale_of(kc));
    store8<DST>(v, idx * 8, vw, kv4::scale_of(vc));
}

// One wave per head of a token: lane l has elements l and l + 64, so a 32-block
// is half a wave's a (blocks 0, 1) or b (2, 3).
constexpr int kD = 128;

__device__ __forceinline__ void half_wave_block(float x, uint8_t* q, uint8_t* s) {
    const int lane = threadIdx.x & 63;
    float am = mx::row16_reduce<true>(__builtin_fabsf(x));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(am), __float_as_uint(am), false, false);
    am = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const uint32_t code = mx::e8m0_code(am);
    uint32_t n = mx::e2m1_code(x * mx::e8m0_inv_scale(code));
    n |= (uint32_t)mx::dpp<mx::kDppQuadNext1>((int)n) << 4;    // even lanes: two nibbles
    n |= (uint32_t)mx::dpp<mx::kDppQuadNext2>((int)n) << 8;    // lane 4j: four
    if (q) {
        if ((lane & 3) == 0) *reinterpret_cast<uint16_t*>(q + lane / 2) = (uint16_t)n;
        if ((lane & 31) == 0) s[lane / 32] = (uint8_t)code;
    }
}

__global__ __launch_bounds__(256) void qk_rope_kv4_kernel(const float* __restrict__ qkv, const uint16_t* __restrict__ qw,
                                                          const uint16_t* __restrict__ kw, float eps, float theta,
                                                          const int32_t* __restrict__ dpos, int M, int Hq,
                                                          uint16_t* __restrict__ q_out, Cache c) {
    const int tok = blockIdx.x, b = tok / M, m = tok - b * M;
    const int lane = threadIdx.x & 63;
    const int nh = Hq + 2 * c.Hkv;
    const int h = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
    if (h >= nh) return;
    const float* row = qkv + ((int64_t)tok * nh + h) * kD;
    const float a = row[lane], bb = row[lane + 64];
    uint16_t ra, rb;
    if (h < Hq + c.Hkv) {
        const uint16_t* nw = h < Hq ? qw : kw;
        hr::norm_rope(a, bb, mx::bf16_to_f32(nw[lane]), mx::bf16_to_f32(nw[lane + 64]), eps,
                      hr::rope_cs(theta, lane, dpos[b] + m), ra, rb);
        if (h < Hq) {
            uint16_t* dst = q_out + ((int64_t)tok * Hq + h) * kD;
            dst[lane] = ra;
            dst[lane + 64] = rb;
            return;
        }
    } else {
        ra = mx::f32_to_bf16_rne(a);
        rb = mx::f32_to_bf16_rne(bb);
    }
    const bool is_v = h >= Hq + c.Hkv;
    const int64_t r = row_of(c, dpos, b, m, h - Hq - (is_v ? c.Hkv : 0));
    if (r < 0) return;
    uint8_t* q = (is_v ? c.vq : c.kq) + r * (kD / 2);
    uint8_t* s = (is_v ? c.vs : c.ks) + r * (kD / 32);
    half_wave_block(mx::bf16_to_f32(ra), q, s);
    half_wave_block(mx::bf16_to_f32(rb), q + 32, s + 2);
}

constexpr int64_t kMostGroups = (1ll << 24) - 1;   // workgroups of 256 threads in one dimension of a launch, whose threads are counted in 32 bits

// T head rows of D values in threads of eight: the grid, or 0 if it is too large.
unsigned grid_of(int64_t heads, int D) {
    const int64_t g = (heads * (D / 8) + 255) / 256;
    return heads < (1ll << 31) && g <= kMostGroups ? (unsigned)g : 0u;
}

}  // namespace

namespace {

// kv4_write's checks of k and v, and its launch: B * M tokens.
template <bool SLOTS>
int write_rows(const char* what, const Cache& c, const void* k, const void* v, int src_dtype, int64_t ldk, int64_t ldv,
               const int32_t* dpos, const int64_t* slots, int64_t tokens, int M, int D, hipStream_t st) {
    MXH_REQUIRE(src_dtype >= MXFP4_DT_BF16 && src_dtype <= MXFP4_DT_F32, "%s: bad dtype %d", what, src_dtype);
    MXH_REQUIRE(ldk >= (int64_t)c.Hkv * D && ldv >= (int64_t)c.Hkv * D, "%s: token stride below Hkv*D=%lld", what,
                (long long)c.Hkv * D);
    const int64_t heads = tokens * c.Hkv;
    const unsigned grid = grid_of(heads, D);
    MXH_REQUIRE(grid > 0, "%s: %lld head rows: too large", what, (long long)heads);
    const int esz = src_dtype == MXFP4_DT_F32 ? 4 : 2;
    auto wide = [&](const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld * esz % 16 == 0; };
    const int vec = (wide(k, ldk) ? 1 : 0) | (wide(v, ldv) ? 2 : 0);
#define MXH_KV4W(SRC)                                                                                                            \
    if (D == 64)                                                                                                                 \
        hipLaunchKernelGGL((kv4_write_kernel<SRC, 3, SLOTS>), dim3(grid), dim3(256), 0, st, k, v, ldk, ldv, vec, c, dpos, slots, M, heads); \
    else                                                                                                                         \
        hipLaunchKernelGGL((kv4_write_kernel<SRC, 4, SLOTS>), dim3(grid), dim3(256), 0, st, k, v, ldk, ldv, vec, c, dpos, slots, M, heads)
    switch (src_dtype) {
        case MXFP4_DT_BF16: MXH_KV4W(MXFP4_DT_BF16); break;
        case MXFP4_DT_F16: MXH_KV4W(MXFP4_DT_F16); break;
        default: MXH_KV4W(MXFP4_DT_F32); break;
    }
#undef MXH_KV4W
    return mxh::launch_status(what);
}

}  // namespace

extern "C" int mxfp4_kv4_write(const void* k, const void* v, int src_dtype, int64_t ldk, int64_t ldv, uint8_t* kq, uint8_t* ks,
                               uint8_t* vq, uint8_t* vs, const int32_t* pages, int n_pages, int page, int max_pages,
                               const int32_t* dpos, int B, int M, int Hkv, int D, void* stream) {
    Cache c;
    const int rc = kv4::make_cache(c, "kv4_write", kq, ks, vq, vs, pages, n_pages, page, max_pages, B, Hkv, D);
    if (rc != MXFP4_OK) return rc;
    MXH_REQUIRE(k && v && dpos, "kv4_write: null pointer");
    MXH_REQUIRE(M > 0, "kv4_write: M=%d", M);
    return write_rows<false>("kv4_write", c, k, v, src_dtype, ldk, ldv, dpos, nullptr, (int64_t)B * M, M, D, mxh::as_stream(stream));
}

extern "C" int mxfp4_kv4_write_slots(const void* k, const void* v, int src_dtype, int64_t ldk, int64_t ldv, uint8_t* kq,
                                     uint8_t* ks, uint8_t* vq, uint8_t* vs, int n_pages, int page, const int64_t* slots, int T,
                                     int Hkv, int D, void* stream) {
    Cache c;
    const int rc = kv4::make_cache(c, "kv4_write_slots", kq, ks, vq, vs, nullptr, n_pages, page, 0, 1, Hkv, D);
    if (rc != MXFP4_OK) return rc;
    MXH_REQUIRE(k && v && slots, "kv4_write_slots: null pointer");
    MXH_REQUIRE(T > 0, "kv4_write_slots: T=%d", T);
    return write_rows<true>("kv4_write_slots", c, k, v, src_dtype, ldk, ldv, nullptr, slots, T, 1, D, mxh::as_stream(stream));
}

extern "C" int mxfp4_kv4_read(const uint8_t* kq, const uint8_t* ks, const uint8_t* vq, const uint8_t* vs, const int32_t* pages,
                              int n_pages, int page, int max_pages, const int32_t* start, void* k, void* v, int dst_dtype,
                              int B, int n, int Hkv, int D, void* stream) {
    Cache c;
    const int rc = kv4::make_cache(c, "kv4_read", kq, ks, vq, vs, pages, n_pages, page, max_pages, B, Hkv, D);
    if (rc != MXFP4_OK) return rc;
    MXH_REQUIRE(k && v, "kv4_read: null pointer");
    MXH_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "kv4_read: outputs must be 16-byte aligned");
    MXH_REQUIRE(dst_dtype >= MXFP4_DT_BF16 && dst_dtype <= MXFP4_DT_F32, "kv4_read: bad dtype %d", dst_dtype);
    MXH_REQUIRE(n > 0, "kv4_read: n=%d", n);
    const int64_t heads = (int64_t)B * n * Hkv;
    const unsigned grid = grid_of(heads, D);
    MXH_REQUIRE(grid > 0, "kv4_read: B*n*Hkv=%lld too large", (long long)heads);
    const hipStream_t st = mxh::as_stream(stream);
#define MXH_KV4R(DST)                                                                                                \
    if (D == 64) hipLaunchKernelGGL((kv4_read_kernel<DST, 3>), dim3(grid), dim3(256), 0, st, c, start, k, v, n, heads); \
    else hipLaunchKernelGGL((kv4_read_kernel<DST, 4>), dim3(grid), dim3(256), 0, st, c, start, k, v, n, heads)
    switch (dst_dtype) {
        case MXFP4_DT_BF16: MXH_KV4R(MXFP4_DT_BF16); break;
        case MXFP4_DT_F16: MXH_KV4R(MXFP4_DT_F16); break;
        default: MXH_KV4R(MXFP4_DT_F32); break;
    }
#undef MXH_KV4R
    return mxh::launch_status("kv4_read");
}

extern "C" int mxfp4_qk_norm_rope_kv4(const float* qkv, const void* q_norm_w, const void* k_norm_w, float eps, float theta,
                                      uint8_t* kq, uint8_t* ks, uint8_t* vq, uint8_t* vs, const int32_t* pages, int n_pages,
                                      int page, int max_pages, const int32_t* dpos, int B, int M, int Hq, int Hkv, int D,
                                      void* q_out, void* stream) {
    Cache c;
    const int rc = kv4::make_cache(c, "qk_norm_rope_kv4", kq, ks, vq, vs, pages, n_pages, page, max_pages, B, Hkv, D);
    if (rc != MXFP4_OK) return rc;
    MXH_REQUIRE(qkv && q_norm_w && k_norm_w && dpos && q_out, "qk_norm_rope_kv4: null pointer");
    MXH_REQUIRE(D == kD, "qk_norm_rope_kv4: D=%d (%d)", D, kD);
    MXH_REQUIRE(M > 0 && Hq > 0 && Hq % Hkv == 0 && (int64_t)B * M <= kMostGroups, "qk_norm_rope_kv4: B=%d M=%d Hq=%d Hkv=%d", B, M,
                Hq, Hkv);
    const int64_t nh = (int64_t)Hq + 2 * Hkv;
    MXH_REQUIRE(nh <= 4 * 65535, "qk_norm_rope_kv4: Hq=%d Hkv=%d", Hq, Hkv);
    hipLaunchKernelGGL(qk_rope_kv4_kernel, dim3(B * M, (unsigned)(nh + 3) / 4), dim3(256), 0, mxh::as_stream(stream), qkv,
                       static_cast<const uint16_t*>(q_norm_w), static_cast<const uint16_t*>(k_norm_w), eps, theta, dpos, M, Hq,
                       static_cast<uint16_t*>(q_out), c);
    return mxh::launch_status("qk_norm_rope_kv4");
}
