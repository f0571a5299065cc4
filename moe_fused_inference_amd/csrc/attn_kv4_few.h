// attn_kv4_few.h -- the kernel of attention over the MXFP4 KV cache for up to 16 query rows
// of a kv head (attn_kv4.hip has its contract, mathematics and figures), without masks
// (attn_kv4.hip) and with (attn_kv4_window.hip, attn_kv4_tree.hip, attn_kv4_tree_window.hip).
#pragma once
#include "attn_kv4.h"
#include "kv4.h"
#include "mx_device.h"
#include "mx_host.h"

#include <type_traits>

namespace {

using namespace mxa;

constexpr int kParts = 3;              // bf16 parts of a probability

// A unit's bytes as a lane loads them.  K: row 16 t + l16, D/8 bytes from D/8 lq on
// (so its dimensions are D/4 lq .., one block's or half a block's) and their code.
// V: positions 16 t + 4 lq + i, columns D/16 l16 ..; a position's codes as one word.
template <int D>
struct Raw {
    typedef uint32_t vec __attribute__((ext_vector_type(D / 32)));
    vec k[2];
    uint32_t ks[2];
    uint32_t v[8];
    vec vs[2];      // four positions' codes
};

// Lane offsets into a tile's rows, in bytes.
template <int D>
struct Lane {
    uint32_t k, ks, v, vs;
    __device__ __forceinline__ explicit Lane(int lane) {
        const int l16 = lane & 15, lq = lane >> 4;
        k = l16 * (D / 2) + lq * (D / 8);
        ks = l16 * (D / 32) + (D == 128 ? lq : lq >> 1);
        v = 4 * lq * (D / 2) + l16 * (D / 32);
        vs = 4 * lq * (D / 32);
    }
};

// row[t]: tile t's first head row (uniform).  STREAM: K does not stay in the caches, and so leaves them to what does (kMuch).
template <bool STREAM, int D>
__device__ __forceinline__ void load_k(Raw<D>& r, const Cache& c, const uint32_t (&row)[2], const Lane<D>& o) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const auto p = reinterpret_cast<const typename Raw<D>::vec*>(c.kq + (uint64_t)row[t] * (D / 2) + o.k);
        r.k[t] = STREAM ? __builtin_nontemporal_load(p) : *p;
        r.ks[t] = *(c.ks + (uint64_t)row[t] * (D / 32) + o.ks);
    }
}
template <int D>
__device__ __forceinline__ void load_v(Raw<D>& r, const Cache& c, const uint32_t (&row)[2], const Lane<D>& o) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint8_t* p = c.vq + (uint64_t)row[t] * (D / 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (D == 128) r.v[4 * t + i] = *reinterpret_cast<const uint32_t*>(p + (o.v + i * (D / 2)));
            else r.v[4 * t + i] = *reinterpret_cast<const uint16_t*>(p + (o.v + i * (D / 2)));
        }
        r.vs[t] = *reinterpret_cast<const typename Raw<D>::vec*>(c.vs + (uint64_t)row[t] * (D / 32) + o.vs);
    }
}

// The scales of the lane's eight V positions, for the packed conversions, which read
// the exponent field alone: the code rotated there, its neighbours around it.
template <int D>
__device__ __forceinline__ void v_scales(const Raw<D>& r, float (&s)[8]) {
    const int l16 = threadIdx.x & 15;
    const uint32_t turn = (D == 128 ? 8 * (l16 >> 2) : 8 * (l16 >> 3)) + 9;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t w = D == 128 ? r.vs[i >> 2][i & 3] : r.vs[i >> 2][(i & 3) >> 1];
        s[i] = __uint_as_float(__builtin_amdgcn_alignbit(w, w, D == 64 && (i & 1) ? turn + 16 : turn));
    }
}
// The values of a word under one scale that bf16 does not hold are taken out of it.
__device__ __forceinline__ void take_out(uint32_t& w, float& scale) {
    const uint32_t code = __float_as_uint(scale) >> 23 & 255u;
    w &= ~(15u * kv4::not_finite(w, code));
    if (code == 255u) scale = 1.0f;
}
// MFMA operands of four column tiles: columns D/16 l16 + 4 H + c x the lane's eight positions.
template <int H>
__device__ __forceinline__ void decode_v(const uint32_t (&v)[8], const float (&s)[8], uint4 (&vd)[4]) {
    uint32_t o[4][4];
#pragma unroll
    for (int p2 = 0; p2 < 4; ++p2) {       // positions 2 p2, 2 p2 + 1
        const uint32_t a0 = kv4::pair_bf16<2 * H>(v[2 * p2], s[2 * p2]), a1 = kv4::pair_bf16<2 * H + 1>(v[2 * p2], s[2 * p2]);
        const uint32_t b0 = kv4::pair_bf16<2 * H>(v[2 * p2 + 1], s[2 * p2 + 1]), b1 = kv4::pair_bf16<2 * H + 1>(v[2 * p2 + 1], s[2 * p2 + 1]);
        o[0][p2] = __builtin_amdgcn_perm(b0, a0, 0x05040100u);
        o[1][p2] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
        o[2][p2] = __builtin_amdgcn_perm(b1, a1, 0x05040100u);
        o[3][p2] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) vd[c] = make_uint4(o[c][0], o[c][1], o[c][2], o[c][3]);
}

template <int D, int NQ, Work W, int NW, bool STREAM, int MASKS>
__global__ __launch_bounds__(64 * NW, 4) void attn_kv4_kernel(Args a) {
    constexpr bool ONE = W == Work::kSequence, WINDOW = MASKS & kWindow, TREE = MASKS & kTree;
    constexpr int R = 16, KT = D / 32, CT = D / 16;
    // q, and after the last unit the waves' sums
    __shared__ union Lds {
        alignas(16) uint16_t qs[NQ * R][D + 8];
        alignas(16) float mo[NW][16][D + 4];
    } lds;
    auto& qs = lds.qs;
    auto& mo = lds.mo;
    __shared__ float mm[NW][16], ml[NW][16];
    const int g = blockIdx.y, G = a.G, rows = a.M * G;     // at most 16
    auto segment = [&](int b, int base, int u0, int u1) {
        int tid = threadIdx.x;
        if constexpr (W == Work::kLine) asm volatile("" : "+v"(tid));   // (a lane's constants are made again for each segment, not held)
        const int lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int l16 = lane & 15, lq = lane >> 4;
        // q, whose parts go to LDS once the first units' loads are on their way.  Rows past the last load nothing: with the last
        // row's in their place 32 sequences of up to 32768 positions took 60.4 us where it took 58.2 on the same card (cards differ: 55 to 58).
        const uint16_t* qb = a.q + (int64_t)b * a.M * a.ldq + (int64_t)g * G * D;
        constexpr int NT = 64 * NW, QN = (R * (D / 8) + NT - 1) / NT;
        uint4 qw[QN];
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int r = (tid + NT * i) / (D / 8), ch = (tid + NT * i) % (D / 8), t = a.token(r);
            qw[i] = make_uint4(0, 0, 0, 0);
            if (r < rows && (R * (D / 8) % NT == 0 || tid + NT * i < R * (D / 8)))
                qw[i] = *reinterpret_cast<const uint4*>(qb + (int64_t)t * a.ldq + (r - t * G) * D + 8 * ch);
        }
        // the first head rows of the wave's units u0 + wave + NW j, j = lane, tiles 0 and 1 (kv4::kNoRow: there is no such tile)
        uint32_t first[2];
        Units un{};      // (WINDOW)
        auto find_rows = [&](int j0) {
            int64_t u = (int64_t)u0 + wave + NW * (j0 + lane);
            if constexpr (WINDOW) u += u < un.sinks ? 0 : un.gap;
            kv4::unit_rows(a.c, b, g, u * kUnit, true, first);
        };
        const Lane<D> off(lane);
        // the wave's j-th unit: its tiles' rows, and which of them exist
        auto locate = [&](int j, uint32_t (&row)[2]) -> int {
            const uint32_t r0 = __builtin_amdgcn_readlane(first[0], j & 63), r1 = __builtin_amdgcn_readlane(first[1], j & 63);
            row[0] = r0 == kv4::kNoRow ? 0 : r0;
            row[1] = r1 == kv4::kNoRow ? 0 : r1;
            return (r0 == kv4::kNoRow ? 0 : 1) | (r1 == kv4::kNoRow ? 0 : 2);
        };
        Raw<D> r;
        int there = 0;
        auto first_loads = [&]() {
            uint32_t row[2];
            find_rows(0);
            there = locate(0, row);
            load_k<STREAM>(r, a.c, row, off);
            load_v(r, a.c, row, off);
        };
        if constexpr (W == Work::kShare && !WINDOW) first_loads();        // of a share of fixed length before dpos is there: what no token sees is masked
        base = __builtin_amdgcn_readfirstlane(base);
        // Positions fit 31 bits: a token before the cache is put at -1, one past it at its end
        auto clamped = [&](int64_t pos) { return (int)(pos < 0 ? -1 : pos < a.c.max_pos ? pos : a.c.max_pos); };
        const int last = min(clamped((int64_t)base + a.M - 1), a.c.max_pos - 1);      // positions past it are no one's
        int lim_min = clamped(base);                                  // the first token sees up to here
        if constexpr (TREE) lim_min = clamped((int64_t)base - 1);     // (and of the drafts its own line)
        // (WINDOW) where the first and the last window begin, and units that some row does not see whole
        int begin_min = 0, begin_max = 0;
        if constexpr (WINDOW) {
            un = units<MASKS>(a, base);
            begin_min = first_begin<MASKS>(a, base, 0);
            begin_max = last_begin<MASKS>(a, base, a.M - 1);
            u1 = min(u1, (int)un.n);
        } else {
            u1 = min(u1, (last + kUnit) / kUnit);
        }
        auto some_hide = [&](int p0) { return p0 + kUnit - 1 > lim_min || (WINDOW && p0 < begin_max && p0 + kUnit > a.sinks); };
        if constexpr (W == Work::kShare && !WINDOW) {
            if (u0 >= u1) return;                               // no record: the merge reads none
        } else {
            if (W == Work::kShare && u0 >= u1) return;
            if (u0 + wave < u1) first_loads();
        }
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int r = (tid + NT * i) / (D / 8), ch = (tid + NT * i) % (D / 8);
            uint4 p[NQ];
            q_parts<NQ>(qw[i], p);
#pragma unroll
            for (int j = 0; j < NQ; ++j)
                if (R * (D / 8) % NT == 0 || r < R) *reinterpret_cast<uint4*>(&qs[j * R + r][8 * ch]) = p[j];
        }
        __syncthreads();
        // 0, or NaN where the row holds an infinity or a NaN (then so is its output)
        float zero = 0.0f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) zero += not_finite(*reinterpret_cast<const uint4*>(&qs[l16][(D / 4) * lq + 8 * kt]));
        zero = over_lq<false>(zero);
        // the lane's query is row l16; rows that are none see everything and write nothing
        const int lim = l16 < rows ? clamped(last_seen<MASKS>(a, base, a.token(l16))) : 1 << 30;
        int begin = 0;
        if constexpr (WINDOW) begin = l16 < rows ? begin_of<MASKS>(a, b, base, a.token(l16)) : 0;
        float m = kNone, l = 0.0f;
        bool wide = false;   // uniform: a row's reference is past kWide
        mx::v4f acc[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[c] = mx::v4f{0.f, 0.f, 0.f, 0.f};
        int dirty = 0;       // uniform: values that are not finite were taken out, among positions that not all rows see
        // Unit u, the wave's j-th.  `more`: the wave's next one is loaded meanwhile (decided in the code, not by a branch:
        // behind one the compiler waits for the older loads as if these had not been issued, that is for all)
        auto unit = [&](int u, int j, auto more_) {
            constexpr bool more = decltype(more_)::value;
            const int p0 = (WINDOW ? (int)un.real(u) : u) * kUnit;
            uint32_t next[2];
            int there_next = 0;
            if constexpr (more) {
                if (((j + 1) & 63) == 0) find_rows(j + 1);
                there_next = locate(j + 1, next);
            }
            mx::v4f sv[2];
            sv[0] = sv[1] = mx::v4f{zero, zero, zero, zero};
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                uint4 qf[NQ];
#pragma unroll
                for (int n = 0; n < NQ; ++n) qf[n] = *reinterpret_cast<const uint4*>(&qs[n * R + l16][(D / 4) * lq + 8 * kt]);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint4 kd = kv4::eight_bf16(r.k[t][kt], kv4::scale_of(r.ks[t]));
#pragma unroll
                    for (int n = 0; n < NQ; ++n) sv[t] = mfma_bf16(kd, qf[n], sv[t]);
                }
            }
            if constexpr (more) load_k<STREAM>(r, a.c, next, off);
            // sv[t][i], s[4 t + i]: position p0 + 16 t + 4 lq + i
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = sv[i >> 2][i & 3];
            const bool masked = __builtin_amdgcn_readfirstlane(some_hide(p0) || there != 3);
            if (masked) {
                int sees = lim - p0 - 4 * lq;        // the last position that the lane's query sees
                asm volatile("" : "+v"(sees));       // (nothing below is computed ahead of the branch)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!(there >> (i >> 2) & 1) || 16 * (i >> 2) + (i & 3) > sees) s[i] = -INFINITY;
                if constexpr (WINDOW) {
                    const int from = begin - p0 - 4 * lq, sinks = a.sinks - p0 - 4 * lq;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int at = 16 * (i >> 2) + (i & 3);
                        if (at < from && at >= sinks) s[i] = -INFINITY;
                    }
                }
                if constexpr (TREE) {
                    const uint32_t bits = tree_bits(a, b, base, min(a.token(l16), a.M - 1), p0) >> (4 * lq);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!(bits >> (16 * (i >> 2) + (i & 3)) & 1)) s[i] = -INFINITY;
                }
            }
            uint4 p[1][kParts];
            float t[8], sum;
            terms(s, a.scale, m, wide, t, sum);
            parts(t, p);
            again(s, a.scale, m, l, wide, sum, p, [](float x) { return over_lq<true>(x); },
                  [&](float al) {
#pragma unroll
                      for (int c = 0; c < CT; ++c)
#pragma unroll
                          for (int i = 0; i < 4; ++i) acc[c][i] *= al;
                  });
            __builtin_amdgcn_sched_barrier(0);   // 128 registers, four waves a SIMD: no operand of the second product before here,
            float vs[8];
            v_scales(r, vs);
            if (masked) {
                // rows past the last token, and of no page, may hold anything: 0 * NaN must not reach a sum
                int sees = last - p0 - 4 * lq;
                asm volatile("" : "+v"(sees));
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!(there >> (i >> 2) & 1) || 16 * (i >> 2) + (i & 3) > sees) {
                        r.v[i] = 0;
                        vs[i] = 1.0f;
                    }
                if constexpr (WINDOW) {      // or before the first window
                    const int from = begin_min - p0 - 4 * lq, sinks = a.sinks - p0 - 4 * lq;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int at = 16 * (i >> 2) + (i & 3);
                        if (at < from && at >= sinks) {
                            r.v[i] = 0;
                            vs[i] = 1.0f;
                        }
                    }
                }
                // nor may what only some rows see reach the others'
                if (WINDOW ? (lim_min < last || begin_min < begin_max) && some_hide(p0) : p0 + kUnit - 1 > lim_min && lim_min < last) {
                    uint32_t large = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) large = max(large, __float_as_uint(vs[i]) & 0x7F800000u);
                    if (__ballot(large >= kv4::kLargeScale)) {
                        dirty = 1;
#pragma unroll
                        for (int i = 0; i < 8; ++i) take_out(r.v[i], vs[i]);
                    }
                }
            }
            auto product = [&](auto half) {
                constexpr int H = decltype(half)::value;
                uint4 vd[4];
                decode_v<H>(r.v, vs, vd);
                if constexpr (H == CT / 4 - 1 && more) load_v(r, a.c, next, off);
#pragma unroll
                for (int k = kParts - 1; k >= 0; --k)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[4 * H + c] = mfma_bf16(vd[c], p[0][k], acc[4 * H + c]);
            };
            product(std::integral_constant<int, 0>{});
            __builtin_amdgcn_sched_barrier(0);   // and one half's at a time
            if constexpr (CT == 8) product(std::integral_constant<int, 1>{});
            there = there_next;
        };
        int u = u0 + wave, j = 0;
        for (; u + NW < u1; u += NW, ++j) unit(u, j, std::true_type{});
        if (u < u1) unit(u, j, std::false_type{});
        // the waves' sums in LDS, then one record (or the output) per row: acc[c][i] is
        // column D/16 (4 lq + i) + c of query l16
        __syncthreads();
        const float ls = over_lq<false>(l);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < CT; c += 4)
                *reinterpret_cast<float4*>(&mo[wave][l16][CT * (4 * lq + i) + c]) = make_float4(acc[c][i], acc[c + 1][i], acc[c + 2][i], acc[c + 3][i]);
        if (lq == 0) {
            mm[wave][l16] = m;
            ml[wave][l16] = ls;
        }
        if (__builtin_amdgcn_readfirstlane(dirty)) {
            if constexpr (MASKS != 0)
                mark_not_finite_masked<D, NW, MASKS>(a, b, base, g, 0, rows, wave, u1 - u0, last, [&](int k) { return WINDOW ? (int)un.real(u0 + k) : u0 + k; }, some_hide, mo[wave]);
            else
                mark_not_finite<D, NW>(a, b, base, g, 0, rows, wave, u0, u1, lim_min, last, mo[wave]);
        }
        __syncthreads();
        // thread: CT columns of a row (8 of 128, 4 of 64)
        const int qr = tid >> 4;
        if (tid < 256 && qr < rows) finish<D, NW, ONE, MASKS>(a, tid, b, base, g, qr, u0, [&](int w) { return mm[w][qr]; }, [&](int w) { return ml[w][qr]; }, [&](int w, int c) { return *reinterpret_cast<const float4*>(&mo[w][qr][c]); });
    };
    each_segment<W, MASKS>(a, segment);
}

template <int MASKS>
int launch_few(const Args& a, int q_dtype, const Plan& p, int D, bool much, hipStream_t st) {
    const dim3 grid(p.shares, a.c.Hkv);
#define MXH_W4(DD, QQ, W)                                                                                          \
    if (much) hipLaunchKernelGGL((attn_kv4_kernel<DD, QQ, Work::W, 4, true, MASKS>), grid, dim3(256), 0, st, a);  \
    else hipLaunchKernelGGL((attn_kv4_kernel<DD, QQ, Work::W, 4, false, MASKS>), grid, dim3(256), 0, st, a)
#define MXH_K4(DD, QQ)                                                                                                   \
    if (p.waves == 16)                                                                                                   \
        hipLaunchKernelGGL((attn_kv4_kernel<DD, QQ, Work::kSequence, 16, false, MASKS>), grid, dim3(1024), 0, st, a);   \
    else if (p.one) { MXH_W4(DD, QQ, kSequence); }                                                                       \
    else if (a.B == 1) { MXH_W4(DD, QQ, kShare); }                                                                       \
    else { MXH_W4(DD, QQ, kLine); }
    if (D == 64) {
        if (q_dtype == MXFP4_DT_BF16) { MXH_K4(64, 1); } else { MXH_K4(64, 2); }
    } else {
        if (q_dtype == MXFP4_DT_BF16) { MXH_K4(128, 1); } else { MXH_K4(128, 2); }
    }
#undef MXH_K4
#undef MXH_W4
    return mxh::launch_status("attn_kv4 (shares)");
}

}  // namespace
