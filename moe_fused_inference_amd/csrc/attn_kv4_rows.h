// attn_kv4_rows.h -- attention over the MXFP4 KV cache for more than 16 query rows of
// a kv head (drafts of many tokens, pieces of a prompt): attn_kv4.hip's contract, shares
// and mathematics, on 32 x 32 MFMAs.
//
// Workgroup (share or sequence, kv head g, group of 32 rows): four waves, each with all
// of the group's rows and every fourth unit of 32 positions, its own running softmax and
// no barrier until their sums meet in LDS.
//
// What bounds it is instruction issue: next to MFMAs a vector instruction takes 4 cycles
// of a SIMD whatever it is, and a 16 x 16 MFMA about 9 of its 16 besides, a 32 x 32 one
// of twice the work hardly any (two waves of each, 64 k MFMAs and 256 k vector
// instructions a SIMD: 741 us with 16 x 16, 1049 with 32 x 32 against 944 for those
// alone).  So the larger shape.  A piece of 512 tokens over 8192 positions (32 / 4 heads
// of 128), us, of the first form of this kernel: loads and conversions alone 62, with
// both products 123, with the softmax 152 (16 x 16 MFMAs: 134, two 32-row tiles a wave:
// 203, they spill).  Then 122 by:
//   - few and wide loads (a load holds the CU's address unit 16 cycles whatever its
//     width): 6 a unit instead of 23; V's rows and the codes are handed to their lanes
//     through the wave's own LDS, with no barrier;
//   - the software pipeline in `step`: unit j + 1's terms between unit j's products, unit
//     j + 2's scores after, K loaded two units ahead and V one;
//   - p in two bf16 parts where 8 or 11 bits go out (fp32 out: three, 137).
// And 114 with the scales spread once into LDS, 16 rotations a unit fewer (the same call
// 108 .. 119 from card to card): 560 to 620 TFLOP/s, 680 for 2048 tokens over 32768.
//
// Operands.  S^T: lane (l32, lh) has row l32 of the unit (a position) and dimensions
// D/2 lh + 8 kt .. of step kt; the product leaves it positions 8 (i / 4) + 4 lh + i % 4 of
// query l32.  O^T: columns D/32 l32 + c of tile c and just those positions, eight a step.
#pragma once
#include "attn_kv4.h"

#include <type_traits>

namespace {

using namespace mxa;

constexpr int kWaves = 4;

__device__ __forceinline__ mx::v16f mfma32(uint4 a, uint4 b, mx::v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// The maximum / sum over the two lanes l, l ^ 32.
template <bool MAX>
__device__ __forceinline__ float over_lh(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float x = __uint_as_float(r[0]), y = __uint_as_float(r[1]);
    return MAX ? fmaxf(x, y) : x + y;
}

// A wave's V nibbles and the scales, of two units in turn.  Row 8 h + 4 lh + i of a tile
// lies at 8 h + 2 i + lh, so that the two rows that a product's halves read at a time
// are neighbours.
template <int D>
struct Stage {
    alignas(16) uint8_t v[2][2][16][D / 2];
    alignas(16) float scale[2][64][D / 32];   // K's of the unit's 32 positions, then V's (scale_at: a lane reads a position's as it is used)
};

template <int D, int NQ, int NP, Work W, int MASKS>
__global__ __launch_bounds__(64 * kWaves, 2) void attn_kv4_rows_kernel(Args a) {
    constexpr bool ONE = W == Work::kSequence, WINDOW = MASKS & kWindow, TREE = MASKS & kTree;
    constexpr int R = 32, KT = D / 16, CT = D / 32;    // rows, steps of S, column tiles (and a lane's columns)
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    typedef uint32_t hvec __attribute__((ext_vector_type(D / 32)));
    // q's parts and the waves' stages, and after the last unit the waves' sums
    __shared__ union Lds {
        struct {
            alignas(16) uint16_t qs[NQ * R][D + 8];
            Stage<D> stage[kWaves];
        } in;
        alignas(16) float mo[kWaves][R][D + 4];
    } lds;
    __shared__ float mm[kWaves][R], ml[kWaves][R];
    const int g = blockIdx.y, r0 = blockIdx.z * R, G = a.G;
    const int rows = a.M * G;
    auto segment = [&](int b, int base, int u0, int u1) {
        int tid = threadIdx.x;
        if constexpr (W == Work::kLine) asm volatile("" : "+v"(tid));   // (a lane's constants are made again for each segment, not held)
        base = __builtin_amdgcn_readfirstlane(base);
        const int lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int l32 = lane & 31, lh = lane >> 5;
        // Positions fit 31 bits: a token before the cache is put at -1, one past it at its end
        auto clamped = [&](int64_t pos) { return (int)(pos < 0 ? -1 : pos < a.c.max_pos ? pos : a.c.max_pos); };
        const int last = min(clamped((int64_t)base + a.M - 1), a.c.max_pos - 1);      // positions past it are no one's
        int lim_min = __builtin_amdgcn_readfirstlane(clamped((int64_t)base + a.token(r0)));        // the group's first token sees up to here
        const int t1 = a.token(min(r0 + R, rows) - 1);                                           // its last token
        const int lim_max = __builtin_amdgcn_readfirstlane(min(clamped(last_seen<MASKS>(a, base, t1)), a.c.max_pos - 1));
        if constexpr (TREE) lim_min = __builtin_amdgcn_readfirstlane(clamped((int64_t)base - 1));     // (and of the drafts its own line)
        // (WINDOW) where the group's first and last window begin; its units: `head` of the sinks, then others
        int begin_min = 0, begin_max = 0, head = 0, tail = 0;
        if constexpr (WINDOW) {
            const Units un = units<MASKS>(a, base);
            begin_min = __builtin_amdgcn_readfirstlane(first_begin<MASKS>(a, base, a.token(r0)));
            begin_max = __builtin_amdgcn_readfirstlane(last_begin<MASKS>(a, base, t1));
            u1 = min(u1, lim_max < 0 ? 0 : min((int)un.n, (int)un.of_real(lim_max / kUnit) + 1));
            if (!ONE && u0 >= u1) return;                       // no row of the group sees the segment: no record
            const int from = max(u0, max((int)un.of_real(begin_min / kUnit), (int)un.sinks));
            head = max(0, min(u1, (int)un.sinks) - u0);
            tail = from - head + (int)un.gap;                   // unit k: u0 + k of the sinks, k + tail after them
            u1 = u0 + head + max(0, u1 - from);
        } else {
            u1 = min(u1, (lim_max + kUnit) / kUnit);
            if (!ONE && u0 >= u1) return;
        }
        auto real = [&](int k) { return WINDOW ? k + (k < head ? u0 : tail) : u0 + k; };     // the group's k-th unit
        auto some_hide = [&](int p0) { return p0 + kUnit - 1 > lim_min || (WINDOW && p0 < begin_max && p0 + kUnit > a.sinks); };
        const int n = u0 + wave < u1 ? (u1 - u0 - wave + kWaves - 1) / kWaves : 0;   // the wave's units: wave + 4 j
        // the first head rows of units j, j = lane, tiles 0 and 1 (kv4::kNoRow: there is no such tile)
        uint32_t first[2];
        auto find_rows = [&](int j0) {
            int64_t u = (int64_t)u0 + wave + kWaves * (j0 + lane);
            if constexpr (WINDOW) u += wave + kWaves * (j0 + lane) < head ? 0 : tail - u0;
            kv4::unit_rows(a.c, b, g, u * kUnit, j0 + lane < n, first);
        };
        struct Unit {
            uint32_t x, y;    // its tiles' first head rows
            int there, p0;    // which of them exist (none past the last unit), and its first position
        };
        auto locate = [&](int j) {
            if ((j & 63) == 0) find_rows(j);
            const uint32_t x = __builtin_amdgcn_readlane(first[0], j & 63), y = __builtin_amdgcn_readlane(first[1], j & 63);
            return Unit{x == kv4::kNoRow ? 0 : x, y == kv4::kNoRow ? 0 : y, (x == kv4::kNoRow ? 0 : 1) | (y == kv4::kNoRow ? 0 : 2), (WINDOW ? real(wave + kWaves * j) : u0 + wave + kWaves * j) * kUnit};
        };
        // a unit's bytes, in few and wide loads.  K: row l32, half lh; codes: those of K's (lane < 32) or V's position l32, one
        // word; V: D/8 bytes of row 16 t + lane / 4
        v4u rk[D / 64];
        hvec rv[2];
        uint32_t rcodes;
        const uint8_t* const codes_of = lane < 32 ? a.c.ks : a.c.vs;
        auto load_k = [&](const Unit& u) {
            const uint64_t at = (uint64_t)(l32 < 16 ? u.x : u.y) + (l32 & 15);
            const uint8_t* p = a.c.kq + at * (D / 2) + lh * (D / 4);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) rk[i] = *reinterpret_cast<const v4u*>(p + 16 * i);
            const uint8_t* s = codes_of + at * (D / 32);
            if constexpr (D == 128) rcodes = *reinterpret_cast<const uint32_t*>(s);
            else rcodes = *reinterpret_cast<const uint16_t*>(s);
        };
        auto load_v = [&](const Unit& u) {
            rv[0] = *reinterpret_cast<const hvec*>(a.c.vq + (uint64_t)u.x * (D / 2) + lane * (D / 8));
            rv[1] = *reinterpret_cast<const hvec*>(a.c.vq + (uint64_t)u.y * (D / 2) + lane * (D / 8));
        };
        Stage<D>& stage = lds.in.stage[wave];
        // rows past the last token, and of no page, may hold anything: 0 * NaN must not reach a sum
        auto ragged = [&](const Unit& u) {
            return __builtin_amdgcn_readfirstlane(u.there != 3 || u.p0 + kUnit - 1 > last || (WINDOW && u.p0 < begin_min && u.p0 + kUnit > a.sinks));
        };
        auto put_codes = [&](int j, const Unit& u) {
            if (ragged(u)) {
                int sees = last - u.p0;
                asm volatile("" : "+v"(sees));       // (nothing below is computed ahead of the branch)
                if (!(u.there >> (l32 >> 4) & 1) || l32 > sees) rcodes = 0x7F7F7F7Fu;
                if (WINDOW && u.p0 + l32 < begin_min && u.p0 + l32 >= a.sinks) rcodes = 0x7F7F7F7Fu;
            }
            typedef float svec __attribute__((ext_vector_type(D / 32)));
            svec x;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) x[i] = scale_at(rcodes, i);
            *reinterpret_cast<svec*>(stage.scale[j & 1][lane]) = x;
        };
        const int v_row = lane >> 2;                 // the lane's row of V in a tile
        int dirty = 0;       // uniform: values that are not finite were taken out, among positions that not all rows see
        const int all_see = min(lim_min, last);      // up to here
        auto put_v = [&](int j, const Unit& u) {
            const bool hide = WINDOW ? some_hide(u.p0) : u.p0 + kUnit - 1 > all_see;
            if (__builtin_amdgcn_readfirstlane(u.there != 3 || hide)) {
                int sees = last - u.p0;
                asm volatile("" : "+v"(sees));
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (!(u.there >> t & 1) || 16 * t + v_row > sees ||
                        (WINDOW && u.p0 + 16 * t + v_row < begin_min && u.p0 + 16 * t + v_row >= a.sinks))
                        rv[t] = 0;
                // nor may what only some rows see reach the others'
                float* scale[2];
                uint32_t large = 0;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    scale[t] = &stage.scale[j & 1][32 + 16 * t + v_row][D == 128 ? lane & 3 : (lane & 3) >> 1];
                    large = max(large, __float_as_uint(*scale[t]) & 0x7F800000u);
                }
                if (hide && __ballot(large >= kv4::kLargeScale)) {
                    dirty = 1;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const uint32_t code = __float_as_uint(*scale[t]) >> 23 & 255u;
                        if (code == 255u) *scale[t] = 1.0f;
#pragma unroll
                        for (int i = 0; i < D / 32; ++i) rv[t][i] &= ~(15u * kv4::not_finite(rv[t][i], code));
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
                *reinterpret_cast<hvec*>(&stage.v[j & 1][t][(v_row & 8) + 2 * (v_row & 3) + ((v_row >> 2) & 1)][(lane & 3) * (D / 8)]) = rv[t];
        };
        Unit ua = locate(0), ub = ua, uc = ua;
        load_k(ua);
        load_v(ua);
        // q (rows past the last are the last)
        constexpr int NT = 64 * kWaves, QN = (R * (D / 8) + NT - 1) / NT;
        uint4 qw[QN];
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int r = min(r0 + (tid + NT * i) / (D / 8), rows - 1), ch = (tid + NT * i) % (D / 8), t = a.token(r);
            qw[i] = *reinterpret_cast<const uint4*>(a.q + ((int64_t)b * a.M + t) * a.ldq + (int64_t)(g * G + r - t * G) * D + 8 * ch);
        }
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int r = (tid + NT * i) / (D / 8), ch = (tid + NT * i) % (D / 8);
            uint4 p[NQ];
            q_parts<NQ>(qw[i], p);
#pragma unroll
            for (int j = 0; j < NQ; ++j)
                if (R * (D / 8) % NT == 0 || r < R) *reinterpret_cast<uint4*>(&lds.in.qs[j * R + r][8 * ch]) = p[j];
        }
        __syncthreads();
        // the lane's query is row r0 + l32; rows that are none see everything and write nothing.
        // zero: 0, or NaN where the row holds an infinity or a NaN (then so is its output)
        const int lim = r0 + l32 < rows ? clamped(last_seen<MASKS>(a, base, a.token(r0 + l32))) : 1 << 30;
        int begin = 0;
        if constexpr (WINDOW) begin = r0 + l32 < rows ? begin_of<MASKS>(a, b, base, a.token(r0 + l32)) : 0;
        float zero = 0.0f, m = kNone, l = 0.0f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) zero += not_finite(*reinterpret_cast<const uint4*>(&lds.in.qs[l32][(D / 2) * lh + 8 * kt]));
        zero = over_lh<false>(zero);
        bool wide = false;
        mx::v16f acc[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[c][i] = 0.0f;

        // S^T of unit j, whose K is in rk
        auto scores = [&](int j, const Unit& u, float (&s)[16]) {
            put_codes(j, u);
            mx::v16f sv;
#pragma unroll
            for (int i = 0; i < 16; ++i) sv[i] = zero;
            float sc[KT / 4];
#pragma unroll
            for (int i = 0; i < KT / 4; ++i) sc[i] = stage.scale[j & 1][l32][KT / 4 * lh + i];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const uint4 kd = kv4::eight_bf16(rk[kt / 4][kt & 3], sc[kt >> 2]);
#pragma unroll
                for (int k = 0; k < NQ; ++k)
                    sv = mfma32(kd, *reinterpret_cast<const uint4*>(&lds.in.qs[k * R + l32][(D / 2) * lh + 8 * kt]), sv);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = sv[i];
        };
        auto masked = [&](const Unit& u, float (&s)[16]) {
            if (__builtin_amdgcn_readfirstlane(some_hide(u.p0) || u.there != 3)) {
                int sees = lim - u.p0 - 4 * lh;      // the last position that the lane's query sees
                asm volatile("" : "+v"(sees));
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(u.there >> (i >> 3) & 1) || 8 * (i >> 2) + (i & 3) > sees) s[i] = -INFINITY;
                if constexpr (WINDOW) {
                    const int from = begin - u.p0 - 4 * lh, sinks = a.sinks - u.p0 - 4 * lh;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int at = 8 * (i >> 2) + (i & 3);
                        if (at < from && at >= sinks) s[i] = -INFINITY;
                    }
                }
                if constexpr (TREE) {
                    const uint32_t bits = tree_bits(a, b, base, min(a.token(r0 + l32), a.M - 1), u.p0) >> (4 * lh);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!(bits >> (8 * (i >> 2) + (i & 3)) & 1)) s[i] = -INFINITY;
                }
            }
        };
        // O^T += V^T P^T of unit j
        auto products = [&](int j, const uint4 (&p)[2][NP]) {
#pragma unroll
            for (int st = 0; st < 2; ++st) {         // eight positions a step
                uint32_t v[8];
                float sc[8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint8_t* x = &stage.v[j & 1][st][8 * h + 2 * i + lh][l32 * (CT / 2)];
                        if constexpr (D == 128) v[4 * h + i] = *reinterpret_cast<const uint16_t*>(x);
                        else v[4 * h + i] = *x;
                        sc[4 * h + i] = stage.scale[j & 1][32 + 16 * st + 8 * h + 4 * lh + i][D == 128 ? l32 >> 3 : l32 >> 4];
                    }
                }
                uint32_t o[CT][4];
                auto columns = [&](auto pair_) {     // columns 2 P, 2 P + 1 of the lane's
                    constexpr int P = decltype(pair_)::value;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t x = kv4::pair_bf16<P>(v[2 * k], sc[2 * k]), y = kv4::pair_bf16<P>(v[2 * k + 1], sc[2 * k + 1]);
                        o[2 * P][k] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                        o[2 * P + 1][k] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                    }
                };
                columns(std::integral_constant<int, 0>{});
                if constexpr (D == 128) columns(std::integral_constant<int, 1>{});
#pragma unroll
                for (int k = NP - 1; k >= 0; --k)
#pragma unroll
                    for (int c = 0; c < CT; ++c) acc[c] = mfma32(make_uint4(o[c][0], o[c][1], o[c][2], o[c][3]), p[st][k], acc[c]);
            }
        };
        auto over = [](float x) { return over_lh<true>(x); };
        auto rescale = [&](float al) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c][i] *= al;
        };
        // A software pipeline, because a wave issues in order: while the matrix unit works on unit j's second product, the
        // vector unit makes unit j + 1's terms, and unit j + 2's scores come after.
        float s[16];
        uint4 pa[2][NP], pb[2][NP];
        auto step = [&](int j, const uint4 (&p)[2][NP], uint4 (&pn)[2][NP]) {     // unit j + 1 exists: ua is it, ub the one after
            masked(ua, s);
            float t[16], sum;
            terms(s, a.scale, m, wide, t, sum);
            parts(t, pn);
            products(j, p);
            again(s, a.scale, m, l, wide, sum, pn, over, rescale);
            put_v(j + 1, ua);
            load_v(ub);
            if (j + 2 < n) scores(j + 2, ub, s);
            load_k(uc);
            ua = ub;
            ub = uc;
            uc = locate(j + 4);
        };
        if (n > 0) {
            scores(0, ua, s);
            ub = locate(1);
            load_k(ub);
            put_v(0, ua);
            load_v(ub);
            masked(ua, s);
            first_terms(s, a.scale, m, l, wide, pa, over);
            ua = ub;
            ub = locate(2);
            if (n > 1) scores(1, ua, s);
            load_k(ub);
            uc = locate(3);
            int j = 0;
            for (; j + 2 < n; j += 2) {
                step(j, pa, pb);
                step(j + 1, pb, pa);
            }
            if (j + 1 < n) {
                step(j, pa, pb);
                products(j + 1, pb);
            } else {
                products(j, pa);
            }
        }
        // the waves' sums in LDS, then one record (or the output) per row: acc[c][i] is column
        // CT (8 (i / 4) + 4 lh + i % 4) + c of query l32
        __syncthreads();
        const float ls = over_lh<false>(l);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float* o = &lds.mo[wave][l32][CT * (8 * (i / 4) + 4 * lh + i % 4)];
            if constexpr (CT == 4) *reinterpret_cast<float4*>(o) = make_float4(acc[0][i], acc[1][i], acc[2][i], acc[3][i]);
            else *reinterpret_cast<float2*>(o) = make_float2(acc[0][i], acc[1][i]);
        }
        if (lh == 0) {
            mm[wave][l32] = m;
            ml[wave][l32] = ls;
        }
        if (__builtin_amdgcn_readfirstlane(dirty)) {
            if constexpr (MASKS != 0)
                mark_not_finite_masked<D, kWaves, MASKS>(a, b, base, g, r0, min(R, rows - r0), wave, u1 - u0, last, real, some_hide, lds.mo[wave]);
            else
                mark_not_finite<D, kWaves>(a, b, base, g, r0, min(R, rows - r0), wave, u0, u1, all_see, last, lds.mo[wave]);
        }
        __syncthreads();
#pragma unroll 1
        for (int qr = tid >> 4; qr < R; qr += NT / 16)
            if (r0 + qr < rows)
                finish<D, kWaves, ONE, MASKS>(a, tid, b, base, g, r0 + qr, u0, [&](int w) { return mm[w][qr]; }, [&](int w) { return ml[w][qr]; },
                                       [&](int w, int c) { return *reinterpret_cast<const float4*>(&lds.mo[w][qr][c]); });
    };
    each_segment<W, MASKS>(a, segment);
}

template <int MASKS, int D, int NQ, int NP>
void launch_rows(const Args& a, const Plan& p, hipStream_t st) {
    const dim3 grid(a.shares, a.c.Hkv, p.groups);
    const auto kernel = p.one      ? attn_kv4_rows_kernel<D, NQ, NP, Work::kSequence, MASKS>
                        : a.B == 1 ? attn_kv4_rows_kernel<D, NQ, NP, Work::kShare, MASKS>
                                   : attn_kv4_rows_kernel<D, NQ, NP, Work::kLine, MASKS>;
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, st, a);
}
template <int MASKS, int D>
void launch_rows(const Args& a, int q_dtype, const Plan& p, bool exact, hipStream_t st) {
    const bool half = q_dtype == MXFP4_DT_F16;
    if (exact) half ? launch_rows<MASKS, D, 2, 3>(a, p, st) : launch_rows<MASKS, D, 1, 3>(a, p, st);
    else half ? launch_rows<MASKS, D, 2, 2>(a, p, st) : launch_rows<MASKS, D, 1, 2>(a, p, st);
}
template <int MASKS>
int launch_rows(const Args& a, int q_dtype, const Plan& p, int D, bool exact, hipStream_t st) {
    if (D == 64) launch_rows<MASKS, 64>(a, q_dtype, p, exact, st);
    else launch_rows<MASKS, 128>(a, q_dtype, p, exact, st);
    return mxh::launch_status("attn_kv4 (rows)");
}

}  // namespace
