// attn_kv4.h -- what the kernels of attention over the MXFP4 cache share: arguments,
// a batch's shares, a unit's softmax, and where a row goes (fp32, bf16 or fp16, and / or
// the MXFP4 rows of its bf16 rounding, o_proj's activations).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv4.h"
#include "mx_device.h"
#include "mxfp4_hip.h"
#include "quant_rows.h"

namespace mxa {

using kv4::Cache;

constexpr int kUnit = 32;              // positions per wave and step
constexpr float kMost = 2048.0f;       // a lane's terms of a unit sum to at most this
constexpr float kWide = 262144.0f;     // a reference past it: an exponent's rounding is up to 2^-6 and more
constexpr float kNone = -3e38f;        // the reference of a row that has seen nothing: exp2(-inf - kNone) = 0
constexpr uint32_t kNoRow = 0xFFFFFFFFu;
constexpr int kFew = 32;               // shares of a sequence that four waves merge at once
constexpr int kMinShare = 4;           // units, one a wave
// Units that take about as long as a workgroup's change to another sequence; whole shares of kMinShare.  4 / 6 / 8 / 9 /
// 12 / 20, us: 48 sequences of up to 8192 positions (four heads) 30.7 / 29.7 / 28.3 / 27.9 / 29.8 / 29.6, 32 of 32768
// 58.6 / 56.1 / 56.8 / 56.6 / 56.5 / 56.4, 300 of 8000 139 / 139 / 138 / 138 / 138 / 141; none at all, 48 of 8192 37.3.
constexpr uint32_t kPad = 8;

struct Out {
    void* o;        // or null
    int dtype;      // MXFP4_DT_*
    uint8_t* oq;    // or null, with os
    uint8_t* os;
};

// Columns c0 .. c0 + N - 1 (N = 8 or 4) of row `row` of (rows, D).  The lanes of a
// 32-block are neighbours (four of 8 columns, eight of 4) and all call it.
template <int N>
__device__ __forceinline__ void store(const Out& t, int64_t row, int D, int c0, const float (&o)[N]) {
    const int64_t at = row * D + c0;
    if (t.o) {
        if (t.dtype == MXFP4_DT_F32) {
            float* p = static_cast<float*>(t.o) + at;
#pragma unroll
            for (int c = 0; c < N; c += 4) *reinterpret_cast<float4*>(p + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        } else {
            uint32_t w[N / 2];
#pragma unroll
            for (int c = 0; c < N; c += 2) {
                if (t.dtype == MXFP4_DT_BF16) {
                    w[c / 2] = mx::f32x2_to_bf16x2(o[c], o[c + 1]);
                } else {
                    w[c / 2] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)o[c]) |
                               (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)o[c + 1]) << 16;
                }
            }
            uint16_t* p = static_cast<uint16_t*>(t.o) + at;
            if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
            else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        }
    }
    if (t.oq) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, am = 0.0f;
#pragma unroll
        for (int c = 0; c < N; ++c) {
            v[c] = mx::bf16_to_f32(mx::f32_to_bf16_rne(o[c]));
            am = fmaxf(am, __builtin_fabsf(v[c]));
        }
        am = fmaxf(am, mx::dpp<mx::kDppQuadXor1>(am));
        am = fmaxf(am, mx::dpp<mx::kDppQuadXor2>(am));
        if constexpr (N == 4) am = fmaxf(am, mx::dpp<mx::kDppRowHalfMirror>(am));
        const uint32_t code = mx::e8m0_code(am);
        const uint32_t packed = mx::e2m1_pack8_short(v, mx::e8m0_inv_scale(code));
        uint8_t* q = t.oq + at / 2;
        if constexpr (N == 8) *reinterpret_cast<uint32_t*>(q) = packed;
        else *reinterpret_cast<uint16_t*>(q) = (uint16_t)packed;
        if (c0 % 32 == 0) t.os[at / 32] = (uint8_t)code;
    }
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ mx::v4f mfma_bf16(uint4 a, uint4 b, mx::v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
}

struct Args {
    const uint16_t* q;
    int64_t ldq;                 // elements between tokens of q
    Cache c;
    const int32_t* dpos;
    int4* places;                // of a sequence, for the merge: its first share, where in that, places a share
    float* part;                 // records
    Out out;
    int per;                     // units of a share of one sequence, or 0: as share_units finds from its length
    int B, M, Hq, G, shares, records;   // shares of the batch, and records a row may have (its stride)
    float scale;                 // log2(e) / sqrt(D)
};

// Units of a sequence whose first token is at base.
__device__ __forceinline__ uint32_t units_of(const Args& a, int base) {
    const int64_t n = (int64_t)base + a.M;
    return (uint32_t)(((int)(n < 0 ? 0 : n < a.c.max_pos ? n : a.c.max_pos) + kUnit - 1) / kUnit);
}
// Inclusive prefix sums over the wave (every lane active).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);    // row_shr 1, 2, 4, 8: within 16 lanes
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast 15: row 0's total to row 1, 2's to 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast 31: the first half's to the second
    return v;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }

// Units of a share for `total` units in the batch: whole rounds of the four waves, as
// few as a.shares of them need, two rounds at least from 32 shares a sequence on (fewer
// records to merge; one token, us with at least 1 / 2 rounds: 4096 positions 8.2 / 9.0,
// 8000 9.8 / 9.1, 32000 16.4 / 13.5).
__device__ __forceinline__ uint32_t share_units(uint64_t total, const Args& a) {
    const uint64_t n = total + a.shares - 1;
    const uint32_t per = (uint32_t)((n >> 32 ? n / a.shares : (uint32_t)n / (uint32_t)a.shares) + 3) & ~3u;
    return max(per, total > (uint64_t)kFew * kMinShare * a.B ? 2u * kMinShare : (uint32_t)kMinShare);
}

// The batch's units stand in one line, sequence after sequence, each behind kPad places
// for what a workgroup spends on a sequence besides its units; share i has places i per
// .. (i + 1) per - 1, so units of one sequence or of several in a row, and all shares are
// about the same work whatever the lengths.  Every wave finds its place by itself: a lane
// per sequence, sums over the wave.  All uniform.
struct Place {
    uint32_t per;
    int b, base;        // a sequence, its dpos, and where it starts
    uint64_t start;
};
// Share blockIdx.x's first sequence; false: it is past the line.
__device__ __forceinline__ bool find_share(const Args& a, Place& p) {
    const int lane = threadIdx.x & 63;
    auto places = [&](int b0, int& base) {
        base = 0;
        if (b0 + lane >= a.B) return 0u;
        base = a.dpos[b0 + lane];
        const uint32_t n = units_of(a, base);
        return n ? n + kPad : 0u;
    };
    int base;
    const uint32_t n0 = places(0, base), to0 = wave_scan(n0);
    uint64_t total = last_lane(to0);
    for (int b0 = 64; b0 < a.B; b0 += 64) {
        int t;
        total += last_lane(wave_scan(places(b0, t)));
    }
    p.per = share_units(total, a);
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x < 64) {
        // The last share, the least full, leaves the places for the merge, which would have to find them again (us with
        // that / without: 48 sequences of up to 8192 positions 28.9 / 27.9, 200 of 8000 108 / 99)
        uint64_t start = kPad;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            int t;
            const uint32_t n = b0 ? places(b0, t) : n0, to = b0 ? wave_scan(n) : to0;
            const uint64_t at = start + to - n;
            const uint64_t share = total >> 32 ? at / p.per : (uint32_t)at / p.per;
            if (b0 + lane < a.B) a.places[b0 + lane] = make_int4((int)share, (int)(at - share * p.per), (int)p.per, 0);
            start += last_lane(to);
        }
    }
    const uint64_t target = (uint64_t)blockIdx.x * p.per;
    if (target >= total) return false;
    p.start = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const uint32_t n = b0 ? places(b0, base) : n0, to = b0 ? wave_scan(n) : to0;
        const uint64_t past = __ballot(p.start + to > target);
        if (past) {
            const int l = (int)__builtin_ctzll(past);
            p.b = b0 + l;
            p.base = __builtin_amdgcn_readlane(base, l);
            p.start += (uint32_t)__builtin_amdgcn_readlane((int)(to - n), l);
            return true;
        }
        p.start += last_lane(to);
    }
    return false;
}

// What a workgroup (blockIdx.x) works on.
enum class Work {
    kSequence,   // a whole sequence
    kShare,      // a share of the batch's one sequence
    kLine,       // a share of the line
};
// Its sequences in turn: segment(b, its dpos, its units u0 .. u1 - 1).
template <Work W, class Segment>
__device__ __forceinline__ void each_segment(const Args& a, Segment segment) {
    if constexpr (W == Work::kSequence) {
        segment(blockIdx.x, __builtin_amdgcn_readfirstlane(a.dpos[blockIdx.x]), 0, INT32_MAX);
        return;
    }
    if constexpr (W == Work::kShare) {      // (a kernel of its own: nine tokens over 23001 positions 25.1 us, in the loop 25.8)
        const int base = a.dpos[0];         // (in flight, where nothing here needs it)
        uint32_t per = a.per;
        if (per == 0) per = share_units(units_of(a, __builtin_amdgcn_readfirstlane(base)), a);
        if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) a.places[0] = make_int4(0, 0, (int)per, 0);
        const uint32_t u0 = blockIdx.x * per;
        segment(0, base, (int)u0, (int)(u0 + per));
        return;
    }
    Place p;
    if (!find_share(a, p)) return;             // uniform
    const uint64_t from = (uint64_t)blockIdx.x * p.per;
    constexpr int pad = kPad;
    for (bool first = true;;) {
        const int n = (int)units_of(a, p.base);
        // the share's beginning and end in units of the sequence, which ends past `from` (per < 2^28)
        const int u1 = (int)min((int64_t)n, (int64_t)(from + p.per - p.start) - pad);
        const int u0 = (int)max((int64_t)0, (int64_t)from - (int64_t)p.start - pad);
        if (u0 < u1) {
            if (!first) __syncthreads();                   // LDS is used again
            first = false;
            segment(p.b, p.base, u0, u1);
        }
        if (n) p.start += n + pad;
        if (++p.b == a.B || p.start >= from + p.per) return;
        p.base = __builtin_amdgcn_readfirstlane(a.dpos[p.b]);
    }
}

// N (a multiple of 8) fp32 terms as NP bf16 parts each, whose sum each is (8 bits a
// part, rounded to nearest, the rest exact): p[k][j] is part j of terms 8 k .. 8 k + 7.
template <int N, int NP>
__device__ __forceinline__ void parts(float (&t)[N], uint4 (&p)[N / 8][NP]) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        uint32_t o[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            o[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{t[2 * i], t[2 * i + 1]}), bf16x2_t));
            if (j + 1 < NP) {
                t[2 * i] -= __uint_as_float(o[i] << 16);
                t[2 * i + 1] -= __uint_as_float(o[i] & 0xFFFF0000u);
            }
        }
#pragma unroll
        for (int k = 0; k < N / 8; ++k) p[k][j] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
    }
}

// The largest of three, a NaN among them left out (as fmaxf, whose operands the
// compiler would first pass through an instruction each).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// a * b rounded, minus c: not one fma.
__device__ __forceinline__ float mul_then_sub(float a, float b, float c) {
#pragma clang fp contract(off)
    const float ab = a * b;
    return ab - c;
}

// The maximum / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
template <bool MAX>
__device__ __forceinline__ float over_lq(float v) {
    auto op = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// Eight elements of q as bf16 parts: bf16 itself, or fp16's 11 bits as 8 + 3.
template <int NQ>
__device__ __forceinline__ void q_parts(uint4 w, uint4 (&p)[NQ]) {
    if constexpr (NQ == 1) {
        p[0] = w;
    } else {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = mx::f16_to_f32((uint16_t)(x[i / 2] >> (16 * (i & 1))));
        uint4 o[1][NQ];
        parts(t, o);
#pragma unroll
        for (int j = 0; j < NQ; ++j) p[j] = o[0][j];
    }
}

// One unit of a row's softmax, in two parts with other work between them.  The lane's N
// scores s to terms t = exp2(s scale - m) and their sum.  The reference m is not the row's
// maximum: any gives the same quotient, and no unit looks for one that need not.  `wide`
// (uniform): a row's reference is past kWide.
template <int N>
__device__ __forceinline__ void terms(const float (&s)[N], float scale, float m, bool wide, float (&t)[N], float& sum) {
    if (!wide) {
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = fmaf(s[i], scale, -m);
    } else {   // such a row's by the rounded product, as in m: the fma's would differ from it by more than a term
        const bool mine = fabsf(m) > kWide;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float near = fmaf(s[i], scale, -m), far = mul_then_sub(s[i], scale, m);
            t[i] = mine ? far : near;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = __builtin_amdgcn_exp2f(t[i]);
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i += 4) sum += (t[i] + t[i + 1]) + (t[i + 2] + t[i + 3]);
}
// The terms of a row with a lane of more than kMost (at its first unit, where m is kNone
// and they are infinite, or past a much larger score) are made again, on the maximum, and
// what was summed before is rescaled (rescale(factor)); over(x): the maximum over the row's
// lanes.  The wave's other rows get the same terms and a factor of 1: a row's bits are its
// own.  p: the terms' parts.  Then l, their sum so far, takes them.
template <int N, int NP, class Over, class Rescale>
__device__ __forceinline__ void again(const float (&s)[N], float scale, float& m, float& l, bool& wide, float sum, uint4 (&p)[N / 8][NP],
                                      Over over, Rescale rescale) {
    if (__ballot(sum > kMost)) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < N; i += 2) top = max3(top, s[i], s[i + 1 < N ? i + 1 : i]);
        const float mn = over(sum) > kMost ? fmaxf(m, over(top) * scale) : m;
        const float al = __builtin_amdgcn_exp2f(m - mn);
        l *= al;
        rescale(al);
        m = mn;
        wide = __ballot(fabsf(mn) > kWide && mn != kNone) != 0ull;
        float t[N];
        terms(s, scale, m, wide, t, sum);
        parts(t, p);
    }
    l += sum;
}

// A code of a position's word, in the exponent field of a scale for the packed
// conversions, which read that field alone: its neighbours are around it.
__device__ __forceinline__ float scale_at(uint32_t word, uint32_t block) {
    return __uint_as_float(__builtin_amdgcn_alignbit(word, word, 8 * block + 9));
}

// w * 0 summed: 0, or NaN where one of eight bf16 is an infinity or a NaN.
__device__ __forceinline__ float not_finite(uint4 w) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    float z = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) z = fmaf(mx::bf16_to_f32((uint16_t)(x[i / 2] >> (16 * (i & 1)))), 0.0f, z);
    return z;
}

// Values that are not finite, in a unit with positions that not all of a workgroup's rows
// see, are taken out of the products (0 times one is NaN), and what sees one is made NaN
// here, in a wave's sums once they lie in LDS (mo: row r0 on; by the wave that put them
// there): from the first unit that is not `all_see`'s alone, positions up to `to` of the
// wave's units (u0 + wave + NW j, up to u1 - 1).
template <int D, int NW>
__device__ __forceinline__ void mark_not_finite(const Args& a, int b, int base, int g, int r0, int rows, int wave, int u0, int u1, int all_see,
                                                int to, float (*mo)[D + 4]) {
    asm volatile("" ::: "memory");                   // (behind the wave's own stores, which LDS keeps in order)
    for (int pos = max((all_see + 1) / kUnit, u0) * kUnit; pos <= to && pos / kUnit < u1; ++pos) {
        if ((pos / kUnit - u0) % NW != wave) continue;
        const int64_t row = kv4::head_row(a.c, b, g, pos);
        if (row < 0) continue;
        const int first = (int)max((int64_t)0, ((int64_t)pos - base) * a.G - r0);      // rows from here on see it
        for (int col = threadIdx.x & 63; col < D; col += 64) {
            const uint32_t w = a.c.vq[row * (D / 2) + col / 2] >> (4 * (col & 1));
            if (kv4::not_finite(w, a.c.vs[row * (D / 32) + col / 32]) & 1)
                for (int r = first; r < rows; ++r) mo[r][col] = __builtin_nanf("");
        }
    }
}

// The end of row r of kv head g of sequence b, a segment from unit u0 on: NW waves' (m, l,
// columns) to one record, or with ONE the output.  16 neighbouring lanes a row (by
// tid), which all call it, D / 16 columns a lane.
template <int D, int NW, bool ONE, class M, class L, class O>
__device__ __forceinline__ void finish(const Args& a, int tid, int b, int base, int g, int r, int u0, M m_of, L l_of, O o_of) {
    constexpr int CT = D / 16;
    const int c0 = CT * (tid & 15);
    const int64_t pos = (int64_t)base + r / a.G;
    if (!ONE && (pos < 0 || pos >= a.c.max_pos || (int64_t)u0 * kUnit > pos)) return;   // no record: the merge reads none
    float gm = m_of(0);
#pragma unroll
    for (int w = 1; w < NW; ++w) gm = fmaxf(gm, m_of(w));
    float o[CT], den = 0.0f;
#pragma unroll
    for (int c = 0; c < CT; ++c) o[c] = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float wt = __builtin_amdgcn_exp2f(m_of(w) - gm);
        den = fmaf(wt, l_of(w), den);
#pragma unroll
        for (int c = 0; c < CT; c += 4) {
            const float4 x = o_of(w, c0 + c);
            o[c] = fmaf(wt, x.x, o[c]);
            o[c + 1] = fmaf(wt, x.y, o[c + 1]);
            o[c + 2] = fmaf(wt, x.z, o[c + 2]);
            o[c + 3] = fmaf(wt, x.w, o[c + 3]);
        }
    }
    if constexpr (ONE) {
        const bool none = pos < 0 || pos >= a.c.max_pos || den == 0.0f;   // nothing seen: zeros
        const float inv = none ? 0.0f : 1.0f / den;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c] = none ? 0.0f : o[c] * inv;
        store<CT>(a.out, ((int64_t)b * a.M + r / a.G) * a.Hq + g * a.G + r % a.G, D, c0, o);
    } else {
        float* rec = a.part + (((int64_t)g * a.M * a.G + r) * a.records + blockIdx.x + b) * (D + 4);
#pragma unroll
        for (int c = 0; c < CT; c += 4) *reinterpret_cast<float4*>(rec + 4 + c0 + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        if (c0 == 0) *reinterpret_cast<float2*>(rec) = make_float2(gm, den);
    }
}

// More than 16 query rows of a kv head (attn_kv4_rows.hip), in groups of 32; exact: p in
// three bf16 parts instead of two.
int attn_rows(const Args& a, int q_dtype, int groups, int D, bool one, bool exact, hipStream_t st);

}  // namespace mxa
