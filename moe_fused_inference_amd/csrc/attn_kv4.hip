// attn_kv4.hip -- attention over the MXFP4 KV cache (kv4.h): M tokens of each of
// B sequences, token m of sequence b at dpos[b] + m over positions 0 .. dpos[b] + m.
//
//   attn_kv4_kernel        workgroup (share of a sequence, kv head g, row group):
//                          the share's positions against up to 32 query rows
//                          (tokens x heads of the kv head), a wave taking every
//                          fourth unit of 32 positions with its own running
//                          softmax; the waves' sums meet in LDS -> one record
//                          (reference, sum, D column sums) per row and share, or
//                          the output where a sequence has one share.
//   attn_kv4_merge_kernel  workgroup (kv head's row, sequence): the row's records
//                          -> its output.
//
// Shares.  dpos lives on the device, so the host fixes only how many shares there
// may be (about a round of workgroups, plus one a sequence); every workgroup adds
// up the batch's lengths, and a share is the same number of units for every
// sequence, so that long and short ones load the chip alike.
//
// Mathematics.  Both products are transposed, S^T = K Q^T and O^T = V^T P^T: an
// MFMA leaves a lane with four positions of each of two 16-position tiles of one
// query, which is its B operand of the second product as it stands, so P passes
// through no LDS.  K and V are bf16, which holds every cache value, two values an
// instruction by the scaled conversion.  P is bf16 parts whose sum is the fp32
// probability at any size.  m is the reference of a row's terms, not their
// maximum: it follows the maximum only past a factor of 2^kSlack.
#include "attn_kv4.h"
#include "kv4.h"
#include "mx_device.h"
#include "mx_host.h"

#include <algorithm>
#include <type_traits>

namespace {

using kv4::Cache;

constexpr int kUnit = 32;              // positions per wave and step
constexpr float kSlack = 8.0f;         // a term is at most 2^8
constexpr float kWide = 262144.0f;     // a reference past it: an exponent's rounding is up to 2^-6 and more
constexpr float kNone = -3e38f;        // the reference of a row that has seen nothing: exp2(-inf - kNone) = 0
constexpr uint32_t kNoRow = 0xFFFFFFFFu;
constexpr int kMaxRT = 2;              // 16-row tiles per workgroup
constexpr int kFew = 32;               // shares of a sequence that four waves merge at once
constexpr int kMinShare = 4;           // units, one a wave
constexpr int kParts = 3;              // bf16 parts of a probability

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
    float* part;
    mxa::Out out;
    int B, M, Hq, G, shares, wanted;   // shares: how many there may be, over the batch
    float scale;                 // log2(e) / sqrt(D)
};

// Units of sequence b.
__device__ __forceinline__ uint32_t units_of(const Args& a, int b) {
    const int64_t n = (int64_t)a.dpos[b] + a.M;
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
__device__ __forceinline__ uint32_t shares_of(uint32_t units, uint32_t per) { return (units + per - 1) / per; }

// Units of a share for `total` units in the batch: a.wanted of them, in whole rounds of
// the four waves, two rounds at least from 32 shares a sequence on (fewer records to
// merge; one token, us with at least 1 / 2 rounds: 4096 positions 8.2 / 9.0, 8000 9.8 /
// 9.1, 32000 16.4 / 13.5).
__device__ __forceinline__ uint32_t share_units(uint64_t total, const Args& a) {
    const uint32_t per = (uint32_t)((total + a.wanted - 1) / a.wanted + 3) & ~3u;
    return max(per, total > (uint64_t)kFew * kMinShare * a.B ? 2u * kMinShare : (uint32_t)kMinShare);
}

// What a share holds -- the same whole rounds of the four waves for every sequence, so
// few units that the batch has at most a.wanted shares, or a few more -- and for share
// number `at` of the batch its sequence b and its number s there, or for at < 0 the
// batch's number of sequence b's first share.  Every wave finds them by itself: a lane
// per sequence, sums over the wave.  All uniform.
struct Place {
    int per, b, s, first;
};
__device__ __forceinline__ bool find_share(const Args& a, int at, Place& p) {
    const int lane = threadIdx.x & 63;
    auto units = [&](int b0) { return b0 + lane < a.B ? units_of(a, b0 + lane) : 0u; };
    if (a.B == 1) {
        const uint32_t nu = units_of(a, 0);
        p.per = (int)share_units(nu, a);
        p.first = p.b = 0;
        p.s = at;
        return at < 0 || (int64_t)at * p.per < nu;
    }
    const uint32_t u0 = units(0);
    uint64_t total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) total += last_lane(wave_scan(b0 ? units(b0) : u0));
    uint32_t per = share_units(total, a);
    for (int i = 0; i < 3; ++i) {      // a sequence's last share is a part of one: longer ones until they are few enough
        uint32_t n = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) n += last_lane(wave_scan(shares_of(b0 ? units(b0) : u0, per)));
        if (n <= (uint32_t)a.wanted) break;
        per = max(per + 4, (uint32_t)((uint64_t)per * n / a.wanted + 3) & ~3u);
    }
    p.per = (int)per;
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int ns = (int)shares_of(b0 ? units(b0) : u0, per), upto = (int)wave_scan(ns);
        int l = p.b - b0;
        if (at >= 0) {
            const uint64_t past = __ballot(before + upto > at);
            l = past ? (int)__builtin_ctzll(past) : 64;
        }
        if (l < 64) {
            p.b = b0 + l;
            p.first = before + __builtin_amdgcn_readlane(upto - ns, l);
            p.s = at - p.first;
            return true;
        }
        before += (int)last_lane(upto);
    }
    return false;
}

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

// row[t]: tile t's first head row (uniform).
template <int D>
__device__ __forceinline__ void load_k(Raw<D>& r, const Cache& c, const uint32_t (&row)[2], const Lane<D>& o) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        r.k[t] = *reinterpret_cast<const typename Raw<D>::vec*>(c.kq + (uint64_t)row[t] * (D / 2) + o.k);
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

// Eight fp32 terms as bf16 parts whose sum each is (8 bits a part, rounded to nearest, the rest exact).
template <int N>
__device__ __forceinline__ void parts(float (&t)[8], uint4 (&p)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{t[2 * i], t[2 * i + 1]}), bf16x2_t));
            if (j + 1 < N) {
                t[2 * i] -= __uint_as_float(o[i] << 16);
                t[2 * i + 1] -= __uint_as_float(o[i] & 0xFFFF0000u);
            }
        }
        p[j] = make_uint4(o[0], o[1], o[2], o[3]);
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
        parts<NQ>(t, p);
    }
}

template <int D, int RT, int NQ, bool ONE, int NW>
__global__ __launch_bounds__(64 * NW, RT == 1 ? 4 : 2) void attn_kv4_kernel(Args a) {
    constexpr int R = 16 * RT, KT = D / 32, CT = D / 16;
    // q, and after the last unit the waves' sums
    __shared__ union Lds {
        alignas(16) uint16_t qs[NQ * R][D + 8];
        alignas(16) float mo[NW][16][D + 4];
    } lds;
    auto& qs = lds.qs;
    auto& mo = lds.mo;
    __shared__ float mm[NW][16], ml[NW][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lq = lane >> 4;
    const int g = blockIdx.y, r0 = blockIdx.z * R, G = a.G;
    const int rows = a.M * G;
    int b = 0, u0 = 0, u1 = INT32_MAX;
    if constexpr (ONE) {
        b = blockIdx.x;
    } else {
        Place pl;
        if (!find_share(a, blockIdx.x, pl)) return;        // uniform
        b = pl.b;
        u0 = pl.s * pl.per;
        u1 = u0 + pl.per;
    }
    // Positions fit 31 bits: a token before the cache is put at -1, one past it at its end
    const int64_t base = __builtin_amdgcn_readfirstlane(a.dpos[b]);
    auto clamped = [&](int64_t pos) { return (int)(pos < 0 ? -1 : pos < a.c.max_pos ? pos : a.c.max_pos); };
    const int last = min(clamped(base + a.M - 1), a.c.max_pos - 1);      // positions past it are no one's
    const int lim_min = clamped(base + r0 / G);                          // the group's first token sees up to here
    const int lim_max = min(clamped(base + (min(r0 + R, rows) - 1) / G), a.c.max_pos - 1);   // its last one
    u1 = min(u1, (lim_max + kUnit) / kUnit);
    if (!ONE && u0 >= u1) return;                           // no record: the merge reads none
    // q, whose parts go to LDS once the first units' loads are on their way
    const uint16_t* qb = a.q + (int64_t)b * a.M * a.ldq + (int64_t)g * G * D;
    constexpr int NT = 64 * NW, QN = (R * (D / 8) + NT - 1) / NT;
    uint4 qw[QN];
#pragma unroll
    for (int i = 0; i < QN; ++i) {
        const int r = r0 + (tid + NT * i) / (D / 8), ch = (tid + NT * i) % (D / 8);
        qw[i] = make_uint4(0, 0, 0, 0);
        if (r < rows && (R * (D / 8) % NT == 0 || tid + NT * i < R * (D / 8)))
            qw[i] = *reinterpret_cast<const uint4*>(qb + (int64_t)(r / G) * a.ldq + (r % G) * D + 8 * ch);
    }
    // the first head rows of the wave's units u0 + wave + NW j, j = lane, tiles 0 and 1 (kNoRow: there is no such tile)
    uint32_t first[2];
    auto find_rows = [&](int j0) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int64_t pos = ((int64_t)u0 + wave + NW * (j0 + lane)) * kUnit + 16 * t;
            first[t] = kNoRow;
            if (pos < a.c.max_pos) {
                const int64_t row = kv4::head_row(a.c, b, g, (int)pos);
                first[t] = row < 0 ? kNoRow : (uint32_t)row;
            }
        }
    };
    const Lane<D> off(lane);
    // the wave's j-th unit: its tiles' rows, and which of them exist
    auto locate = [&](int j, uint32_t (&row)[2]) -> int {
        const uint32_t r0 = __builtin_amdgcn_readlane(first[0], j & 63), r1 = __builtin_amdgcn_readlane(first[1], j & 63);
        row[0] = r0 == kNoRow ? 0 : r0;
        row[1] = r1 == kNoRow ? 0 : r1;
        return (r0 == kNoRow ? 0 : 1) | (r1 == kNoRow ? 0 : 2);
    };
    Raw<D> r;
    int there = 0;
    if (u0 + wave < u1) {
        uint32_t row[2];
        find_rows(0);
        there = locate(0, row);
        load_k(r, a.c, row, off);
        load_v(r, a.c, row, off);
    }
    auto check = [](uint4 w) {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) z = fmaf(mx::bf16_to_f32((uint16_t)(x[i / 2] >> (16 * (i & 1)))), 0.0f, z);
        return z;
    };
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
    float zero[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        zero[rt] = 0.0f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) zero[rt] += check(*reinterpret_cast<const uint4*>(&qs[16 * rt + l16][(D / 4) * lq + 8 * kt]));
        zero[rt] = over_lq<false>(zero[rt]);
    }
    // the lane's query of tile rt: row r0 + 16 rt + l16; rows that are none see everything and write nothing
    int lim[RT];
    float m[RT], l[RT];
    bool wide[RT];   // uniform: a row's reference is past kWide
    mx::v4f acc[RT][CT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = r0 + 16 * rt + l16;
        lim[rt] = r < rows ? clamped(base + r / G) : 1 << 30;
        m[rt] = kNone;
        l[rt] = 0.0f;
        wide[rt] = false;
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[rt][c] = mx::v4f{0.f, 0.f, 0.f, 0.f};
    }
    // Unit u, the wave's j-th.  `more`: the wave's next one is loaded meanwhile (decided in the code, not by a branch:
    // behind one the compiler waits for the older loads as if these had not been issued, that is for all)
    auto unit = [&](int u, int j, auto more_) {
        constexpr bool more = decltype(more_)::value;
        const int p0 = u * kUnit;
        uint32_t next[2];
        int there_next = 0;
        if constexpr (more) {
            if (((j + 1) & 63) == 0) find_rows(j + 1);
            there_next = locate(j + 1, next);
        }
        mx::v4f s[RT][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            uint4 kd[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) kd[kt] = kv4::eight_bf16(r.k[t][kt], kv4::scale_of(r.ks[t]));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                s[rt][t] = mx::v4f{zero[rt], zero[rt], zero[rt], zero[rt]};
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        const uint4 qf = *reinterpret_cast<const uint4*>(&qs[n * R + 16 * rt + l16][(D / 4) * lq + 8 * kt]);
                        s[rt][t] = mfma_bf16(kd[kt], qf, s[rt][t]);
                    }
            }
        }
        if constexpr (more) load_k(r, a.c, next, off);
        // s[rt][t][i]: position p0 + 16 t + 4 lq + i
        uint4 p[RT][kParts];
        const bool masked = __builtin_amdgcn_readfirstlane(p0 + kUnit - 1 > lim_min || there != 3);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (masked) {
                int sees = lim[rt] - p0 - 4 * lq;    // -1 or less: none of the lane's positions
                asm volatile("" : "+v"(sees));       // (nothing below it is computed ahead of the branch)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(there >> t & 1) || 16 * t + i > sees) s[rt][t][i] = -INFINITY;
            }
            const float top = max3(max3(s[rt][0][0], s[rt][0][1], s[rt][0][2]), max3(s[rt][0][3], s[rt][1][0], s[rt][1][1]),
                                   max3(s[rt][1][2], s[rt][1][3], s[rt][1][3]));
            if (__ballot(top * a.scale > m[rt] + kSlack)) {
                const float mn = fmaxf(m[rt], over_lq<true>(top) * a.scale);
                const float al = __builtin_amdgcn_exp2f(m[rt] - mn);
                l[rt] *= al;
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[rt][c][i] *= al;
                m[rt] = mn;
                wide[rt] = __ballot(fabsf(mn) > kWide && mn != kNone) != 0ull;
            }
            float t[8];
            if (!wide[rt]) {
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = fmaf(s[rt][i >> 2][i & 3], a.scale, -m[rt]);
            } else {   // the rounded product, as in m: the fma's would differ from it by more than a term
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = mul_then_sub(s[rt][i >> 2][i & 3], a.scale, m[rt]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = __builtin_amdgcn_exp2f(t[i]);
            l[rt] += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
            parts<kParts>(t, p[rt]);
        }
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
        }
        auto product = [&](auto half) {
            constexpr int H = decltype(half)::value;
            uint4 vd[4];
            decode_v<H>(r.v, vs, vd);
            if constexpr (H == CT / 4 - 1 && more) load_v(r, a.c, next, off);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int k = kParts - 1; k >= 0; --k)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[rt][4 * H + c] = mfma_bf16(vd[c], p[rt][k], acc[rt][4 * H + c]);
        };
        product(std::integral_constant<int, 0>{});
        __builtin_amdgcn_sched_barrier(0);   // and one half's at a time
        if constexpr (CT == 8) product(std::integral_constant<int, 1>{});
        there = there_next;
    };
    int u = u0 + wave, j = 0;
    for (; u + NW < u1; u += NW, ++j) unit(u, j, std::true_type{});
    if (u < u1) unit(u, j, std::false_type{});
    // the waves' sums of each tile in LDS, then one record (or the output) per
    // row: acc[rt][c][i] is column D/16 (4 lq + i) + c of query l16
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        __syncthreads();
        const float ls = over_lq<false>(l[rt]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < CT; c += 4)
                *reinterpret_cast<float4*>(&mo[wave][l16][CT * (4 * lq + i) + c]) =
                    make_float4(acc[rt][c][i], acc[rt][c + 1][i], acc[rt][c + 2][i], acc[rt][c + 3][i]);
        if (lq == 0) {
            mm[wave][l16] = m[rt];
            ml[wave][l16] = ls;
        }
        __syncthreads();
        // thread: CT columns of a row (8 of 128, 4 of 64)
        const int qr = tid >> 4, c0 = CT * (tid & 15);
        const int rr = r0 + 16 * rt + qr;
        if (tid >= 256 || rr >= rows) continue;
        const int64_t pos = base + rr / G;
        if (!ONE && (pos < 0 || pos >= a.c.max_pos || u0 * kUnit > pos)) continue;   // no record: the merge reads none
        float gm = mm[0][qr];
#pragma unroll
        for (int w = 1; w < NW; ++w) gm = fmaxf(gm, mm[w][qr]);
        float o[CT], den = 0.0f;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float wt = __builtin_amdgcn_exp2f(mm[w][qr] - gm);
            den = fmaf(wt, ml[w][qr], den);
#pragma unroll
            for (int c = 0; c < CT; c += 4) {
                const float4 x = *reinterpret_cast<const float4*>(&mo[w][qr][c0 + c]);
                o[c] = fmaf(wt, x.x, o[c]);
                o[c + 1] = fmaf(wt, x.y, o[c + 1]);
                o[c + 2] = fmaf(wt, x.z, o[c + 2]);
                o[c + 3] = fmaf(wt, x.w, o[c + 3]);
            }
        }
        if constexpr (ONE) {
            const bool none = pos < 0 || pos >= a.c.max_pos || den == 0.0f;   // nothing seen: zeros
            const float r = none ? 0.0f : 1.0f / den;
#pragma unroll
            for (int c = 0; c < CT; ++c) o[c] = none ? 0.0f : o[c] * r;
            mxa::store<CT>(a.out, ((int64_t)b * a.M + rr / G) * a.Hq + g * G + rr % G, D, c0, o);
        } else {
            float* rec = a.part + (((int64_t)g * rows + rr) * a.shares + blockIdx.x) * (D + 4);
#pragma unroll
            for (int c = 0; c < CT; c += 4) *reinterpret_cast<float4*>(rec + 4 + c0 + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
            if (c0 == 0) *reinterpret_cast<float2*>(rec) = make_float2(gm, den);
        }
    }
}

// Workgroup (row of kv head g: blockIdx.x = g * rows + r, sequence b): the row's
// records dealt to NW waves, eight loaded at a time (one memory latency for up to
// 8 NW), each with a running reference; a lane holds D / 64 columns.
template <int D, int NW>
__global__ __launch_bounds__(64 * NW) void attn_kv4_merge_kernel(Args a) {
    constexpr int C = D / 64, CT = D / 16, N = 8;
    typedef float cvec __attribute__((ext_vector_type(C)));
    __shared__ float mm[NW], ml[NW];
    __shared__ __align__(16) float mo[NW][D];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rows = a.M * a.G;
    Place p;
    p.b = blockIdx.y;
    find_share(a, -1, p);
    const int g = blockIdx.x / rows, r = blockIdx.x - g * rows;
    const int64_t pos = (int64_t)a.dpos[p.b] + r / a.G;
    const int ns = __builtin_amdgcn_readfirstlane(
        pos < 0 || pos >= a.c.max_pos ? 0 : (int)(pos / kUnit) / p.per + 1);   // shares of positions 0 .. pos
    const float* rec = a.part + ((int64_t)blockIdx.x * a.shares + __builtin_amdgcn_readfirstlane(p.first)) * (D + 4);
    float m = kNone, l = 0.0f;
    cvec o = 0.0f;
    for (int i0 = wave; i0 < ns; i0 += N * NW) {
        float2 st[N];
        cvec v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float* x = rec + (int64_t)min(i0 + k * NW, ns - 1) * (D + 4);
            st[k] = *reinterpret_cast<const float2*>(x);
            v[k] = *reinterpret_cast<const cvec*>(x + 4 + C * lane);
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < N; ++k) top = i0 + k * NW < ns ? fmaxf(top, st[k].x) : top;
        const float al = __builtin_amdgcn_exp2f(m - top);
        l *= al;
        o *= al;
        m = top;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (i0 + k * NW < ns) {
                const float w = __builtin_amdgcn_exp2f(st[k].x - m);
                l = fmaf(w, st[k].y, l);
#pragma unroll
                for (int c = 0; c < C; ++c) o[c] = fmaf(w, v[k][c], o[c]);
            }
        }
    }
    *reinterpret_cast<cvec*>(&mo[wave][C * lane]) = o;
    if (lane == 0) {
        mm[wave] = m;
        ml[wave] = l;
    }
    __syncthreads();
    if (tid >= 16) return;
    float gm = mm[0], den = 0.0f, x[CT];
#pragma unroll
    for (int w = 1; w < NW; ++w) gm = fmaxf(gm, mm[w]);
#pragma unroll
    for (int c = 0; c < CT; ++c) x[c] = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float wt = __builtin_amdgcn_exp2f(mm[w] - gm);
        den = fmaf(wt, ml[w], den);
#pragma unroll
        for (int c = 0; c < CT; ++c) x[c] = fmaf(wt, mo[w][CT * tid + c], x[c]);
    }
    const bool none = den == 0.0f;    // no position, or none on a page: zeros
    const float inv = 1.0f / den;
#pragma unroll
    for (int c = 0; c < CT; ++c) x[c] = none ? 0.0f : x[c] * inv;
    mxa::store<CT>(a.out, ((int64_t)p.b * a.M + r / a.G) * a.Hq + g * a.G + r % a.G, D, CT * tid, x);
}

struct Plan {
    int RT, groups, wanted, shares, most;   // shares the batch should and may have, and one sequence may
    int waves;   // of a workgroup
    bool one;
};
Plan plan(int B, int M, int Hq, int Hkv, int max_pos) {
    Plan p;
    const int64_t tiles = ((int64_t)M * (Hq / Hkv) + 15) / 16;
    p.groups = (int)((tiles + kMaxRT - 1) / kMaxRT);
    p.RT = (int)((tiles + p.groups - 1) / p.groups);
    // shares of the whole batch for one round of workgroups, none
    // below the 128 positions of a round of its waves
    const int kRound = p.RT == 1 ? 1024 : 512;   // four and two workgroups a CU
    int64_t longest = (max_pos + kMinShare * kUnit - 1) / (kMinShare * kUnit);   // shares a sequence may have (share_units)
    if (longest > kFew) longest = std::max<int64_t>(kFew, (longest + 1) / 2);
    const int64_t most = B * longest;
    const int64_t want = (kRound + (int64_t)Hkv * p.groups - 1) / ((int64_t)Hkv * p.groups);
    // Sequences enough for half the CUs, and short: one workgroup of 16 waves each and no merge.  32 / 4 heads, one
    // token, full caches, 16 waves / shares and merge, us: B = 64, 1024 positions 13.7 / 19.9, 2048 19.2 / 24.1; B = 32,
    // 2048 16.5 / 18.5; but B = 8, 2048 15.4 / 11.8, B = 1, 1024 10.8 / 8.1.
    const int64_t wgs = (int64_t)B * Hkv * p.groups;
    const bool wide = p.RT == 1 && longest > 1 && max_pos <= 2048 && wgs >= 128 && wgs <= 256;
    p.waves = wide ? 16 : 4;
    p.one = wide || longest == 1 || want * 4 <= B || (want == 1 && B == 1);
    p.wanted = (int)(want < most ? want : most);
    p.shares = p.one ? B : p.wanted + (B > 1 ? B : 0);
    p.most = (int)(longest < p.shares ? longest : p.shares);
    return p;
}

}  // namespace

extern "C" size_t mxfp4_attn_kv4_workspace_size(int B, int M, int Hq, int Hkv, int D, int max_pos) {
    if (B <= 0 || M <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || D <= 0 || max_pos <= 0) return 0;
    const Plan p = plan(B, M, Hq, Hkv, max_pos);
    return p.one ? 0 : (size_t)p.shares * M * Hq * (D + 4) * sizeof(float);
}

extern "C" int mxfp4_attn_kv4(const void* q, int q_dtype, int64_t ldq, const uint8_t* kq, const uint8_t* ks, const uint8_t* vq,
                              const uint8_t* vs, const int32_t* pages, int n_pages, int page, int max_pages,
                              const int32_t* dpos, void* o, int o_dtype, uint8_t* oq, uint8_t* os, int B, int M, int Hq,
                              int Hkv, int D, void* workspace, size_t workspace_bytes, void* stream) {
    Args a{};
    const int rc = kv4::make_cache(a.c, "attn_kv4", kq, ks, vq, vs, pages, n_pages, page, max_pages, B, Hkv, D);
    if (rc != MXFP4_OK) return rc;
    MXH_REQUIRE(q && dpos, "attn_kv4: null pointer");
    MXH_REQUIRE(q_dtype == MXFP4_DT_BF16 || q_dtype == MXFP4_DT_F16, "attn_kv4: q dtype %d (bf16 or fp16)", q_dtype);
    MXH_REQUIRE(M > 0 && M <= 65535 && Hq > 0 && Hq % Hkv == 0 && Hq <= 65535, "attn_kv4: M=%d Hq=%d Hkv=%d", M, Hq, Hkv);
    MXH_REQUIRE((int64_t)M * (Hq / Hkv) <= 65535 * 16, "attn_kv4: M*Hq/Hkv=%lld (up to %d)", (long long)M * (Hq / Hkv), 65535 * 16);
    MXH_REQUIRE(ldq >= (int64_t)Hq * D && ldq % 8 == 0 && ((uintptr_t)q & 15) == 0,
                "attn_kv4: q rows must be 16-byte aligned, at least Hq*D apart");
    MXH_REQUIRE(o || oq, "attn_kv4: no output (o and oq both null)");
    MXH_REQUIRE(!oq == !os, "attn_kv4: oq and os go together");
    MXH_REQUIRE(o_dtype >= MXFP4_DT_BF16 && o_dtype <= MXFP4_DT_F32, "attn_kv4: o dtype %d", o_dtype);
    MXH_REQUIRE((((uintptr_t)o) & 15) == 0 && ((uintptr_t)oq & 3) == 0, "attn_kv4: o must be 16-byte, oq 4-byte aligned");
    const Plan p = plan(B, M, Hq, Hkv, a.c.max_pos);
    MXH_REQUIRE((int64_t)M * Hq < (1ll << 31), "attn_kv4: M*Hq too large");
    const size_t need = mxfp4_attn_kv4_workspace_size(B, M, Hq, Hkv, D, a.c.max_pos);
    MXH_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                "attn_kv4: workspace must be 16-byte aligned and hold mxfp4_attn_kv4_workspace_size bytes");
    a.q = static_cast<const uint16_t*>(q);
    a.ldq = ldq;
    a.dpos = dpos;
    a.part = static_cast<float*>(workspace);
    a.out = mxa::Out{o, o_dtype, oq, os};
    a.B = B;
    a.M = M;
    a.Hq = Hq;
    a.G = Hq / Hkv;
    a.shares = p.shares;
    a.wanted = p.wanted;
    a.scale = (float)(1.4426950408889634 / sqrt((double)D));
    const hipStream_t st = mxh::as_stream(stream);
    const dim3 grid(p.shares, Hkv, p.groups);
#define MXH_K4(DD, RR, QQ)                                                                                              \
    if (p.waves == 16) {                                                                                               \
        if constexpr (RR == 1) hipLaunchKernelGGL((attn_kv4_kernel<DD, 1, QQ, true, 16>), grid, dim3(1024), 0, st, a); \
    } else if (p.one) {                                                                                                \
        hipLaunchKernelGGL((attn_kv4_kernel<DD, RR, QQ, true, 4>), grid, dim3(256), 0, st, a);                         \
    } else {                                                                                                           \
        hipLaunchKernelGGL((attn_kv4_kernel<DD, RR, QQ, false, 4>), grid, dim3(256), 0, st, a);                        \
    }
#define MXH_K4Q(DD, RR)                  \
    if (q_dtype == MXFP4_DT_BF16) {      \
        MXH_K4(DD, RR, 1);               \
    } else {                             \
        MXH_K4(DD, RR, 2);               \
    }
#define MXH_K4R(DD)                      \
    switch (p.RT) {                      \
        case 1: MXH_K4Q(DD, 1); break;   \
        default: MXH_K4Q(DD, 2); break;  \
    }
    if (D == 64) {
        MXH_K4R(64);
    } else {
        MXH_K4R(128);
    }
#undef MXH_K4R
#undef MXH_K4Q
#undef MXH_K4
    const int rl = mxh::launch_status("attn_kv4 (shares)");
    if (rl != MXFP4_OK || p.one) return rl;
    // 16 waves where a row has more records than four load at once
    const bool many = p.shares > kFew * B && p.most > kFew;
    const dim3 gm(M * Hq, B), bm(many ? 1024 : 256);
    if (D == 64) hipLaunchKernelGGL((many ? attn_kv4_merge_kernel<64, 16> : attn_kv4_merge_kernel<64, 4>), gm, bm, 0, st, a);
    else hipLaunchKernelGGL((many ? attn_kv4_merge_kernel<128, 16> : attn_kv4_merge_kernel<128, 4>), gm, bm, 0, st, a);
    return mxh::launch_status("attn_kv4 (merge)");
}
