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

namespace {

using kv4::Cache;

constexpr int kUnit = 32;              // positions per wave and step
constexpr float kSlack = 8.0f;         // a term is at most 2^8
constexpr float kWide = 262144.0f;     // a reference past it: an exponent's rounding is up to 2^-6 and more
constexpr float kNone = -3e38f;        // the reference of a row that has seen nothing: exp2(-inf - kNone) = 0
constexpr int kMaxRT = 2;              // 16-row tiles per workgroup
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
    int B, M, Hq, G, shares;     // shares: how many there may be, over the batch
    float scale;                 // log2(e) / sqrt(D)
};

// Units of sequence b, and what a share holds: equal whole rounds of the four waves.
__device__ __forceinline__ int units_of(const Args& a, int b) {
    const int64_t n = (int64_t)a.dpos[b] + a.M;
    const int np = (int)(n < 0 ? 0 : n < a.c.max_pos ? n : a.c.max_pos);
    return (np + kUnit - 1) / kUnit;
}
__device__ __forceinline__ int share_of(int64_t units, int wanted) {
    const int64_t per = (units + wanted - 1) / wanted;
    return (int)(per < 4 ? 4 : (per + 3) & ~3ll);
}
__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// The share's units, and for share number `at` of the batch its sequence b and its
// number there, or for at < 0 the first share of sequence b.  Every wave finds them
// by itself: a lane per sequence, sums over the wave.
struct Place {
    int per, b, s, first;
};
__device__ __forceinline__ bool find_share(const Args& a, int at, Place& p) {
    const int lane = threadIdx.x & 63;
    const int wanted = a.shares - a.B;      // the rounding up costs at most one a sequence
    if (a.B == 1) {
        const int nu = units_of(a, 0);
        p.per = share_of(nu, wanted);
        p.first = 0;
        p.b = 0;
        p.s = at;
        return at < 0 || at * (int64_t)p.per < nu;
    }
    int64_t total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) total += b0 + lane < a.B ? units_of(a, b0 + lane) : 0;
    p.per = share_of(wave_sum(total), wanted);
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int ns = b0 + lane < a.B ? (units_of(a, b0 + lane) + p.per - 1) / p.per : 0;
        int upto = ns;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(upto, o);
            if (lane >= o) upto += t;
        }
        if (at < 0) {
            if (p.b < b0 + 64) {
                p.first = before + __builtin_amdgcn_readlane(upto - ns, p.b - b0);
                return true;
            }
        } else {
            const uint64_t past = __ballot(before + upto > at);
            if (past) {
                const int l = (int)__builtin_ctzll(past);
                p.b = b0 + l;
                p.first = before + __builtin_amdgcn_readlane(upto - ns, l);
                p.s = at - p.first;
                return true;
            }
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// A unit's bytes as a lane loads them.  K: row 16 t + l16, D/8 bytes from D/8 lq on
// (so its dimensions are D/4 lq .., one block's or half a block's) and their code.
// V: positions 16 t + 4 lq + i, columns D/16 l16 ..; a position's codes as one word.
template <int D>
struct Raw {
    typedef uint32_t kvec __attribute__((ext_vector_type(D / 32)));
    typedef uint32_t svec __attribute__((ext_vector_type(D / 32)));   // four positions' codes
    kvec k[2];
    uint32_t ks[2];
    uint32_t v[8];
    svec vs[2];
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

template <int D>
__device__ __forceinline__ void load_k(Raw<D>& r, const Cache& c, const int64_t (&row)[2], const Lane<D>& o) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        r.k[t] = *reinterpret_cast<const typename Raw<D>::kvec*>(c.kq + row[t] * (D / 2) + o.k);
        r.ks[t] = *(c.ks + row[t] * (D / 32) + o.ks);
    }
}
template <int D>
__device__ __forceinline__ void load_v(Raw<D>& r, const Cache& c, const int64_t (&row)[2], const Lane<D>& o) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint8_t* p = c.vq + row[t] * (D / 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (D == 128) r.v[4 * t + i] = *reinterpret_cast<const uint32_t*>(p + (o.v + i * (D / 2)));
            else r.v[4 * t + i] = *reinterpret_cast<const uint16_t*>(p + (o.v + i * (D / 2)));
        }
        r.vs[t] = *reinterpret_cast<const typename Raw<D>::svec*>(c.vs + row[t] * (D / 32) + o.vs);
    }
}

// MFMA operands: kd[tile][kt] (positions x 8 dimensions), vd[c] (columns D/16 l16 + c x 8 positions).
template <int D>
__device__ __forceinline__ void decode_k(const Raw<D>& r, uint4 (&kd)[2][D / 32]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int kt = 0; kt < D / 32; ++kt) kd[t][kt] = kv4::eight_bf16(r.k[t][kt], kv4::scale_of(r.ks[t]));
}
template <int D>
__device__ __forceinline__ void decode_v(const Raw<D>& r, uint4 (&vd)[D / 16]) {
    const int l16 = threadIdx.x & 15;
    uint32_t o[D / 16][4];
#pragma unroll
    for (int p2 = 0; p2 < 4; ++p2) {       // positions 2 p2, 2 p2 + 1 of the lane's eight
        uint32_t x[2][D / 32];             // a position's columns, two a word
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * p2 + j;
            uint32_t code;
            if constexpr (D == 128) code = (r.vs[i >> 2][i & 3] >> (8 * (l16 >> 2))) & 0xFFu;
            else code = (r.vs[i >> 2][(i & 3) >> 1] >> (16 * (i & 1) + 8 * (l16 >> 3))) & 0xFFu;
            const float s = kv4::scale_of(code);
            x[j][0] = kv4::pair_bf16<0>(r.v[i], s);
            x[j][1] = kv4::pair_bf16<1>(r.v[i], s);
            if constexpr (D == 128) {
                x[j][2] = kv4::pair_bf16<2>(r.v[i], s);
                x[j][3] = kv4::pair_bf16<3>(r.v[i], s);
            }
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
            o[2 * w][p2] = __builtin_amdgcn_perm(x[1][w], x[0][w], 0x05040100u);
            o[2 * w + 1][p2] = __builtin_amdgcn_perm(x[1][w], x[0][w], 0x07060302u);
        }
    }
#pragma unroll
    for (int cc = 0; cc < D / 16; ++cc) vd[cc] = make_uint4(o[cc][0], o[cc][1], o[cc][2], o[cc][3]);
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

template <int D, int RT, int NQ, bool ONE>
__global__ __launch_bounds__(256, 2) void attn_kv4_kernel(Args a) {
    constexpr int R = 16 * RT, KT = D / 32, CT = D / 16;
    __shared__ __align__(16) uint16_t qs[RT > 1 ? NQ * R : 1][D + 8];
    __shared__ __align__(16) float mo[4][16][D + 4];
    __shared__ float mm[4][16], ml[4][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lq = lane >> 4;
    const int g = blockIdx.y, r0 = blockIdx.z * R, G = a.G;
    const int rows = a.M * G;
    Place pl;
    if constexpr (ONE) {
        pl.b = blockIdx.x;
        pl.s = 0;
    } else {
        if (!find_share(a, blockIdx.x, pl)) return;        // uniform
    }
    const int b = pl.b;
    const int64_t base = a.dpos[b];
    const int64_t last = base + a.M - 1 < a.c.max_pos - 1 ? base + a.M - 1 : a.c.max_pos - 1;   // positions past it are no one's
    int u0 = 0, u1 = (int)((last + kUnit) / kUnit);
    if constexpr (!ONE) {
        u0 = pl.s * pl.per;
        u1 = min(u1, u0 + pl.per);
    }
    // the group's last token sees no further
    const int64_t lim_min = base + r0 / G;                  // the first token of the group sees up to here
    const int64_t lim_max = base + (min(r0 + R, rows) - 1) / G;
    u1 = (int)(lim_max < (int64_t)u1 * kUnit ? (lim_max + kUnit) / kUnit : u1);
    if (!ONE && u0 >= u1) return;                           // no record: the merge reads none
    // the pages of the wave's units u0 + wave + 4 j, j = lane, tiles 0 and 1 (-1: none)
    int pid[2];
    auto load_pages = [&](int j0) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int64_t pos = ((int64_t)u0 + wave + 4 * (j0 + lane)) * kUnit + 16 * t;
            pid[t] = -1;
            if (pos < a.c.max_pos) {
                pid[t] = b;
                if (a.c.pages) {
                    const int id = a.c.pages[(int64_t)b * a.c.max_pages + (pos >> a.c.lg)];
                    pid[t] = (uint32_t)id < (uint32_t)a.c.n_pages ? id : -1;
                }
            }
        }
    };
    const Lane<D> off(lane);
    // unit u, the wave's j-th: its tiles' first head rows, and which of them exist
    auto locate = [&](int u, int j, int64_t (&row)[2]) -> int {
        int there = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int id = __builtin_amdgcn_readlane(pid[t], j & 63);
            const int pos = u * kUnit + 16 * t;
            const int in = a.c.pages ? pos & (a.c.page - 1) : pos;
            there |= id >= 0 ? 1 << t : 0;
            row[t] = id >= 0 ? ((int64_t)id * a.c.Hkv + g) * a.c.page + in : (int64_t)g * a.c.page;
        }
        return there;
    };
    // q: one tile's operands straight into registers, more through LDS.  zero[rt]: 0, or
    // NaN where the row holds an infinity or a NaN (then so is its output)
    const uint16_t* qb = a.q + (int64_t)b * a.M * a.ldq + (int64_t)g * G * D;
    auto q_row = [&](int r) { return qb + (int64_t)(r / G) * a.ldq + (r % G) * D; };
    uint4 q1[RT > 1 ? 1 : KT][NQ];
    float zero[RT];
    auto check = [](uint4 w) {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint16_t e = (uint16_t)(x[i / 2] >> (16 * (i & 1)));
            z = fmaf(NQ == 1 ? mx::bf16_to_f32(e) : mx::f16_to_f32(e), 0.0f, z);
        }
        return z;
    };
    if constexpr (RT == 1) {
        zero[0] = 0.0f;
        const uint16_t* row = q_row(min(r0 + l16, rows - 1)) + (D / 4) * lq;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            uint4 w = *reinterpret_cast<const uint4*>(row + 8 * kt);
            if (r0 + l16 >= rows) w = make_uint4(0, 0, 0, 0);
            zero[0] += check(w);
            q_parts<NQ>(w, q1[kt]);
        }
        zero[0] = over_lq<false>(zero[0]);
    } else {
        for (int i = tid; i < R * (D / 8); i += 256) {
            const int r = i / (D / 8), ch = i % (D / 8);
            uint4 w = make_uint4(0, 0, 0, 0), p[NQ];
            if (r0 + r < rows) w = *reinterpret_cast<const uint4*>(q_row(r0 + r) + 8 * ch);
            q_parts<NQ>(w, p);
#pragma unroll
            for (int j = 0; j < NQ; ++j) *reinterpret_cast<uint4*>(&qs[j * R + r][8 * ch]) = p[j];
        }
    }
    // the lane's query of tile rt: row r0 + 16 rt + l16; rows that are none see everything and write nothing
    int64_t lim[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = r0 + 16 * rt + l16;
        lim[rt] = r < rows ? base + r / G : INT64_MAX;
    }
    float m[RT], l[RT];
    bool wide[RT];   // uniform: a row's reference is past kWide
    mx::v4f acc[RT][CT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = kNone;
        l[rt] = 0.0f;
        wide[rt] = false;
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[rt][c] = mx::v4f{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (RT > 1) {
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            zero[rt] = 0.0f;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const uint4 w = *reinterpret_cast<const uint4*>(&qs[16 * rt + l16][(D / 4) * lq + 8 * kt]);
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) zero[rt] = fmaf(mx::bf16_to_f32((uint16_t)(x[i / 2] >> (16 * (i & 1)))), 0.0f, zero[rt]);
            }
            zero[rt] = over_lq<false>(zero[rt]);
        }
    }
    Raw<D> raw;
    int there = 0;
    if (u0 + wave < u1) {
        int64_t row[2];
        load_pages(0);
        there = locate(u0 + wave, 0, row);
        load_k(raw, a.c, row, off);
        load_v(raw, a.c, row, off);
    }
    for (int u = u0 + wave, j = 0; u < u1; u += 4, ++j) {
        const int64_t p0 = (int64_t)u * kUnit;
        const bool more = u + 4 < u1;
        int64_t next[2] = {0, 0};
        int there_next = 0;
        if (more) {
            if (((j + 1) & 63) == 0) load_pages(j + 1);
            there_next = locate(u + 4, j + 1, next);
        }
        uint4 kd[2][KT];
        decode_k(raw, kd);
        if (more) load_k(raw, a.c, next, off);
        uint4 p[RT][kParts];
        const bool masked = p0 + kUnit - 1 > lim_min || there != 3;   // uniform
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (rt > 0 && r0 + 16 * rt >= rows) break;
            mx::v4f s[2];
            s[0] = s[1] = mx::v4f{zero[rt], zero[rt], zero[rt], zero[rt]};
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    uint4 qf;
                    if constexpr (RT == 1) qf = q1[kt][n];
                    else qf = *reinterpret_cast<const uint4*>(&qs[n * R + 16 * rt + l16][(D / 4) * lq + 8 * kt]);
                    s[0] = mfma_bf16(kd[0][kt], qf, s[0]);
                    s[1] = mfma_bf16(kd[1][kt], qf, s[1]);
                }
            // s[t][i]: position p0 + 16 t + 4 lq + i
            if (masked) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(there >> t & 1) || p0 + 16 * t + 4 * lq + i > lim[rt]) s[t][i] = -INFINITY;
            }
            const float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                    fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            if (__ballot(top * a.scale > m[rt] + kSlack)) {
                const float mn = fmaxf(m[rt], over_lq<true>(top) * a.scale);
                if (u != u0 + wave) {
                    const float al = __builtin_amdgcn_exp2f(m[rt] - mn);
                    l[rt] *= al;
#pragma unroll
                    for (int c = 0; c < CT; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[rt][c][i] *= al;
                }
                m[rt] = mn;
                wide[rt] = __ballot(fabsf(mn) > kWide && mn != kNone) != 0ull;
            }
            float t[8];
            if (!wide[rt]) {
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = fmaf(s[i >> 2][i & 3], a.scale, -m[rt]);
            } else {   // the rounded product, as in m: the fma's would differ from it by more than a term
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = mul_then_sub(s[i >> 2][i & 3], a.scale, m[rt]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = __builtin_amdgcn_exp2f(t[i]);
            l[rt] += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
            parts<kParts>(t, p[rt]);
        }
        if (masked) {   // rows past the last token, and of no page, may hold anything: 0 * NaN must not reach a sum
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(there >> (i >> 2) & 1) || p0 + 16 * (i >> 2) + 4 * lq + (i & 3) > last) {
                    raw.v[i] = 0;
                    if constexpr (D == 128) raw.vs[i >> 2][i & 3] = 0x7F7F7F7Fu;
                    else raw.vs[i >> 2][(i & 3) >> 1] = (i & 1) ? (raw.vs[i >> 2][(i & 3) >> 1] & 0xFFFFu) | 0x7F7F0000u
                                                                : (raw.vs[i >> 2][(i & 3) >> 1] & 0xFFFF0000u) | 0x7F7Fu;
                }
        }
        uint4 vd[CT];
        decode_v(raw, vd);
        if (more) load_v(raw, a.c, next, off);
        there = there_next;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (rt > 0 && r0 + 16 * rt >= rows) break;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int k = kParts - 1; k >= 0; --k) acc[rt][c] = mfma_bf16(vd[c], p[rt][k], acc[rt][c]);
        }
    }
    // the four waves' sums of each tile in LDS, then one record (or the output) per
    // row: acc[rt][c][i] is column D/16 (4 lq + i) + c of query l16
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt > 0) __syncthreads();
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
        if (rr >= rows) continue;
        const int64_t pos = base + rr / G;
        if (!ONE && (pos < 0 || pos >= a.c.max_pos || (int64_t)u0 * kUnit > pos)) continue;   // no record: the merge reads none
        const float gm = fmaxf(fmaxf(mm[0][qr], mm[1][qr]), fmaxf(mm[2][qr], mm[3][qr]));
        float o[CT], den = 0.0f;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
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

// Workgroup (row of kv head g: blockIdx.x = g * rows + r, sequence b), 4 waves a
// quarter of the records each, a lane D / 64 columns.
template <int D>
__global__ __launch_bounds__(256) void attn_kv4_merge_kernel(Args a) {
    constexpr int C = D / 64;
    typedef float cvec __attribute__((ext_vector_type(C)));
    __shared__ float red[4], dred[4];
    __shared__ float nred[4][D];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rows = a.M * a.G;
    Place p;
    p.b = blockIdx.y;
    find_share(a, -1, p);
    const int g = blockIdx.x / rows, r = blockIdx.x - g * rows;
    const int64_t pos = (int64_t)a.dpos[p.b] + r / a.G;
    const int ns = pos < 0 || pos >= a.c.max_pos ? 0 : (int)(pos / ((int64_t)p.per * kUnit)) + 1;   // shares of positions 0 .. pos
    const float* rec = a.part + ((int64_t)blockIdx.x * a.shares + p.first) * (D + 4);
    float gm = kNone;
    for (int i = tid; i < ns; i += 256) gm = fmaxf(gm, rec[(int64_t)i * (D + 4)]);
    gm = mx::wave_reduce_dpp<true>(gm);
    if (lane == 0) red[wave] = gm;
    __syncthreads();
    gm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float den = 0.0f;
    cvec num = 0.0f;
#pragma unroll 8
    for (int i = wave; i < ns; i += 4) {
        const float* x = rec + (int64_t)i * (D + 4);
        const float2 st = *reinterpret_cast<const float2*>(x);
        const cvec v = *reinterpret_cast<const cvec*>(x + 4 + C * lane);
        const float w = __builtin_amdgcn_exp2f(st.x - gm);
        den = fmaf(w, st.y, den);
#pragma unroll
        for (int c = 0; c < C; ++c) num[c] = fmaf(w, v[c], num[c]);
    }
    *reinterpret_cast<cvec*>(&nred[wave][C * lane]) = num;
    if (lane == 0) dred[wave] = den;
    __syncthreads();
    constexpr int CT = D / 16;
    if (tid >= 16) return;
    den = (dred[0] + dred[1]) + (dred[2] + dred[3]);
    const bool none = den == 0.0f;    // no position, or none on a page: zeros
    const float inv = 1.0f / den;
    float o[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int k = CT * tid + c;
        o[c] = none ? 0.0f : ((nred[0][k] + nred[1][k]) + (nred[2][k] + nred[3][k])) * inv;
    }
    mxa::store<CT>(a.out, ((int64_t)p.b * a.M + r / a.G) * a.Hq + g * a.G + r % a.G, D, CT * tid, o);
}

struct Plan {
    int RT, groups, shares;
    bool one;
};
Plan plan(int B, int M, int Hq, int Hkv, int max_pos) {
    Plan p;
    const int64_t tiles = ((int64_t)M * (Hq / Hkv) + 15) / 16;
    p.groups = (int)((tiles + kMaxRT - 1) / kMaxRT);
    p.RT = (int)((tiles + p.groups - 1) / p.groups);
    // shares of the whole batch for one round of workgroups (two per CU), none
    // below the 128 positions of a round of its waves
    const int64_t most = (int64_t)B * ((max_pos + 4 * kUnit - 1) / (4 * kUnit));
    const int64_t want = (512 + (int64_t)Hkv * p.groups - 1) / ((int64_t)Hkv * p.groups);
    p.one = most == B || want * 4 <= B;
    p.shares = p.one ? B : (int)(want < most ? want : most) + B;
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
    a.scale = (float)(1.4426950408889634 / sqrt((double)D));
    const hipStream_t st = mxh::as_stream(stream);
    const dim3 grid(p.shares, Hkv, p.groups);
#define MXH_K4(DD, RR, QQ)                                                                                  \
    if (p.one) hipLaunchKernelGGL((attn_kv4_kernel<DD, RR, QQ, true>), grid, dim3(256), 0, st, a);          \
    else hipLaunchKernelGGL((attn_kv4_kernel<DD, RR, QQ, false>), grid, dim3(256), 0, st, a)
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
    if (D == 64) hipLaunchKernelGGL(attn_kv4_merge_kernel<64>, dim3(M * Hq, B), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(attn_kv4_merge_kernel<128>, dim3(M * Hq, B), dim3(256), 0, st, a);
    return mxh::launch_status("attn_kv4 (merge)");
}
