// attn_kv4.hip -- attention over the MXFP4 KV cache (kv4.h): M tokens of each of
// B sequences, token m of sequence b at dpos[b] + m over positions 0 .. dpos[b] + m.
//
//   attn_kv4_kernel        workgroup (share of the batch, kv head g), up to 16 query
//                          rows (tokens x heads of the kv head): a wave takes every
//                          fourth unit of 32 of the share's positions, with its own
//                          running softmax; the waves' sums meet in LDS -> one record
//                          (reference, sum, D column sums) per row, share and
//                          sequence in it, or the output where a workgroup has a
//                          whole sequence.
//   attn_kv4_rows_kernel   the same for more rows (attn_kv4_rows.hip).
//   attn_kv4_merge_kernel  workgroup (kv head's row, sequence): the row's records
//                          -> its output.
//
// Shares.  dpos lives on the device, so the host fixes only how many shares there
// may be (a round of workgroups); every workgroup adds up the batch's lengths, and
// a share is the same number of units of all sequences laid end to end, so that
// long and short ones load the chip alike.
//
// Mathematics.  Both products are transposed, S^T = K Q^T and O^T = V^T P^T: an
// MFMA leaves a lane with four positions of each of two 16-position tiles of one
// query, which is its B operand of the second product as it stands, so P passes
// through no LDS.  K and V are bf16, which holds every cache value, two values an
// instruction by the scaled conversion.  P is bf16 parts whose sum is the fp32
// probability at any size.  m is the reference of a row's terms, not their maximum:
// it moves to the maximum only where a lane's terms sum past kMost.
//
// What bounds it.  A long batch: memory.  32 sequences of up to 32768 positions (267 MB,
// four heads of 128, eight query heads each) 56.2 us, of which 4.8 the merge, 5.2 TB/s in
// the shares' kernel; a plain streaming read 6.1 TB/s.  Eight sequences of 65536: 107 us,
// 5.35 TB/s in all.  For that: 128 registers, so four waves a SIMD, each with a unit's loads
// ahead (4.3 KB; 69 KB a CU).  Two ahead by buffer descriptors 74 us, V through LDS 68.
// A short call: two launches, each one dependent chain of memory latencies (dpos, page,
// rows; records): 500 positions 4.5 + 3.2 us, 32000 8.1 + 4.9 (5.0 + 3.3 and 9.0 + 5.0
// before a share of one sequence loaded its first unit ahead of dpos).
// Rows are apart: a row's reference moves by its own terms, and values that are not finite
// are kept from the tokens before them (mark_not_finite).  Both are code off the loop's
// path; it costs 48 sequences 26.4 -> 26.5 us, 7 x 3 tokens of 5 heads 8.95 -> 9.1.
#include "attn_kv4.h"
#include "kv4.h"
#include "mx_device.h"
#include "mx_host.h"

#include <algorithm>
#include <type_traits>

namespace {

using namespace mxa;

constexpr int kParts = 3;              // bf16 parts of a probability
// K by streaming loads where there is room for more bytes (the lengths are on the device): half the chip's last cache,
// past which nothing is there any more when the same cache's next call comes.  Plain / so, us: 32 sequences of up to 32768
// positions (571 MB) 59.0 / 55.9, 48 of 8192 (214 MB) 27.9 / 27.2.  Below it a cache that is read again at once stays: 48 of
// 4096 (107 MB) 28.9 / 29.7, 16 of 4096 17.3 / 18.0; where other caches come between, as in a step of many layers (1.5 GB
// of them in turn), it is the same: 31.8 / 31.7, 18.8 / 18.9, one of 32000 13.3 / 13.0.  V too: 48 of 8192 29.0 (its loads
// take half lines).
constexpr int64_t kMuch = 128ll << 20;

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

template <int D, int NQ, Work W, int NW, bool STREAM>
__global__ __launch_bounds__(64 * NW, 4) void attn_kv4_kernel(Args a) {
    constexpr bool ONE = W == Work::kSequence;
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
        // q, whose parts go to LDS once the first units' loads are on their way
        const uint16_t* qb = a.q + (int64_t)b * a.M * a.ldq + (int64_t)g * G * D;
        constexpr int NT = 64 * NW, QN = (R * (D / 8) + NT - 1) / NT;
        uint4 qw[QN];
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int r = (tid + NT * i) / (D / 8), ch = (tid + NT * i) % (D / 8);
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
        auto first_loads = [&]() {
            uint32_t row[2];
            find_rows(0);
            there = locate(0, row);
            load_k<STREAM>(r, a.c, row, off);
            load_v(r, a.c, row, off);
        };
        if constexpr (W == Work::kShare) first_loads();        // of a share of fixed length before dpos is there: what no token sees is masked
        base = __builtin_amdgcn_readfirstlane(base);
        // Positions fit 31 bits: a token before the cache is put at -1, one past it at its end
        auto clamped = [&](int64_t pos) { return (int)(pos < 0 ? -1 : pos < a.c.max_pos ? pos : a.c.max_pos); };
        const int last = min(clamped((int64_t)base + a.M - 1), a.c.max_pos - 1);      // positions past it are no one's
        const int lim_min = clamped(base);                            // the first token sees up to here
        u1 = min(u1, (last + kUnit) / kUnit);
        if constexpr (W == Work::kShare) {
            if (u0 >= u1) return;                               // no record: the merge reads none
        } else {
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
        const int lim = l16 < rows ? clamped((int64_t)base + l16 / G) : 1 << 30;
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
            const int p0 = u * kUnit;
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
            const bool masked = __builtin_amdgcn_readfirstlane(p0 + kUnit - 1 > lim_min || there != 3);
            if (masked) {
                int sees = lim - p0 - 4 * lq;        // the last position that the lane's query sees
                asm volatile("" : "+v"(sees));       // (nothing below is computed ahead of the branch)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!(there >> (i >> 2) & 1) || 16 * (i >> 2) + (i & 3) > sees) s[i] = -INFINITY;
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
                if (p0 + kUnit - 1 > lim_min && lim_min < last) {   // nor may what only some rows see reach the others'
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
        if (__builtin_amdgcn_readfirstlane(dirty)) mark_not_finite<D, NW>(a, b, base, g, 0, rows, wave, u0, u1, lim_min, last, mo[wave]);
        __syncthreads();
        // thread: CT columns of a row (8 of 128, 4 of 64)
        const int qr = tid >> 4;
        if (tid < 256 && qr < rows) finish<D, NW, ONE>(a, tid, b, base, g, qr, u0, [&](int w) { return mm[w][qr]; }, [&](int w) { return ml[w][qr]; }, [&](int w, int c) { return *reinterpret_cast<const float4*>(&mo[w][qr][c]); });
    };
    each_segment<W>(a, segment);
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
    const int b = blockIdx.y, g = blockIdx.x / rows, r = blockIdx.x - g * rows;
    const int4 p = a.places[b];
    const int64_t pos = (int64_t)a.dpos[b] + r / a.G;
    // its records: those of the shares with its sequence's units 0 .. pos / kUnit
    const int ns = __builtin_amdgcn_readfirstlane(
        pos < 0 || pos >= a.c.max_pos ? 0 : min((int)(((uint32_t)p.y + (uint32_t)(pos / kUnit)) / (uint32_t)p.z) + 1, a.shares - p.x));
    const float* rec = a.part + ((int64_t)blockIdx.x * a.records + __builtin_amdgcn_readfirstlane(p.x) + b) * (D + 4);
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
    store<CT>(a.out, ((int64_t)b * a.M + r / a.G) * a.Hq + g * a.G + r % a.G, D, CT * tid, x);
}

struct Plan {
    bool many;       // rows for attn_rows
    int groups, shares, most;   // shares of the batch (with `one` a sequence each), and one sequence may have
    int records;     // of a row
    int waves;       // of a workgroup
    bool one;
};
Plan plan(int B, int M, int Hq, int Hkv, int max_pos) {
    Plan p{};
    const int64_t rows = (int64_t)M * (Hq / Hkv);
    int64_t longest = (max_pos + kMinShare * kUnit - 1) / (kMinShare * kUnit);   // shares a sequence may have (share_units)
    if (longest > kFew) longest = std::max<int64_t>(kFew, (longest + 1) / 2);
    const int64_t most = B * (longest + (B > 1 ? kPad / kMinShare : 0));   // with a share of whole pads
    p.waves = 4;
    if (rows <= 16) {
        p.groups = 1;
        // Sequences enough for half the CUs, and short: one workgroup of 16 waves each and no merge.  32 / 4 heads, one
        // token, full caches, 16 waves / shares and merge, us: B = 64, 1024 positions 13.7 / 19.9, 2048 19.2 / 24.1; B = 32,
        // 2048 16.5 / 18.5; but B = 8, 2048 15.4 / 11.8, B = 1, 1024 10.8 / 8.1.
        const int64_t wgs = (int64_t)B * Hkv;
        if (longest > 1 && max_pos <= 2048 && wgs >= 128 && wgs <= 256) p.waves = 16;
    } else {
        p.many = true;
        p.groups = (int)((rows + 31) / 32);
    }
    // shares of the whole batch for one round of workgroups, four or two a CU, and none that starts a second round
    const int64_t want = std::max<int64_t>(1, (p.many ? 512 : 1024) / ((int64_t)Hkv * p.groups));
    // A workgroup for a sequence, no shares and no merge, where there are many and short ones.  us, shares / one, one
    // token, sequences of one length and (in brackets) of 0 .. that: 512 workgroups, 2048 positions 43.9 / 31.1 (30.8 /
    // 26.0), 4096 63.5 / 57.3 (38.2 / 49.2); 2048 workgroups, 8192 positions 446 / 406 (238 / 247).  Nine tokens, 384
    // workgroups: 2048 positions 54.0 / 38.3 (43.0 / 36.6), 4096 79.5 / 69.0 (56.5 / 65.6).  One piece of a prompt of
    // 128 tokens, 128 workgroups: 1024 positions 22.7 / 15.8, 8192 49.8 / 84.1.
    // What it gives away is a batch of one long sequence among short ones, which the host cannot know: one of 8192 positions
    // among 255 of 64, eight kv heads, 32 / 142 (all of 8192: 406 / 376), one of 32768 among 63, 64 kv heads, 85 / 1048 (3008 / 2899).
    const int64_t wgs = (int64_t)B * Hkv * p.groups;
    p.one = p.waves == 16 || longest == 1 || want * 4 <= B || (want == 1 && B == 1) || max_pos <= (p.many ? 8 : 4) * wgs;
    p.shares = p.one ? B : (int)std::min(want, most);
    p.records = p.shares + B - 1;
    p.most = (int)std::min<int64_t>(longest, p.shares);
    return p;
}

// The sizes that the entry takes (plan's integers are good for these).
constexpr int64_t kMostRows = 65535 * 16;    // of a kv head: M * Hq / Hkv
bool takes_heads(int M, int Hq, int Hkv) {
    return M > 0 && M <= 65535 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq <= 65535;
}
bool takes(int B, int M, int Hq, int Hkv, int D, int max_pos) {
    return B > 0 && B <= 65535 && takes_heads(M, Hq, Hkv) && (int64_t)M * (Hq / Hkv) <= kMostRows && (D == 64 || D == 128) &&
           max_pos > 0 && max_pos <= kv4::kMaxPos;
}

// Waves of a merge: about as many as load a row's records at once.  4 / 8 / 16, us: nine tokens over 23001 positions (42
// shares) 23.4 / 23.4 / 25.2; one token over 16000, 16 heads (64 shares) 15.8 / 15.3 / 16.3
int merge_waves(const Plan& p, int B) { return p.shares <= kFew * B || p.most <= kFew ? 4 : p.most <= 2 * kFew ? 8 : 16; }

int merge(const Args& a, const Plan& p, int D, hipStream_t st) {
    const int nw = merge_waves(p, a.B);
    const dim3 grid(a.M * a.Hq, a.B), block(64 * nw);
#define MXH_M4(DD)                                                                               \
    if (nw == 4) hipLaunchKernelGGL((attn_kv4_merge_kernel<DD, 4>), grid, block, 0, st, a);      \
    else if (nw == 8) hipLaunchKernelGGL((attn_kv4_merge_kernel<DD, 8>), grid, block, 0, st, a); \
    else hipLaunchKernelGGL((attn_kv4_merge_kernel<DD, 16>), grid, block, 0, st, a)
    if (D == 64) { MXH_M4(64); } else { MXH_M4(128); }
#undef MXH_M4
    return mxh::launch_status("attn_kv4 (merge)");
}

}  // namespace

extern "C" size_t mxfp4_attn_kv4_workspace_size(int B, int M, int Hq, int Hkv, int D, int max_pos) {
    if (!takes(B, M, Hq, Hkv, D, max_pos)) return 0;
    const Plan p = plan(B, M, Hq, Hkv, max_pos);
    return p.one ? 0 : (size_t)B * sizeof(int4) + (size_t)p.records * M * Hq * (D + 4) * sizeof(float);
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
    MXH_REQUIRE(takes_heads(M, Hq, Hkv), "attn_kv4: M=%d Hq=%d Hkv=%d", M, Hq, Hkv);
    MXH_REQUIRE((int64_t)M * (Hq / Hkv) <= kMostRows, "attn_kv4: M*Hq/Hkv=%lld (up to %lld)", (long long)M * (Hq / Hkv),
                (long long)kMostRows);
    MXH_REQUIRE(ldq >= (int64_t)Hq * D && ldq % 8 == 0 && ((uintptr_t)q & 15) == 0,
                "attn_kv4: q rows must be 16-byte aligned, at least Hq*D apart");
    MXH_REQUIRE(o || oq, "attn_kv4: no output (o and oq both null)");
    MXH_REQUIRE(!oq == !os, "attn_kv4: oq and os go together");
    MXH_REQUIRE(o_dtype >= MXFP4_DT_BF16 && o_dtype <= MXFP4_DT_F32, "attn_kv4: o dtype %d", o_dtype);
    MXH_REQUIRE((((uintptr_t)o) & 15) == 0 && ((uintptr_t)oq & 3) == 0, "attn_kv4: o must be 16-byte, oq 4-byte aligned");
    // p in three bf16 parts, all of fp32's 24 bits, for outputs that show them; for more than 16 rows to bf16 or fp16 alone,
    // in two: each rounds to nearest, so a term is off by 2^-18 of itself at most, an output by that of sum p |v|, 2^-9 (fp16:
    // 2^-6) of its own rounding's half step where its terms do not cancel.  The denominator sums fp32 terms.  A piece of 512 tokens over 8192
    // positions, two / three: 119 / 137 us; 0.23 % / 0.01 % of the bf16 outputs are the neighbour of the nearest (of fp32
    // torch operators 0.09 %), and the error against 64 bits, which is bf16's own, is 1.66e-3 of the norm for all three.
    const bool exact = (o && o_dtype == MXFP4_DT_F32) || oq;
    const Plan p = plan(B, M, Hq, Hkv, a.c.max_pos);
    // (the threads of a launch are counted in 32 bits)
    MXH_REQUIRE(p.one || (int64_t)M * Hq * merge_waves(p, B) * 64 < (1ll << 32), "attn_kv4: M*Hq=%lld too large", (long long)M * Hq);
    const size_t need = mxfp4_attn_kv4_workspace_size(B, M, Hq, Hkv, D, a.c.max_pos);
    MXH_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                "attn_kv4: workspace must be 16-byte aligned and hold mxfp4_attn_kv4_workspace_size bytes");
    a.q = static_cast<const uint16_t*>(q);
    a.ldq = ldq;
    a.dpos = dpos;
    a.places = static_cast<int4*>(workspace);
    a.part = reinterpret_cast<float*>(a.places + B);
    a.out = Out{o, o_dtype, oq, os};
    a.B = B;
    a.M = M;
    a.Hq = Hq;
    a.G = Hq / Hkv;
    a.shares = p.shares;
    a.records = p.records;
    a.per = B == 1 && (int64_t)p.shares * kMinShare * kUnit >= a.c.max_pos ? kMinShare : 0;
    a.scale = (float)(1.4426950408889634 / sqrt((double)D));
    const hipStream_t st = mxh::as_stream(stream);
    if (p.many) {
        const int rr = attn_rows(a, q_dtype, p.groups, D, p.one, exact, st);
        if (rr != MXFP4_OK || p.one) return rr;
        return merge(a, p, D, st);
    }
    const dim3 grid(p.shares, Hkv);
    const bool much = std::min((int64_t)B * a.c.max_pos, (int64_t)n_pages * page) * Hkv * (D + D / 16) > kMuch;
#define MXH_W4(DD, QQ, W)                                                                                          \
    if (much) hipLaunchKernelGGL((attn_kv4_kernel<DD, QQ, Work::W, 4, true>), grid, dim3(256), 0, st, a);          \
    else hipLaunchKernelGGL((attn_kv4_kernel<DD, QQ, Work::W, 4, false>), grid, dim3(256), 0, st, a)
#define MXH_K4(DD, QQ)                                                                                                        \
    if (p.waves == 16) hipLaunchKernelGGL((attn_kv4_kernel<DD, QQ, Work::kSequence, 16, false>), grid, dim3(1024), 0, st, a); \
    else if (p.one) { MXH_W4(DD, QQ, kSequence); }                                                                            \
    else if (B == 1) { MXH_W4(DD, QQ, kShare); }                                                                              \
    else { MXH_W4(DD, QQ, kLine); }
    if (D == 64) {
        if (q_dtype == MXFP4_DT_BF16) { MXH_K4(64, 1); } else { MXH_K4(64, 2); }
    } else {
        if (q_dtype == MXFP4_DT_BF16) { MXH_K4(128, 1); } else { MXH_K4(128, 2); }
    }
#undef MXH_K4
#undef MXH_W4
    const int rl = mxh::launch_status("attn_kv4 (shares)");
    if (rl != MXFP4_OK || p.one) return rl;
    return merge(a, p, D, st);
}
