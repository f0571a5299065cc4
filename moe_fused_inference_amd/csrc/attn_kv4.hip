// attn_kv4.hip -- attention over the MXFP4 KV cache (kv4.h): M tokens of each of
// B sequences, token m of sequence b at dpos[b] + m over positions 0 .. dpos[b] + m,
// or of those the last ones and the first (a window with sinks), or with M drafts that
// form a tree its ancestors among them (attn_kv4.h, Masks).
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
//                          -> its output; attn_kv4_merge_rows_kernel, 16 rows.
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
// With a window a call is short, so the chains of latencies weigh more: 48 sequences, a
// window of 2000, 16.6 us in one launch (2.8 TB/s: 192 workgroups of 16 waves, each with a
// unit's loads ahead); one of 4096 9.7 (5.8 + 2.9: 1.4 until dpos is there, 2.1 for the
// first unit's bytes).  A tree of 26 drafts over 4026 positions 16.0: two units a wave
// behind 5 us of prologue, and the merge.  The second unit's K beside the first's was no
// faster (17.0 / 17.0, a window's piece of 512 tokens 23.2 / 23.6): what a wave waits for
// is the first bytes.
#include "attn_kv4_few.h"

#include <algorithm>

namespace {

// K by streaming loads where there is room for more bytes (the lengths are on the device): half the chip's last cache,
// past which nothing is there any more when the same cache's next call comes.  Plain / so, us: 32 sequences of up to 32768
// positions (571 MB) 59.0 / 55.9, 48 of 8192 (214 MB) 27.9 / 27.2.  Below it a cache that is read again at once stays: 48 of
// 4096 (107 MB) 28.9 / 29.7, 16 of 4096 17.3 / 18.0; where other caches come between, as in a step of many layers (1.5 GB
// of them in turn), it is the same: 31.8 / 31.7, 18.8 / 18.9, one of 32000 13.3 / 13.0.  V too: 48 of 8192 29.0 (its loads
// take half lines).
constexpr int64_t kMuch = 128ll << 20;

// Row r of kv head g, of sequence b: its records.
struct Records {
    int g, token, head, n;
    const float* at;
};
template <int D, int MASKS>
__device__ __forceinline__ Records records_of(const Args& a, int4 p, int base, int b, int row) {
    const int rows = a.M * a.G, g = (int)a.by_rows(row), r = row - g * rows, t = a.token(r);
    const int64_t pos = (int64_t)base + t;
    // those of the shares with its sequence's units up to the last that it sees
    uint32_t top = (uint32_t)(pos / kUnit);
    if constexpr (MASKS != 0) top = units<MASKS>(a, base).of_real((uint32_t)(last_seen<MASKS>(a, base, t) / kUnit));
    const int n = pos < 0 || pos >= a.c.max_pos ? 0 : min((int)(((uint32_t)p.y + top) / (uint32_t)p.z) + 1, a.shares - p.x);
    return Records{g, t, r - t * a.G, n, a.part + ((int64_t)row * a.records + p.x + b) * (D + 4)};
}

// Workgroup (row of kv head g: blockIdx.x = g * rows + r, sequence b): the row's
// records dealt to NW waves, eight loaded at a time (one memory latency for up to
// 8 NW), each with a running reference; a lane holds D / 64 columns.
template <int D, int NW, int MASKS>
__global__ __launch_bounds__(64 * NW) void attn_kv4_merge_kernel(Args a) {
    constexpr int C = D / 64, CT = D / 16, N = 8;
    typedef float cvec __attribute__((ext_vector_type(C)));
    __shared__ float mm[NW], ml[NW];
    __shared__ __align__(16) float mo[NW][D];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = blockIdx.y;
    const Records rs = records_of<D, MASKS>(a, a.places[b], a.dpos[b], b, blockIdx.x);
    const int ns = __builtin_amdgcn_readfirstlane(rs.n);
    const float* rec = rs.at;
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
        float mn = m;
#pragma unroll
        for (int k = 0; k < N; ++k) mn = i0 + k * NW < ns ? fmaxf(mn, st[k].x) : mn;
        const float al = __builtin_amdgcn_exp2f(m - mn);
        l *= al;
        o *= al;
        m = mn;
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
    store<CT>(a.out, ((int64_t)b * a.M + rs.token) * a.Hq + rs.g * a.G + rs.head, D, CT * tid, x);
}

// The same, to the same bits, where there are many rows of up to kFew records (Plan::across): 16 lanes a row, a lane D / 16 columns, with
// the four waves' sums of the kernel above as four in registers.
template <int D, int MASKS>
__global__ __launch_bounds__(256) void attn_kv4_merge_rows_kernel(Args a) {
    constexpr int CT = D / 16, N = 4;
    const int tid = threadIdx.x, t = tid & 15, b = blockIdx.y;
    const int row = blockIdx.x * 16 + (tid >> 4), total = a.M * a.Hq;
    const Records rs = records_of<D, MASKS>(a, a.places[b], a.dpos[b], b, min(row, total - 1));
    // the states of records t and t + 16, and the reference of those of t's class modulo 4
    float2 st[2];
    float ref = kNone;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        st[i] = make_float2(kNone, 0.0f);
        if (t + 16 * i < rs.n) st[i] = *reinterpret_cast<const float2*>(rs.at + (int64_t)(t + 16 * i) * (D + 4));
        ref = fmaxf(ref, st[i].x);
    }
    ref = fmaxf(ref, mx::dpp<0x124>(ref));               // row_ror 4, 8
    ref = fmaxf(ref, mx::dpp<0x128>(ref));
    float w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = __builtin_amdgcn_exp2f(st[i].x - ref);
    float l[N], o[N][CT];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        l[k] = 0.0f;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[k][c] = 0.0f;
    }
    for (int i0 = 0; __any(i0 < rs.n); i0 += N) {
        float4 v[N][CT / 4];
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int c = 0; c < CT / 4; ++c)
                v[k][c] = *reinterpret_cast<const float4*>(rs.at + (int64_t)min(i0 + k, max(rs.n - 1, 0)) * (D + 4) + 4 + CT * t + 4 * c);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int from = (i0 & 15) + k;
            const float wt = __shfl(i0 < 16 ? w[0] : w[1], from, 16), ly = __shfl(i0 < 16 ? st[0].y : st[1].y, from, 16);
            if (i0 + k < rs.n) {
                l[k] = fmaf(wt, ly, l[k]);
#pragma unroll
                for (int c = 0; c < CT; ++c) o[k][c] = fmaf(wt, reinterpret_cast<const float*>(&v[k][c / 4])[c % 4], o[k][c]);
            }
        }
    }
    float m[N], gm, den = 0.0f, x[CT];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        m[k] = __shfl(ref, k, 16);
        gm = k ? fmaxf(gm, m[k]) : m[k];
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) x[c] = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float wt = __builtin_amdgcn_exp2f(m[k] - gm);
        den = fmaf(wt, l[k], den);
#pragma unroll
        for (int c = 0; c < CT; ++c) x[c] = fmaf(wt, o[k][c], x[c]);
    }
    const bool none = den == 0.0f;    // no position, or none on a page: zeros
    const float inv = 1.0f / den;
#pragma unroll
    for (int c = 0; c < CT; ++c) x[c] = none ? 0.0f : x[c] * inv;
    if (row < total) store<CT>(a.out, ((int64_t)b * a.M + rs.token) * a.Hq + rs.g * a.G + rs.head, D, CT * t, x);
}

// room: positions of a sequence that its tokens may see together (room_of); fewer than there are: a window's.
Plan plan(int B, int M, int Hq, int Hkv, int max_pos, int room) {
    Plan p{};
    const bool window = room < max_pos;
    max_pos = room;
    const int64_t rows = (int64_t)M * (Hq / Hkv);
    int64_t longest = (max_pos + kMinShare * kUnit - 1) / (kMinShare * kUnit);   // shares a sequence may have (share_units)
    const int64_t across = longest + (B > 1 ? 1 : 0);                            // where it begins within one, and others are short
    if (longest > kFew) longest = std::max<int64_t>(kFew, (longest + 1) / 2);
    const int64_t most = B * (longest + (B > 1 ? kPad / kMinShare : 0));   // with a share of whole pads
    p.waves = 4;
    if (rows <= 16) p.groups = 1;
    else {
        p.many = true;
        p.groups = (int)((rows + 31) / 32);
    }
    const int64_t wgs = (int64_t)B * Hkv * p.groups;
    if (!p.many && !window) {
        // Sequences enough for half the CUs, and short: one workgroup of 16 waves each and no merge.  32 / 4 heads, one
        // token, full caches, 16 waves / shares and merge, us: B = 64, 1024 positions 13.7 / 19.9, 2048 19.2 / 24.1; B = 32,
        // 2048 16.5 / 18.5; but B = 8, 2048 15.4 / 11.8, B = 1, 1024 10.8 / 8.1.
        if (longest > 1 && max_pos <= 2048 && wgs >= 128 && wgs <= 256) p.waves = 16;
    }
    // shares of the whole batch for one round of workgroups, four or two a CU (up to 16 rows with a window three: four / three,
    // us: 8 sequences, 4096 positions 17.9 / 15.8, 32 of 8192 41.4 / 39.8, of 16384 67.6 / 62.1, one 10.1 / 10.1), and none that
    // starts a second round
    const int64_t want = std::max<int64_t>(1, (p.many ? 512 : window ? 768 : 1024) / ((int64_t)Hkv * p.groups));
    // A workgroup for a sequence, no shares and no merge, where there are many and short ones.  us, shares / one, one
    // token, sequences of one length and (in brackets) of 0 .. that: 512 workgroups, 2048 positions 43.9 / 31.1 (30.8 /
    // 26.0), 4096 63.5 / 57.3 (38.2 / 49.2); 2048 workgroups, 8192 positions 446 / 406 (238 / 247).  Nine tokens, 384
    // workgroups: 2048 positions 54.0 / 38.3 (43.0 / 36.6), 4096 79.5 / 69.0 (56.5 / 65.6).  One piece of a prompt of
    // 128 tokens, 128 workgroups: 1024 positions 22.7 / 15.8, 8192 49.8 / 84.1.
    // What it gives away is a batch of one long sequence among short ones, which the host cannot know: one of 8192 positions
    // among 255 of 64, eight kv heads, 32 / 142 (all of 8192: 406 / 376), one of 32768 among 63, 64 kv heads, 85 / 1048 (3008 / 2899).
    p.one = p.waves == 16 || longest == 1 || want * 4 <= B || (want == 1 && B == 1) || max_pos <= (p.many ? 8 : 4) * wgs;
    if (window) {
        // A window bounds what a long sequence among short ones takes, and most sequences fill it, so a workgroup has a
        // whole one further up: up to 16 rows of 16 waves, where each has a CU to itself.  us, shares / one (4, 16 waves), one
        // token, 8 query heads a kv head: 4 workgroups, 256 positions 8.5 / 7.7, 7.7, 512 8.6 / 9.5, 9.3; 32, 512 10.4 / 9.7,
        // 9.4, 1024 11.7 / 13.3, 12.2; 64, 2048 18.4 / 20.5, 17.5, 3000 18.6 / 26.0, 21.5; 128, 4096 28.5 / 37.2, 27.7, 8192
        // 41.5 / 70.0, 45.9; 256, 512 20.2 / 10.5, 11.1, 2048 29.3 / 21.8, 19.2, 8192 65.8 / 75.4, 59.0; 512, 2048 45.8 /
        // 30.8, 39.9, 8192 120 / 109, 114; 800, 1024 47.1 / 29.3, 48.9, 4096 103 / 91, 113.
        // More rows, shares / one: 4 workgroups, 128 positions 10.9 / 9.9, 256 10.9 / 11.7; 32, 256 12.4 / 11.8, 512 13.2 /
        // 14.7; 128, 1024 21.1 / 20.9 (one sequence), 22.9 / 20.5 (eight), 2048 25.6 / 30.7, 30.4 / 31.1; 256, 2048 33.1 / 31.2,
        // 39.9 / 31.6, 4096 48.0 / 50.1, 56.1 / 50.6; 400, 4096 78.3 / 69.0; 512, 8192 131 / 125, 145 / 127 (32 sequences).
        // The bounds take the slower form in two places of these: 32 workgroups, 1024 (12.2 for 11.7), and more rows of eight
        // sequences, 256, 4096 (56.1 for 50.6; of one 48.0 is the faster), as they do not ask how many sequences there are.
        const bool own = wgs <= 256;
        constexpr int few = 3 * kMinShare * kUnit;
        if (p.many) {
            p.one = p.one || max_pos <= 2 * kMinShare * kUnit || max_pos <= (wgs < 384 ? 15 : 24) * wgs;
        } else {
            p.one = p.one || max_pos <= few || max_pos <= (own ? 34 : 16) * wgs;
            if (p.one && own && max_pos > few) p.waves = 16;
        }
    }
    p.shares = p.one ? B : (int)std::min(want, most);
    p.records = p.shares + B - 1;
    p.most = (int)std::min<int64_t>(longest, p.shares);
    p.across = (int)std::min<int64_t>(across, p.shares);
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

template <int MASKS>
int merge(const Args& a, const Plan& p, int D, hipStream_t st) {
    // 16 lanes a row where there are many.  us, a workgroup / 16 lanes: 288 rows 12.9 / 18.5, 832 18.0 / 20.0, 1536 22.6 /
    // 23.2, 2048 23.6 / 22.8, 3328 28.3 / 26.4, 4096 47.9 / 44.1 (one sequence), 23.1 / 20.6 (eight).
    if (p.across <= kFew && (int64_t)a.B * a.M * a.Hq >= 2048) {
        const dim3 grid((a.M * a.Hq + 15) / 16, a.B);
        if (D == 64) hipLaunchKernelGGL((attn_kv4_merge_rows_kernel<64, MASKS>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((attn_kv4_merge_rows_kernel<128, MASKS>), grid, dim3(256), 0, st, a);
        return mxh::launch_status("attn_kv4 (merge of rows)");
    }
    const int nw = merge_waves(p, a.B);
    const dim3 grid(a.M * a.Hq, a.B), block(64 * nw);
#define MXH_M4(DD)                                                                                       \
    if (nw == 4) hipLaunchKernelGGL((attn_kv4_merge_kernel<DD, 4, MASKS>), grid, block, 0, st, a);      \
    else if (nw == 8) hipLaunchKernelGGL((attn_kv4_merge_kernel<DD, 8, MASKS>), grid, block, 0, st, a); \
    else hipLaunchKernelGGL((attn_kv4_merge_kernel<DD, 16, MASKS>), grid, block, 0, st, a)
    if (D == 64) { MXH_M4(64); } else { MXH_M4(128); }
#undef MXH_M4
    return mxh::launch_status("attn_kv4 (merge)");
}

// Positions of a sequence that its tokens may see together, rounded up to units: max_pos, or with a window (0: none) the
// sinks' units and those that M windows reach into.
int room_of(int M, int max_pos, int window, int sinks) {
    if (window == 0) return max_pos;
    const int64_t units = ((int64_t)sinks + kUnit - 1) / kUnit + ((int64_t)window + M + kUnit - 1) / kUnit + 1;
    return (int)std::min<int64_t>(max_pos, units * kUnit);
}

size_t workspace_of(const Plan& p, int B, int M, int Hq, int D) {
    return p.one ? 0 : (size_t)B * sizeof(int4) + (size_t)p.records * M * Hq * (D + 4) * sizeof(float);
}

}  // namespace

int mxa::attn_few(const Args& a, int q_dtype, const Plan& p, int D, bool much, hipStream_t st) {
    return launch_few<0>(a, q_dtype, p, D, much, st);
}

extern "C" size_t mxfp4_attn_kv4_workspace_size(int B, int M, int Hq, int Hkv, int D, int max_pos) {
    return mxfp4_attn_kv4_masked_workspace_size(B, M, Hq, Hkv, D, max_pos, 0, 0);
}

extern "C" size_t mxfp4_attn_kv4_masked_workspace_size(int B, int M, int Hq, int Hkv, int D, int max_pos, int window, int sinks) {
    if (!takes(B, M, Hq, Hkv, D, max_pos) || window < 0 || sinks < 0) return 0;
    return workspace_of(plan(B, M, Hq, Hkv, max_pos, room_of(M, max_pos, window, sinks)), B, M, Hq, D);
}

extern "C" int mxfp4_attn_kv4(const void* q, int q_dtype, int64_t ldq, const uint8_t* kq, const uint8_t* ks, const uint8_t* vq,
                              const uint8_t* vs, const int32_t* pages, int n_pages, int page, int max_pages,
                              const int32_t* dpos, void* o, int o_dtype, uint8_t* oq, uint8_t* os, int B, int M, int Hq,
                              int Hkv, int D, void* workspace, size_t workspace_bytes, void* stream) {
    return mxfp4_attn_kv4_masked(q, q_dtype, ldq, kq, ks, vq, vs, pages, n_pages, page, max_pages, dpos, 0, 0, nullptr, o, o_dtype, oq,
                                 os, B, M, Hq, Hkv, D, workspace, workspace_bytes, stream);
}

extern "C" int mxfp4_attn_kv4_masked(const void* q, int q_dtype, int64_t ldq, const uint8_t* kq, const uint8_t* ks, const uint8_t* vq,
                                     const uint8_t* vs, const int32_t* pages, int n_pages, int page, int max_pages,
                                     const int32_t* dpos, int window, int sinks, const int32_t* tree, void* o, int o_dtype,
                                     uint8_t* oq, uint8_t* os, int B, int M, int Hq, int Hkv, int D, void* workspace,
                                     size_t workspace_bytes, void* stream) {
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
    MXH_REQUIRE(window >= 0 && sinks >= 0, "attn_kv4: window=%d sinks=%d", window, sinks);
    MXH_REQUIRE(window > 0 || sinks == 0, "attn_kv4: sinks=%d without a window", sinks);
    // a token's line of ancestors is inside its window, which need not look where in the line each of them is
    MXH_REQUIRE(!tree || window == 0 || window >= M, "attn_kv4: a window of %d for a tree of %d", window, M);
    MXH_REQUIRE(((uintptr_t)tree & 3) == 0, "attn_kv4: tree must be 4-byte aligned");
    // p in three bf16 parts, all of fp32's 24 bits, for outputs that show them; for more than 16 rows to bf16 or fp16 alone,
    // in two: each rounds to nearest, so a term is off by 2^-18 of itself at most, an output by that of sum p |v|, 2^-9 (fp16:
    // 2^-6) of its own rounding's half step where its terms do not cancel.  The denominator sums fp32 terms.  A piece of 512 tokens over 8192
    // positions, two / three: 119 / 137 us; 0.23 % / 0.01 % of the bf16 outputs are the neighbour of the nearest (of fp32
    // torch operators 0.09 %), and the error against 64 bits, which is bf16's own, is 1.66e-3 of the norm for all three.
    const bool exact = (o && o_dtype == MXFP4_DT_F32) || oq;
    const bool asked = window > 0;
    if (window >= (int64_t)a.c.max_pos + (tree ? M : 0)) window = 0;      // it reaches every position
    if (window == 0) sinks = 0;
    const int room = room_of(M, a.c.max_pos, window, sinks);
    const Plan p = plan(B, M, Hq, Hkv, a.c.max_pos, room);
    // (the threads of a launch are counted in 32 bits)
    MXH_REQUIRE(p.one || (int64_t)M * Hq * merge_waves(p, B) * 64 < (1ll << 32), "attn_kv4: M*Hq=%lld too large", (long long)M * Hq);
    const size_t need = workspace_of(p, B, M, Hq, D);
    MXH_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                "attn_kv4: a workspace of %zu bytes, must be 16-byte aligned and hold %zu, which %s says", workspace ? workspace_bytes : 0,
                need, asked ? "mxfp4_attn_kv4_masked_workspace_size" : "mxfp4_attn_kv4_workspace_size");
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
    a.by_G = Divisor(a.G);
    a.by_rows = Divisor(M * a.G);
    a.by_shares = Divisor(p.shares);
    a.records = p.records;
    a.per = B == 1 && (int64_t)p.shares * kMinShare * kUnit >= room ? kMinShare : 0;
    a.window = window;
    a.sinks = std::min(sinks, a.c.max_pos);
    a.tree = reinterpret_cast<const uint32_t*>(tree);
    a.words = (M + 31) / 32;
    a.scale = (float)(1.4426950408889634 / sqrt((double)D));
    const hipStream_t st = mxh::as_stream(stream);
    const bool much = std::min((int64_t)B * room, (int64_t)n_pages * page) * Hkv * (D + D / 16) > kMuch;
    const int masks = (window ? kWindow : 0) | (tree ? kTree : 0);
    using Few = decltype(&attn_few);
    using Rows = decltype(&attn_rows);
    static constexpr Few few[4] = {attn_few, attn_few_window, attn_few_tree, attn_few_tree_window};
    static constexpr Rows rows[4] = {attn_rows, attn_rows_window, attn_rows_tree, attn_rows_tree_window};
    const int rl = p.many ? rows[masks](a, q_dtype, p, D, exact, st) : few[masks](a, q_dtype, p, D, much, st);
    if (rl != MXFP4_OK || p.one) return rl;
    static constexpr decltype(&merge<0>) join[4] = {merge<0>, merge<kWindow>, merge<kTree>, merge<kWindow | kTree>};
    return join[masks](a, p, D, st);
}
