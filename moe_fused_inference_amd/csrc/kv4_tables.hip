// kv4_tables.hip -- the page table of a batch from its sequences' lengths: pages come off and go
// back to a stack of free ones, and the newest tokens get their places.
//
// A sequence holds its pages in one range of its row, [lo, hi) (`span`), and below it those of the
// first `sinks` positions; what lies between went back behind its window.  From old and new range it is plain how many it gives back and takes;
// sums over the sequences before it say which of the call's R returned and A taken pages these are.
// Returned page r goes to place count + R - 1 - r of the stack and taken page a comes from place
// count + R - 1 - a, as if all were returned before any is taken: so taken page a < R is returned
// page a, handed on by the thread that returns it, the others are from the stack as it was, and no
// thread waits for another.
//
//   kv4_pages_kernel  every workgroup makes the sums of the whole batch (a few loads and a scan); the
//                     pages that move are dealt out over all threads, which find a page's sequence
//                     by search in the sums.  Alone, it does everything.
//   kv4_slots_kernel  otherwise: the tokens' places, and its last workgroup the ranges and the count,
//                     which the other launch's workgroups still read.
//
// Bound by the launch and by dependent loads: lengths, returned entries, the stack's, the tokens'.
// 48 sequences of up to 125 pages, nine tokens each, 4.7 us (6.1 with a wave a sequence), and 3.7 for
// the shorter lengths after it; 300 prompts of up to 4000 tokens in pages of 16 4.3 + 7.0 us, 2.7 TB/s
// of places written, and 4.5 + 2.8 for the pages' way back.
#include "attn_kv4.h"
#include "mx_host.h"

#include <algorithm>

namespace {

constexpr int kMostSequences = 4096;
constexpr int kMostTokens = 1 << 30, kMostPages = 1 << 30;      // (sums of tokens, and of pages that lack, end there)

struct Tables {
    int32_t* pages;
    int2* span;             // [lo, hi) of each sequence
    int32_t* free;
    int32_t* state;         // free pages, and pages that the sequences lack after the last call
    const int32_t* lens;
    const int32_t* news;    // or null
    int32_t* starts;        // of the tokens; or null, with slots, seq, pos
    int64_t* slots;
    int32_t* seq;
    int32_t* pos;
    int B, max_pages, n_pages, lg, window, sink_pages, T;
};

// A sequence's pages before the call and after it, and how many move.  No entry of the table is both returned and taken: the
// threads that do either do not wait for each other.
struct Range {
    int s, w, hi;      // pages 0 .. s - 1 of the sinks, and w .. hi - 1
};
struct Move {
    Range has, needs;
    int lo2;           // the new range's begin (needs.w, but for the sinks)
    int gone;          // pages that it needs and no call gives: gone back in an earlier one, or past its row
    __device__ __forceinline__ int back0() const { return max(0, has.s - needs.s); }
    __device__ __forceinline__ int back1() const { return max(0, min(needs.w, has.hi) - has.w); }
    __device__ __forceinline__ int from2() const { return max(has.w, max(needs.w, needs.hi)); }
    __device__ __forceinline__ int back() const { return back0() + back1() + max(0, has.hi - from2()); }
    __device__ __forceinline__ int back_at(int r) const {     // the r-th returned
        if (r < back0()) return needs.s + r;
        r -= back0();
        return r < back1() ? has.w + r : from2() + r - back1();
    }
    // Taken: of the sinks; before its range (where it begins anew), from its end on, so that what it gets is one range with
    // what it has; behind it
    __device__ __forceinline__ int take0() const { return max(0, needs.s - has.s); }
    __device__ __forceinline__ int top1() const { return min(has.w, needs.hi); }
    __device__ __forceinline__ int take1() const { return max(0, top1() - needs.w); }
    __device__ __forceinline__ int from() const { return max(needs.w, has.hi); }
    __device__ __forceinline__ int take() const { return take0() + take1() + max(0, needs.hi - from()); }
    __device__ __forceinline__ int take_at(int a) const {
        if (a < take0()) return has.s + a;
        a -= take0();
        return a < take1() ? top1() - 1 - a : from() + a - take1();
    }
    // Its range when it has got only the first `got` of them.
    __device__ __forceinline__ int2 range(int got) const {
        int lo = lo2, hi = needs.hi;
        if (got < take()) {
            const int rest = got - take0();
            if (rest >= 0 && rest < take1()) {
                lo = top1() - rest;
                hi = min(has.hi, needs.hi);
            } else {
                hi = take_at(got);
            }
        }
        return make_int2(min(lo, hi), hi);
    }
};
// What a sequence's moves come from: its range, length and new tokens.
struct Lengths {
    int lo, hi, len, news;
};
__device__ __forceinline__ Lengths lengths_of(const Tables& t, int b) {
    const int2 s = t.span[b];
    return Lengths{s.x, s.y, t.lens[b], t.news ? t.news[b] : 0};
}
__device__ __forceinline__ Move move_of(const Tables& t, const Lengths& x) {
    Move m;
    const int hi = min(max(x.hi, 0), t.max_pages), lo = min(max(x.lo, 0), hi), sinks = t.sink_pages;
    const int64_t room = (int64_t)t.max_pages << t.lg;
    const int64_t len = min((int64_t)max(x.len, 0), room);
    const int hi2 = (int)((len + (1 << t.lg) - 1) >> t.lg);
    int first = 0;                                      // the first page that a window of the call's first token, or the next, reaches
    if (t.window) first = (int)(max((int64_t)0, len - max(x.news, 0) - t.window + 1) >> t.lg);
    const bool anew = x.len > 0 && x.news >= x.len && lo > sinks;      // every position is new, and pages are gone
    m.lo2 = min(max(anew ? 0 : lo, first), hi2);
    m.gone = max(0, m.lo2 - max(first, sinks));
    if (x.len > room) {
        const int all = (int)(((int64_t)x.len + (1 << t.lg) - 1) >> t.lg);
        const int from = t.window ? (int)(max((int64_t)0, (int64_t)x.len - max(x.news, 0) - t.window + 1) >> t.lg) : 0;
        m.gone += max(0, all - max(t.max_pages, from)) + max(0, min(min(sinks, from), all) - t.max_pages);
    }
    m.has = Range{min(sinks, hi), max(lo, sinks), hi};
    m.needs = Range{min(sinks, hi2), max(m.lo2, sinks), hi2};
    return m;
}

// Sums over the sequences before each, of a batch of CAP at most, by NT threads.  KEEP: their lengths too, so that nothing
// is loaded again.
template <int NT, int CAP, bool KEEP>
struct Sums {
    static constexpr int kWaves = NT / 64;
    int back[CAP], take[CAP], token[CAP];
    uint32_t wave[3][kWaves];
    int total[3];
    unsigned long long gone;   // in all
    Lengths lengths[KEEP ? CAP : 1];
    __device__ __forceinline__ Lengths of(const Tables& t, int b) const {
        if constexpr (KEEP) return lengths[b];
        return lengths_of(t, b);
    }
};
__device__ __forceinline__ uint32_t capped_scan(uint32_t v) {      // wave_scan whose sums end at kMostTokens
    auto add = [](uint32_t a, uint32_t b) { return min(a + b, (uint32_t)kMostTokens); };
    v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true));
    v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true));
    v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true));
    v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true));
    v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
    v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
    return v;
}
template <int NT, int CAP, bool KEEP>
__device__ __forceinline__ void sum_up(const Tables& t, Sums<NT, CAP, KEEP>& s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t before[3] = {0, 0, 0};
    if (threadIdx.x == 0) s.gone = 0;
    for (int b0 = 0; b0 < t.B; b0 += NT) {
        const int b = b0 + threadIdx.x;
        uint32_t n[3] = {0, 0, 0}, to[3], gone = 0;
        if (b < t.B) {
            const Lengths x = lengths_of(t, b);
            const Move m = move_of(t, x);
            if constexpr (KEEP) s.lengths[b] = x;
            n[0] = m.back();
            n[1] = m.take();
            n[2] = min(max(x.news, 0), kMostTokens);
            gone = m.gone;
        }
        to[0] = mxa::wave_scan(n[0]);
        to[1] = mxa::wave_scan(n[1]);
        to[2] = capped_scan(n[2]);
        if (lane == 63)
            for (int i = 0; i < 3; ++i) s.wave[i][wave] = to[i];
        __syncthreads();
        if (__any(gone)) {                                       // seldom: no part of the sums
            const uint32_t all = capped_scan(gone);
            if (lane == 63) atomicAdd(&s.gone, (unsigned long long)all);
        }
        uint32_t at[3], sum[3];
        for (int i = 0; i < 3; ++i) {
            at[i] = sum[i] = before[i];
            for (int w = 0; w < Sums<NT, CAP, KEEP>::kWaves; ++w) {
                const uint32_t x = s.wave[i][w];
                if (w < wave) at[i] += x;
                sum[i] += x;
                if (i == 2) {
                    at[i] = min(at[i], (uint32_t)kMostTokens);
                    sum[i] = min(sum[i], (uint32_t)kMostTokens);
                }
            }
            before[i] = sum[i];
        }
        // (the sum before it: a capped one is not the sum with it less its own)
        const uint32_t prev = __shfl_up(to[2], 1);
        if (b < t.B) {
            s.back[b] = (int)(at[0] + to[0] - n[0]);
            s.take[b] = (int)(at[1] + to[1] - n[1]);
            s.token[b] = (int)min(at[2] + (lane ? prev : 0u), (uint32_t)kMostTokens);
        }
        if (b0 + NT < t.B) __syncthreads();
    }
    if (threadIdx.x == 0)
        for (int i = 0; i < 3; ++i) s.total[i] = (int)before[i];
    __syncthreads();
}

// The last sequence whose sum before it is at most i.
__device__ __forceinline__ int find(const int* sums, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sums[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The pages that move, by n threads of which this is the i-th.  count: free pages before the call.
template <class S>
__device__ __forceinline__ void move_pages(const Tables& t, const S& s, int i, int n, int count) {
    const int R = s.total[0], A = s.total[1];
    auto taken = [&](int a, int32_t id) {
        const int b = find(s.take, t.B, a);
        t.pages[(int64_t)b * t.max_pages + move_of(t, s.of(t, b)).take_at(a - s.take[b])] = id;
    };
    for (uint32_t r = i; r < (uint32_t)R; r += n) {
        const int b = find(s.back, t.B, (int)r);
        int32_t* const at = t.pages + (int64_t)b * t.max_pages + move_of(t, s.of(t, b)).back_at((int)r - s.back[b]);
        const int32_t id = *at;
        *at = -1;
        const int64_t place = (int64_t)count + R - 1 - r;
        if (place < t.n_pages) t.free[place] = id;
        if (r < (uint32_t)A) taken((int)r, id);                        // at once
    }
    for (uint32_t a = R + i; a < (uint32_t)A; a += n) {
        const int64_t place = (int64_t)count + R - 1 - a;
        if (place >= 0) taken((int)a, t.free[place]);
    }
}
// Sequence b's new range: what it took, where pages lack.
template <class S>
__device__ __forceinline__ int2 new_span(const Tables& t, const S& s, int b, int count) {
    const Move m = move_of(t, s.of(t, b));
    return m.range((int)min((int64_t)m.take(), max((int64_t)0, (int64_t)count + s.total[0] - s.take[b])));
}
__device__ __forceinline__ int free_count(const Tables& t) { return min(max(t.state[0], 0), t.n_pages); }
// Free pages after the call, and how many are needed and not there: R and A returned and taken, `gone` gone.
__device__ __forceinline__ int2 new_state(const Tables& t, int count, int R, int A, uint64_t gone) {
    const int64_t there = (int64_t)count + R, got = min((int64_t)A, there);
    return make_int2((int)min(there - got, (int64_t)t.n_pages), (int)min(A - got + gone, (uint64_t)kMostPages));
}

// Token `at`, of sequence b, at position p.
__device__ __forceinline__ int32_t page_of(const Tables& t, int b, int64_t p) {
    return p >= 0 && p < (int64_t)t.max_pages << t.lg ? t.pages[(int64_t)b * t.max_pages + (p >> t.lg)] : -1;
}
__device__ __forceinline__ void place_token(const Tables& t, int at, int b, int64_t p, int32_t id) {
    t.slots[at] = (uint32_t)id < (uint32_t)t.n_pages ? ((int64_t)id << t.lg) + (p & ((1 << t.lg) - 1)) : -1;
    t.seq[at] = b;
    t.pos[at] = (int32_t)p;
}
__device__ __forceinline__ void no_token(const Tables& t, int at) {
    t.slots[at] = -1;
    t.seq[at] = -1;
    t.pos[at] = -1;
}

template <int NT, int CAP, bool ALONE>
__global__ __launch_bounds__(NT) void kv4_pages_kernel(Tables t) {
    __shared__ Sums<NT, CAP, ALONE> s;
    const int count = free_count(t);
    sum_up(t, s);
    move_pages(t, s, (int)(blockIdx.x * NT + threadIdx.x), (int)(gridDim.x * NT), count);
    if (t.starts && blockIdx.x == 0)
        for (int b = threadIdx.x; b <= t.B; b += NT) t.starts[b] = b < t.B ? s.token[b] : s.total[2];
    if constexpr (ALONE) {
        for (int b = threadIdx.x; b < t.B; b += NT) t.span[b] = new_span(t, s, b, count);
        __syncthreads();                                 // the table is written, and the count has been read
        if (threadIdx.x == 0) *reinterpret_cast<int2*>(t.state) = new_state(t, count, s.total[0], s.total[1], s.gone);
        for (int at = threadIdx.x; at < t.T; at += NT) {
            if (at >= s.total[2]) {
                no_token(t, at);
                continue;
            }
            const int b = find(s.token, t.B, at);
            const Lengths x = s.of(t, b);
            const int64_t p = (int64_t)x.len - x.news + at - s.token[b];
            place_token(t, at, b, p, page_of(t, b, p));
        }
    }
}

// Workgroup (x, y): tokens of sequence x, part y of them, a thread kTokens at a time, and a share of the places past the
// last token.  The last x alone, past the sequences: the ranges and the count.
constexpr int kTokens = 4;
template <int NT, int CAP>
__global__ __launch_bounds__(NT) void kv4_slots_kernel(Tables t) {
    const int b = blockIdx.x, i = blockIdx.y * NT + threadIdx.x, n = gridDim.y * NT;
    if (t.starts) {                              // (every workgroup some, as the tokens may be few)
        const int64_t all = (int64_t)gridDim.x * n;
        for (int64_t at = (int64_t)t.starts[t.B] + (int64_t)b * n + i; at < t.T; at += all) no_token(t, (int)at);
    }
    if (b + 1 < (int)gridDim.x) {
        if (t.starts[b] >= t.T) return;
        const int start = t.starts[b], news = t.news[b], end = min(max(news, 0), t.T - start);
        const int64_t first = (int64_t)t.lens[b] - news;
        for (int j0 = i; j0 < end; j0 += kTokens * n) {
            int32_t id[kTokens];
#pragma unroll
            for (int k = 0; k < kTokens; ++k) id[k] = page_of(t, b, first + min(j0 + (int64_t)k * n, (int64_t)end - 1));
#pragma unroll
            for (int k = 0; k < kTokens; ++k) {
                const int64_t j = j0 + (int64_t)k * n;
                if (j < end) place_token(t, start + (int)j, b, first + j, id[k]);
            }
        }
        return;
    }
    if (blockIdx.y) return;
    __shared__ Sums<NT, CAP, false> s;
    const int count = free_count(t);
    sum_up(t, s);
    for (int q = threadIdx.x; q < t.B; q += NT) t.span[q] = new_span(t, s, q, count);      // (each reads its own alone)
    if (threadIdx.x == 0) *reinterpret_cast<int2*>(t.state) = new_state(t, count, s.total[0], s.total[1], s.gone);
}

// Entries of the table, and sequences, up to which one workgroup does everything.  us for two calls, nine tokens or as many
// as it says and the shorter lengths again, one workgroup / two launches, on the device: 48 sequences, 28800 entries 8.7 /
// 11.3, 8160 tokens 14.3 / 11.5; 300, 30000 entries, 8100 tokens 17.1 / 14.0, 20100 29.5 / 14.3, 90000 entries, 2700 tokens
// 12.3 / 14.2; 1000, 32000 entries, 2000 tokens 14.3 / 21.0, 8000 20.5 / 21.1, 20000 34.1 / 21.0, 100000 entries, 9000
// tokens 21.6 / 20.7; one, 2000 tokens 8.0 / 11.0, 8000 10.2 / 11.1, 20000 15.1 / 11.4.  So tokens decide, between 4000 and
// 8000 for most batches, and fewer launches are less for the host (9 / 17 us from Python); entries alone do not.
constexpr int64_t kFewEntries = 32768;
constexpr int kFewTokens = 8192, kFewSequences = 1024;
constexpr int kThreads = 512;

}  // namespace

extern "C" int mxfp4_kv4_tables(int32_t* pages, int32_t* span, int32_t* free, int32_t* state, const int32_t* lens,
                                const int32_t* news, int window, int sinks, int B, int max_pages, int n_pages, int page,
                                int32_t* starts, int64_t* slots, int32_t* seq, int32_t* pos, int T, void* stream) {
    MXH_REQUIRE(pages && span && free && state && lens, "kv4_tables: null pointer");
    MXH_REQUIRE((((uintptr_t)span | (uintptr_t)state) & 7) == 0, "kv4_tables: span and state must be 8-byte aligned");
    MXH_REQUIRE(B > 0 && B <= kMostSequences, "kv4_tables: B=%d (up to %d sequences)", B, kMostSequences);
    MXH_REQUIRE(max_pages > 0 && n_pages > 0, "kv4_tables: max_pages=%d n_pages=%d", max_pages, n_pages);
    MXH_REQUIRE(page >= kv4::kTile && (page & (page - 1)) == 0, "kv4_tables: page=%d must be a power of two from %d on", page, kv4::kTile);
    MXH_REQUIRE((int64_t)max_pages * page <= kv4::kMaxPos, "kv4_tables: more than 2^30 positions a sequence");
    MXH_REQUIRE((int64_t)B * max_pages < (1ll << 31), "kv4_tables: B*max_pages=%lld too large", (long long)B * max_pages);
    MXH_REQUIRE(window >= 0 && sinks >= 0 && (window > 0 || sinks == 0), "kv4_tables: window=%d sinks=%d", window, sinks);
    MXH_REQUIRE(!news == !starts, "kv4_tables: news and starts go together");
    MXH_REQUIRE(T >= 0 && T <= kMostTokens, "kv4_tables: T=%d", T);
    MXH_REQUIRE(T == 0 || (starts && slots && seq && pos), "kv4_tables: %d tokens without news or a place for them", T);
    MXH_REQUIRE(((uintptr_t)slots & 7) == 0, "kv4_tables: slots must be 8-byte aligned");
    int lg = 0;
    while ((1 << lg) < page) ++lg;
    const int sink_pages = sinks > 0 ? (int)(((int64_t)sinks + page - 1) >> lg) : 0;
    const Tables t{pages, reinterpret_cast<int2*>(span), free, state, lens, news, starts, slots, seq, pos, B, max_pages, n_pages, lg,
                   window, sink_pages, T};
    const hipStream_t st = mxh::as_stream(stream);
    if (B <= kFewSequences && (int64_t)B * max_pages <= kFewEntries && T <= kFewTokens) {
        hipLaunchKernelGGL((kv4_pages_kernel<1024, kFewSequences, true>), dim3(1), dim3(1024), 0, st, t);
        return mxh::launch_status("kv4_tables");
    }
    const int64_t entries = ((int64_t)B * max_pages + kThreads - 1) / kThreads;
    hipLaunchKernelGGL((kv4_pages_kernel<kThreads, kMostSequences, false>), dim3((unsigned)std::min<int64_t>(entries, 256)), dim3(kThreads),
                       0, st, t);
    const int rc = mxh::launch_status("kv4_tables");
    if (rc != MXFP4_OK) return rc;
    const int64_t parts = ((int64_t)T / B + kTokens * kThreads - 1) / (kTokens * kThreads);
    hipLaunchKernelGGL((kv4_slots_kernel<kThreads, kMostSequences>), dim3(T ? B + 1 : 1, (unsigned)(parts < 1 ? 1 : parts > 64 ? 64 : parts)),
                       dim3(kThreads), 0, st, t);
    return mxh::launch_status("kv4_tables (slots)");
}
