// kv4_tables.hip -- the page table of a batch from its sequences' lengths: pages come off and go
// back to a stack of free ones, and the newest tokens get their places.
//
// A sequence holds its pages in one range of its row, [lo, hi) (`span`), and below it those of the
// first `sinks` positions.  From old and new range it is plain how many it gives back and takes;
// sums over the sequences before it say which of the call's R returned and A taken pages these are.
// Returned page r goes to place count + R - 1 - r of the stack and taken page a comes from place
// count + R - 1 - a, as if all were returned before any is taken: so taken page a < R is returned
// page a, handed on by the thread that returns it, the others are from the stack as it was, and no
// thread waits for another.
//
//   kv4_pages_kernel  every workgroup makes the sums of the whole batch (a few loads and a scan) and
//                     moves the pages of some sequences.  Alone, it does everything.
//   kv4_slots_kernel  otherwise: the tokens' places, and its first workgroup the ranges and the count,
//                     which the other launch's workgroups still read.
//
// Bound by the launch and by dependent loads: lengths, returned entries, the stack's, the tokens'.
#include "attn_kv4.h"
#include "mx_host.h"

namespace {

constexpr int kMostSequences = 4096;
constexpr int kMostTokens = 1 << 30;

struct Tables {
    int32_t* pages;
    int2* span;             // [lo, hi) of each sequence
    int32_t* free;
    int32_t* state;         // free pages, and pages that the last call lacked
    const int32_t* lens;
    const int32_t* news;    // or null
    int32_t* starts;        // of the tokens; or null, with slots, seq, pos
    int64_t* slots;
    int32_t* seq;
    int32_t* pos;
    int B, max_pages, n_pages, lg, window, sink_pages, T;
};

// A sequence's pages before the call and after it, and how many move.
struct Move {
    int lo, hi, lo2, hi2, s1, s2, w1, w2;      // ranges; the ends of the sinks' pages; where the windows' begin
    __device__ __forceinline__ int back0() const { return max(0, s1 - s2); }
    __device__ __forceinline__ int back1() const { return max(0, min(w2, hi) - w1); }
    __device__ __forceinline__ int from2() const { return max(w1, max(w2, hi2)); }
    __device__ __forceinline__ int back() const { return back0() + back1() + max(0, hi - from2()); }
    __device__ __forceinline__ int back_at(int r) const {     // the r-th returned
        if (r < back0()) return s2 + r;
        r -= back0();
        return r < back1() ? w1 + r : from2() + r - back1();
    }
    __device__ __forceinline__ int take0() const { return max(0, s2 - s1); }
    __device__ __forceinline__ int take() const { return take0() + max(0, hi2 - max(w2, hi)); }
    __device__ __forceinline__ int take_at(int a) const { return a < take0() ? s1 + a : max(w2, hi) + a - take0(); }
};
__device__ __forceinline__ Move move_of(const Tables& t, int b) {
    Move m;
    const int2 s = t.span[b];
    m.hi = min(max(s.y, 0), t.max_pages);
    m.lo = min(max(s.x, 0), m.hi);
    const int64_t room = (int64_t)t.max_pages << t.lg;
    const int64_t len = min((int64_t)max(t.lens[b], 0), room);
    m.hi2 = (int)((len + (1 << t.lg) - 1) >> t.lg);
    int64_t first = 0;                                  // the first page that a window of the call's first token, or the next, reaches
    if (t.window) first = max((int64_t)0, len - max(t.news ? t.news[b] : 0, 0) - t.window + 1) >> t.lg;
    m.lo2 = (int)min(max((int64_t)m.lo, first), (int64_t)m.hi2);
    m.s1 = min(t.sink_pages, m.hi);
    m.s2 = min(t.sink_pages, m.hi2);
    m.w1 = max(m.lo, t.sink_pages);
    m.w2 = max(m.lo2, t.sink_pages);
    return m;
}

// Sums over the sequences before each, of a batch, by NT threads.
template <int NT>
struct Sums {
    static constexpr int kWaves = NT / 64;
    int back[kMostSequences], take[kMostSequences], token[kMostSequences];
    uint32_t wave[3][kWaves];
    int total[3];
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
template <int NT>
__device__ __forceinline__ void sum_up(const Tables& t, Sums<NT>& s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t before[3] = {0, 0, 0};
    for (int b0 = 0; b0 < t.B; b0 += NT) {
        const int b = b0 + threadIdx.x;
        uint32_t n[3] = {0, 0, 0}, to[3];
        if (b < t.B) {
            const Move m = move_of(t, b);
            n[0] = m.back();
            n[1] = m.take();
            n[2] = t.news ? min(max(t.news[b], 0), kMostTokens) : 0;
        }
        to[0] = mxa::wave_scan(n[0]);
        to[1] = mxa::wave_scan(n[1]);
        to[2] = capped_scan(n[2]);
        if (lane == 63)
            for (int i = 0; i < 3; ++i) s.wave[i][wave] = to[i];
        __syncthreads();
        uint32_t at[3], sum[3];
        for (int i = 0; i < 3; ++i) {
            at[i] = sum[i] = before[i];
            for (int w = 0; w < Sums<NT>::kWaves; ++w) {
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
        if (b < t.B) {
            s.back[b] = (int)(at[0] + to[0] - n[0]);
            s.take[b] = (int)(at[1] + to[1] - n[1]);
            // (the sum before it: a capped one is not the sum with it less its own)
            const uint32_t prev = __shfl_up(to[2], 1);
            s.token[b] = (int)min(at[2] + (lane ? prev : 0u), (uint32_t)kMostTokens);
        }
        __syncthreads();
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

// The pages of sequence b, by n threads of which this is the i-th.  count: free pages before the call; R, A: the call's.
template <int NT>
__device__ __forceinline__ void move_pages(const Tables& t, const Sums<NT>& s, int b, int i, int n, int count) {
    const Move m = move_of(t, b);
    const int R = s.total[0], A = s.total[1];
    int32_t* const row = t.pages + (int64_t)b * t.max_pages;
    for (int k = i; k < m.back(); k += n) {
        const int r = s.back[b] + k, at = m.back_at(k);
        const int32_t id = row[at];
        row[at] = -1;
        const int64_t place = (int64_t)count + R - 1 - r;
        if (place < t.n_pages) t.free[place] = id;
        if (r < A) {                                    // taken at once
            const int to = find(s.take, t.B, r);
            t.pages[(int64_t)to * t.max_pages + move_of(t, to).take_at(r - s.take[to])] = id;
        }
    }
    for (int k = i; k < m.take(); k += n) {
        const int64_t place = (int64_t)count + R - 1 - (s.take[b] + k);
        if (place >= 0 && place < count) row[m.take_at(k)] = t.free[place];
    }
}
// Sequence b's new range: what it took, where pages lack.
template <int NT>
__device__ __forceinline__ int2 new_span(const Tables& t, const Sums<NT>& s, int b, int count) {
    const Move m = move_of(t, b);
    const int n = m.take(), got = (int)min((int64_t)n, max((int64_t)0, (int64_t)count + s.total[0] - s.take[b]));
    int hi = m.hi2;
    if (got < n) hi = got < m.take0() ? m.s1 + got : max(m.w2, m.hi) + got - m.take0();
    return make_int2(min(m.lo2, hi), hi);
}
__device__ __forceinline__ int free_count(const Tables& t) { return min(max(t.state[0], 0), t.n_pages); }
// Free pages after the call, and how many lacked.
__device__ __forceinline__ int2 new_state(const Tables& t, int count, int R, int A) {
    const int64_t there = (int64_t)count + R;
    return make_int2((int)min(there - min((int64_t)A, there), (int64_t)t.n_pages), (int)(A - min((int64_t)A, there)));
}

// The tokens of sequence b, the first of which is token `start`, by n threads of which this is the i-th.
__device__ __forceinline__ void place_tokens(const Tables& t, int b, int start, int i, int n) {
    const int count = min(max(t.news[b], 0), t.T - start);
    const int64_t first = (int64_t)t.lens[b] - t.news[b], room = (int64_t)t.max_pages << t.lg;
    for (int j = i; j < count; j += n) {
        const int64_t p = first + j;
        int64_t slot = -1;
        if (p >= 0 && p < room) {
            const int32_t id = t.pages[(int64_t)b * t.max_pages + (p >> t.lg)];
            if ((uint32_t)id < (uint32_t)t.n_pages) slot = ((int64_t)id << t.lg) + (p & ((1 << t.lg) - 1));
        }
        t.slots[start + j] = slot;
        t.seq[start + j] = b;
        t.pos[start + j] = (int32_t)p;
    }
}
__device__ __forceinline__ void no_token(const Tables& t, int at) {
    t.slots[at] = -1;
    t.seq[at] = -1;
    t.pos[at] = -1;
}

template <int NT, bool ALONE>
__global__ __launch_bounds__(NT) void kv4_pages_kernel(Tables t) {
    __shared__ Sums<NT> s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int count = free_count(t);
    sum_up(t, s);
    if constexpr (ALONE) {
        for (int b = wave; b < t.B; b += NT / 64) move_pages(t, s, b, lane, 64, count);
    } else {
        for (int b = blockIdx.x; b < t.B; b += gridDim.x) move_pages(t, s, b, threadIdx.x, NT, count);
    }
    if (t.starts && blockIdx.x == 0)
        for (int b = threadIdx.x; b <= t.B; b += NT) t.starts[b] = b < t.B ? s.token[b] : s.total[2];
    if constexpr (ALONE) {
        __syncthreads();                                 // every range has been read, and the table is written
        for (int b = threadIdx.x; b < t.B; b += NT) t.span[b] = new_span(t, s, b, count);      // (each reads its own alone)
        if (threadIdx.x == 0) *reinterpret_cast<int2*>(t.state) = new_state(t, count, s.total[0], s.total[1]);
        if (!t.starts) return;
        for (int b = wave; b < t.B; b += NT / 64)
            if (s.token[b] < t.T) place_tokens(t, b, s.token[b], lane, 64);
        for (int i = s.total[2] + threadIdx.x; i < t.T; i += NT) no_token(t, i);
    }
}

// Workgroup (x, y): tokens of sequence x, part y of them; past the sequences, those that there are none of.  The last x
// alone: the ranges and the count.
template <int NT>
__global__ __launch_bounds__(NT) void kv4_slots_kernel(Tables t) {
    const int b = blockIdx.x, i = blockIdx.y * NT + threadIdx.x, n = gridDim.y * NT;
    if (b < t.B) {
        if (t.starts && t.starts[b] < t.T) place_tokens(t, b, t.starts[b], i, n);
        return;
    }
    if (t.starts)
        for (int64_t at = (int64_t)t.starts[t.B] + i; at < t.T; at += n) no_token(t, (int)at);
    if (blockIdx.y) return;
    __shared__ Sums<NT> s;
    const int count = free_count(t);
    sum_up(t, s);
    for (int q = threadIdx.x; q < t.B; q += NT) t.span[q] = new_span(t, s, q, count);
    if (threadIdx.x == 0) *reinterpret_cast<int2*>(t.state) = new_state(t, count, s.total[0], s.total[1]);
}

// Entries of the table up to which one workgroup does everything.
constexpr int64_t kFewEntries = 32768;
constexpr int kFewTokens = 8192;

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
                   window, sink_pages < max_pages ? sink_pages : max_pages, T};
    const hipStream_t st = mxh::as_stream(stream);
    if ((int64_t)B * max_pages <= kFewEntries && T <= kFewTokens) {
        hipLaunchKernelGGL((kv4_pages_kernel<1024, true>), dim3(1), dim3(1024), 0, st, t);
        return mxh::launch_status("kv4_tables");
    }
    hipLaunchKernelGGL((kv4_pages_kernel<256, false>), dim3(B < 256 ? B : 256), dim3(256), 0, st, t);
    const int rc = mxh::launch_status("kv4_tables");
    if (rc != MXFP4_OK) return rc;
    const int64_t parts = ((int64_t)T / B + 1023) / 1024;
    hipLaunchKernelGGL(kv4_slots_kernel<256>, dim3(B + 1, (unsigned)(parts < 1 ? 1 : parts > 64 ? 64 : parts)), dim3(256), 0, st, t);
    return mxh::launch_status("kv4_tables (slots)");
}
