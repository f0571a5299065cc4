// kv4_tree.hip -- what a tree of drafts needs besides its attention (attn_kv4.hip): its masks
// before a step's layers, and the accepted path's rows moved together after them.
//
//   tree_masks_kernel  parents -> each draft's ancestors and itself as bits, and its depth.
//                      A wave takes 64 consecutive drafts: by doubling (six steps over the
//                      lanes) each has its line within them, as 64 bits, and where the line
//                      leaves them.  Parents come before their children, so a draft's words
//                      are then its 64 bits, those of where it left, and so on back.
//   kv4_keep_kernel    row dpos[b] + path[b][k] -> dpos[b] + k of every layer's cache.
//
// Both are bound by the launch and a few dependent loads.
#include "kv4.h"
#include "mx_host.h"

namespace {

constexpr int kMostDrafts = 4096;
constexpr int kThreads = 256;

// Workgroup (sequence, kThreads drafts from c0 on), which makes the bits of the drafts before them too.
__global__ __launch_bounds__(kThreads) void tree_masks_kernel(const int32_t* __restrict__ parents, uint32_t* __restrict__ tree,
                                                              int32_t* __restrict__ depth, int M) {
    extern __shared__ uint64_t lds[];
    const int b = blockIdx.x, c0 = blockIdx.y * kThreads, words = (M + 31) / 32;
    const int top = min(M, c0 + kThreads), blocks = (top + 63) / 64;
    uint64_t* const bits = lds;                                  // of each draft, within its 64
    int* const out = reinterpret_cast<int*>(lds + 64 * blocks);  // where its line goes on: an earlier 64's draft, -1 nowhere, -2 it is none
    const int lane = threadIdx.x & 63;
    for (int k = threadIdx.x >> 6; k < blocks; k += kThreads / 64) {
        const int m = 64 * k + lane;
        const int p = m < M ? parents[(int64_t)b * M + m] : -2;
        const bool valid = p >= -1 && p < m;
        uint64_t a = valid ? 1ull << lane : 0;
        int link = valid && p >= 64 * k ? p - 64 * k : lane;     // itself where the line leaves
        int to = valid ? p : -2;
#pragma unroll
        for (int s = 0; s < 6; ++s) {
            const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)a, link), hi = (uint32_t)__shfl((int)(uint32_t)(a >> 32), link);
            to = __shfl(to, link);
            link = __shfl(link, link);
            a |= (uint64_t)hi << 32 | lo;
        }
        bits[m] = a;
        out[m] = to;
    }
    __syncthreads();
    const int m = c0 + threadIdx.x;
    if (m >= M) return;
    int n = 0, at = m;
    while (at >= 0) {
        n += __builtin_popcountll(bits[at]);
        at = out[at];
    }
    const bool none = at == -2;
    depth[(int64_t)b * M + m] = none ? -1 : n - 1;
    uint32_t* const row = tree + ((int64_t)b * M + m) * words;
    at = none ? -1 : m;
    for (int k = (words - 1) / 2; k >= 0; --k) {
        uint64_t a = 0;
        if (at >= 64 * k) {
            a = bits[at];
            at = out[at];
        }
        row[2 * k] = (uint32_t)a;
        if (2 * k + 1 < words) row[2 * k + 1] = (uint32_t)(a >> 32);
    }
}

constexpr int kLayers = 64;      // of a launch
struct Layers {
    uint8_t* t[kLayers][4];      // kq, ks, vq, vs
};

// Workgroup (sequence and kv head, layer): a thread 16 bytes of a row's nibbles, or its codes, of keys or of values, of as
// many drafts as there are threads for.  What is moved is read before any of it is written; a later round reads only rows
// from its own drafts on (path[b][k] >= k), and writes none before.
template <int D>
__global__ __launch_bounds__(kThreads) void kv4_keep_kernel(Layers layers, kv4::Cache c, const int32_t* __restrict__ dpos,
                                                            const int32_t* __restrict__ path, int A) {
    constexpr int Q = D / 32, kItems = 2 * Q + 2, R = kThreads / kItems;
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    const int b = blockIdx.x / c.Hkv, g = blockIdx.x - b * c.Hkv, lane = threadIdx.x & 63;
    const int32_t* const line = path + (int64_t)b * A;
    uint8_t* const* const t = layers.t[blockIdx.y];
    const int64_t base = dpos[b];
    const int k = threadIdx.x / kItems, item = threadIdx.x - k * kItems;
    int n = A;                                                    // its drafts, up to the first that is none
    for (int i0 = 0; i0 < A; i0 += 64) {
        const uint64_t end = __ballot(i0 + lane < A && line[min(i0 + lane, A - 1)] < 0);
        if (end) {
            n = i0 + (int)__builtin_ctzll(end);
            break;
        }
    }
    for (int k0 = 0; k0 < n; k0 += R) {
        const int i = k0 + k;
        int64_t from = -1, to = -1;
        if (k < R && i < n) {
            const int64_t src = base + line[i], dst = base + i;
            if (line[i] > i && dst >= 0 && src < c.max_pos) {
                from = kv4::head_row(c, b, g, (int)src);
                to = kv4::head_row(c, b, g, (int)dst);
            }
        }
        const bool moves = from >= 0 && to >= 0;
        v4u w = 0;
        uint8_t* const q = t[item < Q ? 0 : 2] + 16 * (item < Q ? item : item - Q);     // of a nibble item
        uint8_t* const s = t[item == 2 * Q ? 1 : 3];                                    // of a code item
        if (moves) {
            if (item < 2 * Q) w = *reinterpret_cast<const v4u*>(q + from * (D / 2));
            else if constexpr (D == 128) w[0] = *reinterpret_cast<const uint32_t*>(s + from * 4);
            else w[0] = *reinterpret_cast<const uint16_t*>(s + from * 2);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // the rows are here, not on their way, when another wave writes
        __syncthreads();
        if (moves) {
            if (item < 2 * Q) *reinterpret_cast<v4u*>(q + to * (D / 2)) = w;
            else if constexpr (D == 128) *reinterpret_cast<uint32_t*>(s + to * 4) = w[0];
            else *reinterpret_cast<uint16_t*>(s + to * 2) = (uint16_t)w[0];
        }
    }
}

}  // namespace

extern "C" int mxfp4_tree_masks(const int32_t* parents, int32_t* tree, int32_t* depth, int B, int M, void* stream) {
    MXH_REQUIRE(parents && tree && depth, "tree_masks: null pointer");
    MXH_REQUIRE(B > 0 && B <= 65535 && M > 0 && M <= kMostDrafts, "tree_masks: B=%d M=%d (up to %d drafts)", B, M, kMostDrafts);
    const int chunks = (M + kThreads - 1) / kThreads;
    const size_t lds = (size_t)((M + 63) / 64 * 64) * (sizeof(uint64_t) + sizeof(int));
    hipLaunchKernelGGL(tree_masks_kernel, dim3(B, chunks), dim3(kThreads), lds, mxh::as_stream(stream), parents,
                       reinterpret_cast<uint32_t*>(tree), depth, M);
    return mxh::launch_status("tree_masks");
}

extern "C" int mxfp4_kv4_keep(uint8_t* const* kq, uint8_t* const* ks, uint8_t* const* vq, uint8_t* const* vs, int n_layers,
                              const int32_t* pages, int n_pages, int page, int max_pages, const int32_t* dpos,
                              const int32_t* path, int B, int A, int Hkv, int D, void* stream) {
    MXH_REQUIRE(kq && ks && vq && vs && dpos && path, "kv4_keep: null pointer");
    MXH_REQUIRE(n_layers > 0 && n_layers <= 65535, "kv4_keep: n_layers=%d", n_layers);
    MXH_REQUIRE(A > 0, "kv4_keep: A=%d", A);
    kv4::Cache c;
    for (int l = 0; l < n_layers; ++l) {
        const int rc = kv4::make_cache(c, "kv4_keep", kq[l], ks[l], vq[l], vs[l], pages, n_pages, page, max_pages, B, Hkv, D);
        if (rc != MXFP4_OK) return rc;
    }
    MXH_REQUIRE((int64_t)B * Hkv < (1 << 24), "kv4_keep: B*Hkv=%lld too large", (long long)B * Hkv);
    for (int l0 = 0; l0 < n_layers; l0 += kLayers) {
        const int n = n_layers - l0 < kLayers ? n_layers - l0 : kLayers;
        Layers t{};
        for (int l = 0; l < n; ++l) {
            t.t[l][0] = kq[l0 + l];
            t.t[l][1] = ks[l0 + l];
            t.t[l][2] = vq[l0 + l];
            t.t[l][3] = vs[l0 + l];
        }
        const dim3 grid(B * Hkv, n);
        if (D == 64) hipLaunchKernelGGL(kv4_keep_kernel<64>, grid, dim3(kThreads), 0, mxh::as_stream(stream), t, c, dpos, path, A);
        else hipLaunchKernelGGL(kv4_keep_kernel<128>, grid, dim3(kThreads), 0, mxh::as_stream(stream), t, c, dpos, path, A);
        const int rc = mxh::launch_status("kv4_keep");
        if (rc != MXFP4_OK) return rc;
    }
    return MXFP4_OK;
}
