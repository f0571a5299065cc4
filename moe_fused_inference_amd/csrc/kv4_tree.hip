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
// Both are bound by the launch and a few dependent loads: one tree of 26 drafts 1.7 us, 64 of 500
// 4.5; a path's five rows in 48 layers 4.4, 32 paths 7.5 (0.9 TB/s of rows, read and written, that are 64 and 4 bytes).
#include "kv4.h"
#include "mx_host.h"

namespace {

constexpr int kMostDrafts = 4096;
constexpr int kThreads = 256;

// Workgroup (sequence, 64 drafts from c0 on), which makes the bits of the drafts before them too; then four threads a
// draft, each every fourth 64 bits of its row, so that what they store lies together.  64 trees of 500, us: 6.0 with a
// thread a draft and 256 drafts a workgroup.  WIDE: a row is whole words of 64 bits.
template <bool WIDE>
__global__ __launch_bounds__(kThreads) void tree_masks_kernel(const int32_t* __restrict__ parents, uint32_t* __restrict__ tree,
                                                              int32_t* __restrict__ depth, int M) {
    extern __shared__ uint64_t lds[];
    const int b = blockIdx.x, c0 = blockIdx.y * 64, words = (M + 31) / 32, blocks = blockIdx.y + 1;
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
    const int m = c0 + (threadIdx.x >> 2), part = threadIdx.x & 3;
    if (m >= M) return;
    int n = 0, at = m;
    while (at >= 0) {
        n += __builtin_popcountll(bits[at]);
        at = out[at];
    }
    const bool none = at == -2;
    if (part == 0) depth[(int64_t)b * M + m] = none ? -1 : n - 1;
    uint32_t* const row = tree + ((int64_t)b * M + m) * words;
    at = none ? -1 : m;
    for (int k = (words - 1) / 2; k >= 0; --k) {
        uint64_t a = 0;
        if (at >= 64 * k) {
            a = bits[at];
            at = out[at];
        }
        if ((k & 3) != part) continue;
        if constexpr (WIDE) {
            *reinterpret_cast<uint64_t*>(row + 2 * k) = a;
        } else {
            row[2 * k] = (uint32_t)a;
            if (2 * k + 1 < words) row[2 * k + 1] = (uint32_t)(a >> 32);
        }
    }
}

constexpr int kLayers = 64;      // of a launch
struct Layers {
    uint8_t* t[kLayers][4];      // kq, ks, vq, vs
};

constexpr int kAtOnce = 4;       // of a workgroup

// Workgroup (sequence and kv head, kAtOnce layers) of T threads: a thread 16 bytes of a row's nibbles, or its codes, of
// keys or of values, in every layer, of as many drafts as there are threads for.  What is moved is read before any of it is
// written; a later round reads only rows from its own drafts on (path[b][k] >= k), and writes none before.  32 paths of up to
// 9, 48 layers, us: 10.2 with a layer a workgroup of 256 threads, most of which had nothing to move.
template <int D, int T>
__global__ __launch_bounds__(T) void kv4_keep_kernel(Layers layers, int n_layers, kv4::Cache c, const int32_t* __restrict__ dpos,
                                                     const int32_t* __restrict__ path, int A) {
    constexpr int Q = D / 32, kItems = 2 * Q + 2, R = T / kItems, U = kAtOnce;
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    const int b = blockIdx.x / c.Hkv, g = blockIdx.x - b * c.Hkv, lane = threadIdx.x & 63;
    const int l0 = blockIdx.y * U, nl = min(U, n_layers - l0);
    const int32_t* const line = path + (int64_t)b * A;
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
    const bool codes = item >= 2 * Q;
    auto tensor = [&](int u) {                                    // (uniform loads, and a choice)
        uint8_t* const* const t = layers.t[l0 + u];
        return item < Q ? t[0] : item < 2 * Q ? t[2] : item == 2 * Q ? t[1] : t[3];
    };
    const uint32_t stride = codes ? D / 32 : D / 2, off = codes ? 0 : 16 * (item < Q ? item : item - Q);
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
        v4u w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            w[u] = 0;
            if (!moves || u >= nl) continue;
            const uint8_t* const p = tensor(u) + from * stride + off;
            if (!codes) w[u] = *reinterpret_cast<const v4u*>(p);
            else if constexpr (D == 128) w[u][0] = *reinterpret_cast<const uint32_t*>(p);
            else w[u][0] = *reinterpret_cast<const uint16_t*>(p);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // the rows are here, not on their way, when another wave writes
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!moves || u >= nl) continue;
            uint8_t* const p = tensor(u) + to * stride + off;
            if (!codes) *reinterpret_cast<v4u*>(p) = w[u];
            else if constexpr (D == 128) *reinterpret_cast<uint32_t*>(p) = w[u][0];
            else *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[u][0];
        }
    }
}
template <int D>
void launch_keep(const Layers& t, int n, const kv4::Cache& c, const int32_t* dpos, const int32_t* path, int B, int A, hipStream_t st) {
    const dim3 grid(B * c.Hkv, (n + kAtOnce - 1) / kAtOnce);
    const int items = 2 * (D / 32) + 2;      // threads a draft
    if (A * (int64_t)items <= 64) hipLaunchKernelGGL((kv4_keep_kernel<D, 64>), grid, dim3(64), 0, st, t, n, c, dpos, path, A);
    else if (A * (int64_t)items <= 128) hipLaunchKernelGGL((kv4_keep_kernel<D, 128>), grid, dim3(128), 0, st, t, n, c, dpos, path, A);
    else hipLaunchKernelGGL((kv4_keep_kernel<D, 256>), grid, dim3(256), 0, st, t, n, c, dpos, path, A);
}

}  // namespace

extern "C" int mxfp4_tree_masks(const int32_t* parents, int32_t* tree, int32_t* depth, int B, int M, void* stream) {
    MXH_REQUIRE(parents && tree && depth, "tree_masks: null pointer");
    MXH_REQUIRE(B > 0 && B <= 65535 && M > 0 && M <= kMostDrafts, "tree_masks: B=%d M=%d (up to %d drafts)", B, M, kMostDrafts);
    const int chunks = (M + 63) / 64;
    const size_t lds = (size_t)(chunks * 64) * (sizeof(uint64_t) + sizeof(int));
    const bool wide = (M + 31) / 32 % 2 == 0 && ((uintptr_t)tree & 7) == 0;
    hipLaunchKernelGGL(wide ? tree_masks_kernel<true> : tree_masks_kernel<false>, dim3(B, chunks), dim3(kThreads), lds,
                       mxh::as_stream(stream), parents, reinterpret_cast<uint32_t*>(tree), depth, M);
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
        if (D == 64) launch_keep<64>(t, n, c, dpos, path, B, A, mxh::as_stream(stream));
        else launch_keep<128>(t, n, c, dpos, path, B, A, mxh::as_stream(stream));
        const int rc = mxh::launch_status("kv4_keep");
        if (rc != MXFP4_OK) return rc;
    }
    return MXFP4_OK;
}
