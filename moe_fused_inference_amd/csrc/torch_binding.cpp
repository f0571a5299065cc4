// Compiled torch/pybind binding of the C ABI (include/mxfp4_hip.h).
//
// The module has two submodules with the surfaces of the reference's two
// compiled extensions:
//   linear  -- mxfp4_linear_ext  (src/ext/mxfp4_binding.cpp:21-50): forward
//   decode  -- mxfp4_decode_ext  (src/ext/mxfp4_decode_binding.cpp:44-243):
//              prequant, lin_pq, moe_gateup, moe_down, moe_combine,
//              moe_gateup_tab, moe_down_tab, attn_decode, kv_write
// and a third of this library's own:
//   kv4     -- the MXFP4 KV cache: write, read, attn, attn_mx, write_slots, tree_masks, keep, tables (kv4.py)
// Names, argument order and meaning, output shapes and dtypes, and the
// argument-check messages are the reference's.  Each op is a thin shim:
// checks, torch allocations on the input's device (caching allocator), then
// one or two C-ABI calls on torch's current HIP stream.  Host pointer
// tables go to the kernels as launch arguments (no device table, no
// blocking copy, where the reference builds an int64 device table per
// call).  Compiled by the host compiler (no device code here) and linked
// against libmxfp4_hip.so.
#include <torch/extension.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <vector>

#include "mxfp4_hip.h"

namespace {

void require(bool cond, const char* msg) {
    if (!cond) throw std::runtime_error(msg);
}

// A non-zero C-ABI status becomes a RuntimeError with the library's message.
void check(int status, const char* what) {
    if (status != 0) {
        throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(status) +
                                 "): " + mxfp4_last_error());
    }
}

void* stream_of(const torch::Tensor& t) {
    return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

const uint8_t* u8(const torch::Tensor& t) { return static_cast<const uint8_t*>(t.data_ptr()); }
uint8_t* u8m(const torch::Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }
float* f32(const torch::Tensor& t) { return static_cast<float*>(t.data_ptr()); }

// Host pointer table of cuda uint8 tensors (the checks of
// src/ext/mxfp4_decode_binding.cpp:44-60), read straight from the Python
// list (or tuple): no std::vector<Tensor> of reference-counted copies, and the
// pointer array is a per-thread buffer reused from call to call (slot 0 = the
// packed data table, 1 = the scale table).  cols0 = size(1) of the first entry.
struct PtrTable {
    const uint8_t* const* p;
    int64_t cols0;
};

PtrTable ptr_table(const py::handle& seq, int slot, int64_t expect, const char* count_msg) {
    PyObject* fast = PySequence_Fast(seq.ptr(), "pointer table must be a list of tensors");
    if (fast == nullptr) throw py::error_already_set();
    const py::object keep = py::reinterpret_steal<py::object>(fast);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    require((int64_t)n == expect, count_msg);
    require(n > 0, "empty pointer table");
    thread_local std::vector<const uint8_t*> buf[2];
    std::vector<const uint8_t*>& p = buf[slot];
    p.resize((size_t)n);
    PyObject** items = PySequence_Fast_ITEMS(fast);
    int64_t cols0 = 0;
    for (Py_ssize_t i = 0; i < n; ++i) {
        require(THPVariable_Check(items[i]), "ptr table entries must be cuda uint8");
        const at::Tensor& t = THPVariable_Unpack(items[i]);
        require(t.is_cuda() && t.scalar_type() == torch::kUInt8, "ptr table entries must be cuda uint8");
        if (i == 0) cols0 = t.dim() >= 2 ? t.size(1) : 0;
        p[(size_t)i] = static_cast<const uint8_t*>(t.data_ptr());
    }
    return {p.data(), cols0};
}

int dtype_code(c10::ScalarType s) {
    return s == torch::kBFloat16 ? 0 : s == torch::kHalf ? 1 : 2;
}

// ---- mxfp4_linear_ext -------------------------------------------------------

// x (M,K) half|bf16, wp (N,Kp/2) u8, wsc (N,Kp/32) u8 -> f32 (M,N); activations
// are rounded to fp16 and MXFP4-quantized per 32-block (mxfp4_binding.cpp:21-45).
torch::Tensor forward(torch::Tensor x, torch::Tensor wp, torch::Tensor wsc) {
    require(x.is_cuda(), "x must be cuda");
    require(wp.is_cuda() && wsc.is_cuda(), "weights must be cuda");
    require(wp.scalar_type() == torch::kUInt8 && wsc.scalar_type() == torch::kUInt8,
            "weight tensors must be uint8");
    torch::Tensor xh = (x.scalar_type() == torch::kHalf || x.scalar_type() == torch::kBFloat16)
                           ? x : x.to(torch::kHalf);
    xh = xh.contiguous();
    wp = wp.contiguous();
    wsc = wsc.contiguous();
    const int M = (int)x.size(0), K = (int)x.size(1);
    const int N = (int)wp.size(0), Kp = (int)wp.size(1) * 2;
    auto y = torch::empty({M, N}, x.options().dtype(torch::kFloat32));
    if (M == 0 || N == 0) return y;
    const size_t wsb = mxfp4_linear_workspace_size(M, Kp);
    auto ws = torch::empty({(int64_t)wsb + 256}, x.options().dtype(torch::kUInt8));
    void* aligned = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(ws.data_ptr()) + 255) & ~uintptr_t(255));
    check(mxfp4_linear_forward(xh.data_ptr(), dtype_code(xh.scalar_type()), u8(wp), u8(wsc), f32(y),
                               M, N, K, Kp, aligned, wsb, stream_of(x)), "forward");
    return y;
}

// ---- mxfp4_decode_ext -------------------------------------------------------

// x (M,K) bf16 -> [xq (M,Kp/2) u8, xsc (M,Kp/32) u8], Kp = ceil32(K).
std::vector<torch::Tensor> prequant(torch::Tensor x) {
    require(x.is_cuda(), "x must be cuda");
    require(x.scalar_type() == torch::kBFloat16, "x must be bfloat16");
    x = x.contiguous();
    const int M = (int)x.size(0), K = (int)x.size(1);
    const int Kp = (K + 31) / 32 * 32;
    auto opts = x.options().dtype(torch::kUInt8);
    auto xq = torch::empty({M, Kp / 2}, opts);
    auto xsc = torch::empty({M, Kp / 32}, opts);
    if (M && Kp) {
        check(mxfp4_prequant(x.data_ptr(), K, M, K, Kp, u8m(xq), u8m(xsc), stream_of(x)), "prequant");
    }
    return {xq, xsc};
}

// Pre-quantized static linear -> f32 (M,N); Kp = 2*wp.size(1).
torch::Tensor lin_pq(torch::Tensor xq, torch::Tensor xsc, torch::Tensor wp, torch::Tensor wsc,
                     int64_t M_, int64_t N_, int64_t K_) {
    xq = xq.contiguous(); xsc = xsc.contiguous();
    wp = wp.contiguous(); wsc = wsc.contiguous();
    const int M = (int)M_, N = (int)N_, K = (int)K_;
    const int Kp = (int)wp.size(1) * 2;
    auto y = torch::empty({M, N}, xq.options().dtype(torch::kFloat32));
    check(mxfp4_lin_pq(u8(xq), u8(xsc), u8(wp), u8(wsc), f32(y), M, N, K, Kp, stream_of(xq)), "lin_pq");
    return y;
}

// Grouped gate+up over a token-major table of 2E*M weights -> f32 (M*E, 2N).
torch::Tensor moe_gateup(torch::Tensor xq, torch::Tensor xsc, const py::object& wps, const py::object& wscs,
                         int64_t E_, int64_t M_, int64_t N_, int64_t K_) {
    const int E = (int)E_, M = (int)M_, N = (int)N_, K = (int)K_;
    require((int64_t)py::len(wps) == 2 * E_ * M_, "wps must be 2E*M");
    require((int64_t)py::len(wscs) == 2 * E_ * M_, "wscs must be 2E*M");
    const PtrTable tw = ptr_table(wps, 0, 2 * E_ * M_, "wps must be 2E*M");
    const PtrTable ts = ptr_table(wscs, 1, 2 * E_ * M_, "wscs must be 2E*M");
    const int Kp = (int)tw.cols0 * 2;
    auto gu = torch::empty({(int64_t)M * E, 2 * N}, xq.options().dtype(torch::kFloat32));
    check(mxfp4_moe_gateup(u8(xq), u8(xsc), tw.p, ts.p, f32(gu), E, M, N, K, Kp, stream_of(xq)), "moe_gateup");
    return gu;
}

// Fused silu(gate)*up -> MXFP4 -> down over E*M weights -> f32 (M*E, N).
torch::Tensor moe_down(torch::Tensor gu, const py::object& wps, const py::object& wscs, int64_t E_, int64_t M_,
                       int64_t N_, int64_t K_) {
    const int E = (int)E_, M = (int)M_, N = (int)N_, K = (int)K_;
    require((int64_t)py::len(wps) == E_ * M_, "wps must be E*M");
    require(gu.size(0) == (int64_t)M * E && gu.size(1) == 2 * (int64_t)K, "gu (M*E,2K)");
    const PtrTable tw = ptr_table(wps, 0, E_ * M_, "wps must be E*M");
    const PtrTable ts = ptr_table(wscs, 1, E_ * M_, "wscs must be E*M");
    const int Kp = (int)tw.cols0 * 2;
    gu = gu.contiguous();
    auto yd = torch::empty({(int64_t)M * E, N}, gu.options());
    check(mxfp4_moe_down(f32(gu), tw.p, ts.p, f32(yd), E, M, N, K, Kp, stream_of(gu)), "moe_down");
    return yd;
}

// out[m,c] = sum_{e<min(E,8)} w[m,e]*yd[m*E+e,c] -> f32 (M,N); E = w.numel()/M.
torch::Tensor moe_combine(torch::Tensor yd, torch::Tensor w, int64_t M_) {
    yd = yd.contiguous(); w = w.contiguous();
    const int M = (int)M_;
    require(M > 0, "w (M,E)");
    const int E = (int)(w.numel() / M);
    const int N = (int)yd.size(1);
    require((int64_t)M * E == w.numel(), "w (M,E)");
    require(yd.size(0) == (int64_t)M * E, "yd (M*E,N)");
    auto out = torch::empty({M, N}, yd.options());
    check(mxfp4_moe_combine(f32(yd), N, f32(w), E, f32(out), M, N, stream_of(yd)), "moe_combine");
    return out;
}

// moe_gateup with device int64 pointer tables; Kp = 2*xq.size(1).
torch::Tensor moe_gateup_tab(torch::Tensor xq, torch::Tensor xsc, torch::Tensor wps_tab,
                             torch::Tensor wscs_tab, int64_t E_, int64_t M_, int64_t N_, int64_t K_) {
    const int E = (int)E_, M = (int)M_, N = (int)N_, K = (int)K_;
    const int Kp = (int)xq.size(1) * 2;
    auto gu = torch::empty({(int64_t)M * E, 2 * N}, xq.options().dtype(torch::kFloat32));
    check(mxfp4_moe_gateup_devtab(u8(xq), u8(xsc), static_cast<const int64_t*>(wps_tab.data_ptr()),
                                  static_cast<const int64_t*>(wscs_tab.data_ptr()), f32(gu), E, M, N, K,
                                  Kp, stream_of(xq)),
          "moe_gateup_tab");
    return gu;
}

// moe_down with device int64 pointer tables; Kp = ceil32(gu.size(1)/2).
torch::Tensor moe_down_tab(torch::Tensor gu, torch::Tensor wps_tab, torch::Tensor wscs_tab, int64_t E_,
                           int64_t M_, int64_t N_, int64_t K_) {
    const int E = (int)E_, M = (int)M_, N = (int)N_, K = (int)K_;
    const int Kp = (int)((gu.size(1) / 2 + 31) / 32 * 32);
    auto yd = torch::empty({(int64_t)M * E, N}, gu.options());
    check(mxfp4_moe_down_devtab(f32(gu), static_cast<const int64_t*>(wps_tab.data_ptr()),
                                static_cast<const int64_t*>(wscs_tab.data_ptr()), f32(yd), E, M, N, K, Kp,
                                stream_of(gu)),
          "moe_down_tab");
    return yd;
}

void check_kv(const torch::Tensor& kvk, const torch::Tensor& kvv, const torch::Tensor& dpos) {
    require(kvk.scalar_type() == torch::kUInt8 && kvv.scalar_type() == torch::kUInt8 && kvk.dim() == 3 &&
                kvv.sizes() == kvk.sizes(),
            "kvk/kvv must be uint8 (max_pos,Hkv,D) tensors of one shape");
    require(kvk.is_contiguous() && kvv.is_contiguous(), "kvk/kvv must be contiguous");
    require(dpos.scalar_type() == torch::kInt32 && dpos.is_cuda(), "dpos must be a cuda int32 tensor");
}

// Decode attention over one layer's E4M3 KV cache -> f32 (M,Hq,D).  q (M,Hq,D)
// bf16 (roped); dpos (1,) int32 on the device, token m attends to 0..dpos+m;
// sc (M,Hq,max_pos) f32 receives the raw scores (mxfp4_decode_binding.cpp:213-230).
torch::Tensor attn_decode(torch::Tensor q, torch::Tensor kvk, torch::Tensor kvv, torch::Tensor dpos,
                          torch::Tensor sc, int64_t M_) {
    require(q.dim() == 3 && q.scalar_type() == torch::kBFloat16 && q.is_cuda(),
            "q must be a cuda bf16 (M,Hq,D) tensor");
    q = q.contiguous();
    const int M = (int)M_;
    check_kv(kvk, kvv, dpos);
    const int Hq = (int)q.size(1), D = (int)q.size(2);
    const int max_pos = (int)kvk.size(0), Hkv = (int)kvk.size(1);
    require(q.size(0) >= M, "q has fewer than M rows");
    require(sc.scalar_type() == torch::kFloat32 && sc.is_contiguous() && sc.numel() >= (int64_t)M * Hq * max_pos,
            "sc must be a contiguous f32 buffer of M*Hq*max_pos elements");
    auto o = torch::empty({M, Hq, D}, q.options().dtype(torch::kFloat32));
    const size_t wsb = mxfp4_attn_decode_workspace_size(M, Hq, max_pos);
    auto ws = torch::empty({(int64_t)wsb}, q.options().dtype(torch::kUInt8));
    check(mxfp4_attn_decode(q.data_ptr(), u8(kvk), u8(kvv), static_cast<const int*>(dpos.data_ptr()), f32(sc),
                            f32(o), M, Hq, Hkv, D, max_pos, ws.data_ptr(), wsb, stream_of(q)),
          "attn_decode");
    return o;
}

// k/v (M,Hkv,D) bf16 -> E4M3 bytes at rows dpos+m of kvk/kvv (max_pos,Hkv,D)
// u8, in place (mxfp4_decode_binding.cpp:161-173).
void kv_write(torch::Tensor k, torch::Tensor v, torch::Tensor kvk, torch::Tensor kvv, torch::Tensor dpos,
              int64_t M_) {
    require(k.scalar_type() == torch::kBFloat16 && v.scalar_type() == torch::kBFloat16 && k.is_cuda() &&
                v.is_cuda(),
            "k/v must be cuda bf16");
    k = k.contiguous(); v = v.contiguous();
    const int M = (int)M_;
    check_kv(kvk, kvv, dpos);
    const int max_pos = (int)kvk.size(0), Hkv = (int)kvk.size(1), D = (int)kvk.size(2);
    require(k.numel() >= (int64_t)M * Hkv * D && v.numel() >= (int64_t)M * Hkv * D,
            "k/v have fewer than M*Hkv*D elements");
    check(mxfp4_kv_write(k.data_ptr(), v.data_ptr(), u8m(kvk), u8m(kvv), static_cast<const int*>(dpos.data_ptr()),
                         M, Hkv, D, max_pos, stream_of(k)),
          "kv_write");
}

// ---- the MXFP4 KV cache (kv4.py) -----------------------------------------------

// The cache tensors and where the batch's sequences lie in them, checked:
// kq, vq u8 (n_pages, Hkv, page, D/2), ks, vs u8 (n_pages, Hkv, page, D/32),
// pages int32 (B, max_pages) or none, at (dpos or start) int32 (B) or none.
struct Kv4 {
    uint8_t *kq, *ks, *vq, *vs;
    const int32_t* pages;
    const int32_t* at;
    int n_pages, page, max_pages, B, Hkv, D;
};

// torch::empty on t's device, without the dispatcher: about half its time, which a small call's two or three show.
torch::Tensor empty_on(const torch::Tensor& t, at::IntArrayRef sizes, c10::ScalarType dt) {
    return at::detail::empty_cuda(sizes, dt, t.device(), c10::nullopt);
}

int as_int(int64_t v, const char* msg) {
    require(v >= 0 && v <= 0x7FFFFFFF, msg);
    return (int)v;
}

Kv4 kv4_cache(const torch::Tensor& kq, const torch::Tensor& ks, const torch::Tensor& vq, const torch::Tensor& vs,
              const c10::optional<torch::Tensor>& pages, const c10::optional<torch::Tensor>& at, const char* at_msg) {
    require(kq.scalar_type() == torch::kUInt8 && ks.scalar_type() == torch::kUInt8 && vq.scalar_type() == torch::kUInt8 &&
                vs.scalar_type() == torch::kUInt8,
            "cache tensors must be uint8");
    require(kq.dim() == 4 && ks.dim() == 4 && vq.sizes() == kq.sizes() && vs.sizes() == ks.sizes() &&
                ks.size(0) == kq.size(0) && ks.size(1) == kq.size(1) && ks.size(2) == kq.size(2) &&
                ks.size(3) * 16 == kq.size(3),
            "kq/vq must be (n_pages,Hkv,page,D/2), ks/vs (n_pages,Hkv,page,D/32)");
    require(kq.is_contiguous() && ks.is_contiguous() && vq.is_contiguous() && vs.is_contiguous(),
            "cache tensors must be contiguous");
    const auto dev = kq.device();
    require(ks.device() == dev && vq.device() == dev && vs.device() == dev, "cache tensors must be on one device");
    Kv4 c{u8m(kq), u8m(ks), u8m(vq), u8m(vs), nullptr, nullptr, 0, 0, 0, 0, 0, 0};
    c.n_pages = as_int(kq.size(0), "too many pages");
    c.Hkv = as_int(kq.size(1), "too many heads");
    require(c.Hkv > 0, "a cache needs a kv head at least");     // (query heads are divided by it)
    c.page = as_int(kq.size(2), "page too long");
    c.D = as_int(kq.size(3) * 2, "head_dim too large");
    c.B = c.n_pages;
    if (pages.has_value()) {
        require(pages->scalar_type() == torch::kInt32 && pages->dim() == 2 && pages->is_contiguous() && pages->device() == dev,
                "pages must be a contiguous int32 (B,max_pages) tensor on the cache's device");
        c.pages = static_cast<const int32_t*>(pages->data_ptr());
        c.B = as_int(pages->size(0), "too many sequences");
        c.max_pages = as_int(pages->size(1), "too many pages");
        // a table of no columns has no address, which would stand for no table
        require(c.max_pages > 0 || c.B == 0, "pages must have a column at least");
    }
    if (at.has_value()) {
        require(at->scalar_type() == torch::kInt32 && at->is_contiguous() && at->device() == dev && at->numel() == c.B, at_msg);
        c.at = static_cast<const int32_t*>(at->data_ptr());
    }
    require(kq.is_cuda(), "cache tensors must be cuda");
    return c;
}

// (B,M,H,D) of the cache's device whose tokens lie at one stride, H*D contiguous: itself, or a copy.
torch::Tensor token_rows(const torch::Tensor& t) {
    const bool ok = t.stride(3) == 1 && t.stride(2) == t.size(3) && t.stride(1) >= t.size(2) * t.size(3) &&
                    (t.size(0) == 1 || t.stride(0) == t.size(1) * t.stride(1));
    return ok ? t : t.contiguous();
}
int64_t token_stride(const torch::Tensor& t) {
    return t.size(1) > 1 ? t.stride(1) : t.size(0) > 1 ? t.stride(0) : t.size(2) * t.size(3);
}
bool is_float16s(const torch::Tensor& t) { return t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kHalf; }

void kv4_write(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& kq, const torch::Tensor& ks,
               const torch::Tensor& vq, const torch::Tensor& vs, const torch::Tensor& dpos,
               const c10::optional<torch::Tensor>& pages) {
    const Kv4 c = kv4_cache(kq, ks, vq, vs, pages, dpos, "dpos must be a contiguous int32 (B,) tensor on the cache's device");
    require(k.device() == kq.device() && v.device() == kq.device(), "k/v must be on the cache's device");
    require((is_float16s(k) || k.scalar_type() == torch::kFloat32) && v.scalar_type() == k.scalar_type(),
            "k/v must be bfloat16, float16 or float32, both of one type");
    require(k.dim() == 4 && v.sizes() == k.sizes() && k.size(0) == c.B && k.size(2) == c.Hkv && k.size(3) == c.D,
            "k/v must be (B,M,Hkv,D)");
    const int M = as_int(k.size(1), "too many tokens");
    if (M == 0 || c.B == 0) return;
    const c10::DeviceGuard guard(kq.device());
    const torch::Tensor kc = token_rows(k), vc = token_rows(v);
    check(mxfp4_kv4_write(kc.data_ptr(), vc.data_ptr(), dtype_code(kc.scalar_type()), token_stride(kc), token_stride(vc), c.kq,
                          c.ks, c.vq, c.vs, c.pages, c.n_pages, c.page, c.max_pages, c.at, c.B, M, c.Hkv, c.D, stream_of(kq)),
          "kv4_write");
}

std::vector<torch::Tensor> kv4_read(const torch::Tensor& kq, const torch::Tensor& ks, const torch::Tensor& vq,
                                    const torch::Tensor& vs, int64_t n_, const c10::optional<torch::Tensor>& start,
                                    const c10::optional<torch::Tensor>& pages, const py::object& dtype) {
    const Kv4 c = kv4_cache(kq, ks, vq, vs, pages, start, "start must be a contiguous int32 (B,) tensor on the cache's device");
    const auto dt = torch::python::detail::py_object_to_dtype(dtype);
    require(dt == torch::kBFloat16 || dt == torch::kHalf || dt == torch::kFloat32, "dtype must be bfloat16, float16 or float32");
    const int n = as_int(n_, "n must not be negative");
    const c10::DeviceGuard guard(kq.device());
    auto k = empty_on(kq, {c.B, n, c.Hkv, c.D}, dt), v = empty_on(kq, {c.B, n, c.Hkv, c.D}, dt);
    if (n != 0 && c.B != 0) {
        check(mxfp4_kv4_read(c.kq, c.ks, c.vq, c.vs, c.pages, c.n_pages, c.page, c.max_pages, c.at, k.data_ptr(), v.data_ptr(),
                             dtype_code(dt), c.B, n, c.Hkv, c.D, stream_of(kq)),
              "kv4_read");
    }
    return {k, v};
}

// What its tokens see of the cache: a window (0: all) with sinks, and the words of a tree or null.
struct Masks {
    int window, sinks;
    const int32_t* tree;
};
Masks kv4_masks(const torch::Tensor& q, const c10::optional<int64_t>& window, int64_t sinks, const c10::optional<torch::Tensor>& tree) {
    Masks m{0, 0, nullptr};
    if (window.has_value()) {
        require(*window > 0, "window must be positive");
        m.window = (int)std::min<int64_t>(*window, 0x7FFFFFFF);
    }
    require(sinks >= 0, "sinks must not be negative");
    require(sinks == 0 || window.has_value(), "sinks need a window");
    m.sinks = (int)std::min<int64_t>(sinks, 0x7FFFFFFF);
    if (tree.has_value()) {
        require(tree->scalar_type() == torch::kInt32 && tree->dim() == 3 && tree->is_contiguous() && tree->device() == q.device() &&
                    tree->size(0) == q.size(0) && tree->size(1) == q.size(1) && tree->size(2) == (q.size(1) + 31) / 32,
                "tree must be a contiguous int32 (B,M,ceil(M/32)) tensor on the cache's device");
        m.tree = static_cast<const int32_t*>(tree->data_ptr());
        require(m.window == 0 || m.window >= q.size(1), "a tree needs a window of M at least");
    }
    return m;
}

// The attention of q (B,M,Hq,D) over the cache into o and / or oq, os (undefined: not wanted).
void kv4_attn_into(const torch::Tensor& q, const Kv4& c, const Masks& mk, const torch::Tensor& kq, const torch::Tensor& o,
                   const torch::Tensor& oq, const torch::Tensor& os) {
    const int M = (int)q.size(1), Hq = (int)q.size(2);
    const torch::Tensor qc0 = token_rows(q);
    const bool aligned = (reinterpret_cast<uintptr_t>(qc0.data_ptr()) & 15) == 0 && token_stride(qc0) % 8 == 0;
    const torch::Tensor qc = aligned ? qc0 : qc0.clone(at::MemoryFormat::Contiguous);
    const int64_t max_pos = c.pages ? (int64_t)c.max_pages * c.page : c.page;
    require(max_pos <= (1ll << 30), "attn_decode4: more than 2^30 positions a sequence");
    const size_t wsb = mxfp4_attn_kv4_masked_workspace_size(c.B, M, Hq, c.Hkv, c.D, (int)max_pos, mk.window, mk.sinks);
    torch::Tensor ws;
    if (wsb) ws = empty_on(kq, {(int64_t)wsb}, torch::kUInt8);
    check(mxfp4_attn_kv4_masked(qc.data_ptr(), dtype_code(qc.scalar_type()), token_stride(qc), c.kq, c.ks, c.vq, c.vs, c.pages,
                                c.n_pages, c.page, c.max_pages, c.at, mk.window, mk.sinks, mk.tree,
                                o.defined() ? o.data_ptr() : nullptr, o.defined() ? dtype_code(o.scalar_type()) : 2,
                                oq.defined() ? u8m(oq) : nullptr, os.defined() ? u8m(os) : nullptr, c.B, M, Hq, c.Hkv, c.D,
                                wsb ? ws.data_ptr() : nullptr, wsb, stream_of(kq)),
          "attn_decode4");
}

Kv4 kv4_attn_args(const torch::Tensor& q, const torch::Tensor& kq, const torch::Tensor& ks, const torch::Tensor& vq,
                  const torch::Tensor& vs, const torch::Tensor& dpos, const c10::optional<torch::Tensor>& pages) {
    const Kv4 c = kv4_cache(kq, ks, vq, vs, pages, dpos, "dpos must be a contiguous int32 (B,) tensor on the cache's device");
    require(q.device() == kq.device() && is_float16s(q), "q must be bfloat16 or float16 on the cache's device");
    require(q.dim() == 4 && q.size(0) == c.B && q.size(3) == c.D && q.size(2) > 0 && q.size(2) % c.Hkv == 0,
            "q must be (B,M,Hq,D), Hq a multiple of Hkv");
    as_int(q.size(1), "too many tokens");
    as_int(q.size(2), "too many heads");
    return c;
}

torch::Tensor kv4_attn(const torch::Tensor& q, const torch::Tensor& kq, const torch::Tensor& ks, const torch::Tensor& vq,
                       const torch::Tensor& vs, const torch::Tensor& dpos, const c10::optional<torch::Tensor>& pages,
                       const py::object& dtype, const c10::optional<int64_t>& window, int64_t sinks,
                       const c10::optional<torch::Tensor>& tree) {
    const Kv4 c = kv4_attn_args(q, kq, ks, vq, vs, dpos, pages);
    const Masks mk = kv4_masks(q, window, sinks, tree);
    const auto dt = torch::python::detail::py_object_to_dtype(dtype);
    require(dt == torch::kBFloat16 || dt == torch::kHalf || dt == torch::kFloat32, "dtype must be bfloat16, float16 or float32");
    const c10::DeviceGuard guard(kq.device());
    auto o = empty_on(q, q.sizes(), dt);
    if (o.numel() != 0) kv4_attn_into(q, c, mk, kq, o, torch::Tensor(), torch::Tensor());
    return o;
}

std::vector<torch::Tensor> kv4_attn_mx(const torch::Tensor& q, const torch::Tensor& kq, const torch::Tensor& ks,
                                       const torch::Tensor& vq, const torch::Tensor& vs, const torch::Tensor& dpos,
                                       const c10::optional<torch::Tensor>& pages, const c10::optional<int64_t>& window,
                                       int64_t sinks, const c10::optional<torch::Tensor>& tree) {
    const Kv4 c = kv4_attn_args(q, kq, ks, vq, vs, dpos, pages);
    const Masks mk = kv4_masks(q, window, sinks, tree);
    const c10::DeviceGuard guard(kq.device());
    const int64_t T = q.size(0) * q.size(1), row = q.size(2) * q.size(3);
    auto oq = empty_on(kq, {T, row / 2}, torch::kUInt8), os = empty_on(kq, {T, row / 32}, torch::kUInt8);
    if (T != 0) kv4_attn_into(q, c, mk, kq, torch::Tensor(), oq, os);
    return {oq, os};
}

// k, v (T,Hkv,D) -> the pool's rows at slots (T) int64.
void kv4_write_slots(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& kq, const torch::Tensor& ks,
                     const torch::Tensor& vq, const torch::Tensor& vs, const torch::Tensor& slots) {
    const Kv4 c = kv4_cache(kq, ks, vq, vs, c10::nullopt, c10::nullopt, "");
    require(k.device() == kq.device() && v.device() == kq.device(), "k/v must be on the cache's device");
    require((is_float16s(k) || k.scalar_type() == torch::kFloat32) && v.scalar_type() == k.scalar_type(),
            "k/v must be bfloat16, float16 or float32, both of one type");
    require(k.dim() == 3 && v.sizes() == k.sizes() && k.size(1) == c.Hkv && k.size(2) == c.D, "k/v must be (T,Hkv,D)");
    require(slots.scalar_type() == torch::kInt64 && slots.is_contiguous() && slots.device() == kq.device() && slots.dim() == 1 &&
                slots.numel() == k.size(0),
            "slots must be a contiguous int64 (T,) tensor on the cache's device");
    const int T = as_int(k.size(0), "too many tokens");
    if (T == 0) return;
    const c10::DeviceGuard guard(kq.device());
    const torch::Tensor kc = token_rows(k.unsqueeze(0)), vc = token_rows(v.unsqueeze(0));
    check(mxfp4_kv4_write_slots(kc.data_ptr(), vc.data_ptr(), dtype_code(kc.scalar_type()), token_stride(kc), token_stride(vc), c.kq,
                                c.ks, c.vq, c.vs, c.n_pages, c.page, static_cast<const int64_t*>(slots.data_ptr()), T, c.Hkv, c.D,
                                stream_of(kq)),
          "kv4_write_slots");
}

bool is_i32(const torch::Tensor& t, int64_t dim) { return t.scalar_type() == torch::kInt32 && t.dim() == dim && t.is_contiguous(); }
int32_t* i32m(const torch::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

// parents (B,M) -> [tree (B,M,ceil(M/32)), depth (B,M)].
std::vector<torch::Tensor> kv4_tree_masks(const torch::Tensor& parents) {
    require(is_i32(parents, 2), "parents must be a contiguous int32 (B,M) tensor");
    require(parents.is_cuda(), "parents must be cuda");
    const int B = as_int(parents.size(0), "too many sequences"), M = as_int(parents.size(1), "too many drafts");
    const c10::DeviceGuard guard(parents.device());
    auto tree = empty_on(parents, {B, M, (M + 31) / 32}, torch::kInt32), depth = empty_on(parents, {B, M}, torch::kInt32);
    if (B != 0 && M != 0) check(mxfp4_tree_masks(i32m(parents), i32m(tree), i32m(depth), B, M, stream_of(parents)), "tree_masks");
    return {tree, depth};
}

// The rows dpos[b] + path[b,k] of every layer's cache -> dpos[b] + k.  caches: a sequence of (kq, ks, vq, vs), read as it
// is (48 layers: 192 tensors; as vectors of tensors they took 9 us of the call's 17).
void kv4_keep(const py::handle& caches, const torch::Tensor& dpos, const torch::Tensor& path, const c10::optional<torch::Tensor>& pages) {
    const auto fast = [](PyObject* o, const char* msg) {
        PyObject* const f = PySequence_Fast(o, msg);
        if (!f) throw py::error_already_set();
        return py::reinterpret_steal<py::object>(f);
    };
    const py::object list = fast(caches.ptr(), "caches must be a sequence");
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list.ptr());
    require(n > 0, "kv4_keep needs a cache at least");
    std::vector<uint8_t*> p[4];
    for (auto& x : p) x.reserve(n);
    Kv4 c{};
    torch::Tensor first[4];
    for (Py_ssize_t l = 0; l < n; ++l) {
        const py::object cache = fast(PySequence_Fast_GET_ITEM(list.ptr(), l), "a cache is four tensors");
        require(PySequence_Fast_GET_SIZE(cache.ptr()) == 4, "a cache is four tensors");
        const at::Tensor* t[4];
        for (int i = 0; i < 4; ++i) {
            PyObject* const o = PySequence_Fast_GET_ITEM(cache.ptr(), i);
            require(THPVariable_Check(o), "a cache is four tensors");
            t[i] = &THPVariable_Unpack(o);
        }
        if (l == 0) {
            c = kv4_cache(*t[0], *t[1], *t[2], *t[3], pages, dpos, "dpos must be a contiguous int32 (B,) tensor on the cache's device");
            for (int i = 0; i < 4; ++i) first[i] = *t[i];
        } else {
            for (int i = 0; i < 4; ++i)
                require(t[i]->scalar_type() == torch::kUInt8 && t[i]->sizes() == first[i].sizes() && t[i]->is_contiguous() &&
                            t[i]->device() == first[0].device(),
                        "caches must be contiguous, of one shape and device");
        }
        for (int i = 0; i < 4; ++i) p[i].push_back(u8m(*t[i]));
    }
    const torch::Tensor& kq = first[0];
    require(is_i32(path, 2) && path.device() == kq.device() && path.size(0) == c.B,
            "path must be a contiguous int32 (B,A) tensor on the cache's device");
    const int A = as_int(path.size(1), "too many drafts");
    if (A == 0 || c.B == 0) return;
    const c10::DeviceGuard guard(kq.device());
    check(mxfp4_kv4_keep(p[0].data(), p[1].data(), p[2].data(), p[3].data(), as_int((int64_t)n, "too many caches"), c.pages,
                         c.n_pages, c.page, c.max_pages, c.at, i32m(path), c.B, A, c.Hkv, c.D, stream_of(kq)),
          "kv4_keep");
}

// The table of a batch follows its lengths, in place; with `news` -> [slots, seq, pos (T), starts (B+1)].
std::vector<torch::Tensor> kv4_tables(const torch::Tensor& pages, const torch::Tensor& span, const torch::Tensor& free,
                                      const torch::Tensor& state, int64_t page_, const c10::optional<int64_t>& window, int64_t sinks,
                                      const torch::Tensor& lens, const c10::optional<torch::Tensor>& news, int64_t T_) {
    const auto dev = pages.device();
    require(is_i32(pages, 2) && pages.size(1) > 0, "pages must be a contiguous int32 (B,max_pages) tensor");
    const int B = as_int(pages.size(0), "too many sequences"), max_pages = as_int(pages.size(1), "too many pages");
    require(is_i32(span, 2) && span.size(0) == B && span.size(1) == 2 && span.device() == dev, "span must be a contiguous int32 (B,2) tensor on the table's device");
    require(is_i32(free, 1) && free.device() == dev, "free must be a contiguous int32 (n_pages,) tensor on the table's device");
    require(is_i32(state, 1) && state.numel() == 2 && state.device() == dev, "state must be a contiguous int32 (2,) tensor on the table's device");
    require(is_i32(lens, 1) && lens.numel() == B && lens.device() == dev, "lens must be a contiguous int32 (B,) tensor on the table's device");
    if (news.has_value())
        require(is_i32(*news, 1) && news->numel() == B && news->device() == dev, "new must be a contiguous int32 (B,) tensor on the table's device");
    const int page = as_int(page_, "page too long"), T = as_int(T_, "T must not be negative");
    require(T == 0 || news.has_value(), "T tokens need new");
    if (window.has_value()) require(*window > 0, "window must be positive");
    require(sinks >= 0 && (sinks == 0 || window.has_value()), "sinks need a window");
    require(pages.is_cuda(), "tables must be cuda");
    const c10::DeviceGuard guard(dev);
    torch::Tensor slots, seq, pos, starts;
    if (news.has_value()) {
        slots = empty_on(pages, {T}, torch::kInt64);
        seq = empty_on(pages, {T}, torch::kInt32);
        pos = empty_on(pages, {T}, torch::kInt32);
        starts = empty_on(pages, {(int64_t)B + 1}, torch::kInt32);
    }
    if (B == 0) {
        if (news.has_value()) {
            for (const auto& t : {slots, seq, pos}) t.fill_(-1);
            starts.zero_();
            return {slots, seq, pos, starts};
        }
        return {};
    }
    const bool some = news.has_value();
    check(mxfp4_kv4_tables(i32m(pages), i32m(span), i32m(free), i32m(state), i32m(lens), some ? i32m(*news) : nullptr,
                           window.has_value() ? (int)std::min<int64_t>(*window, 0x7FFFFFFF) : 0, (int)std::min<int64_t>(sinks, 0x7FFFFFFF),
                           B, max_pages, as_int(free.numel(), "too many pages"), page, some ? i32m(starts) : nullptr,
                           T ? static_cast<int64_t*>(slots.data_ptr()) : nullptr, T ? i32m(seq) : nullptr, T ? i32m(pos) : nullptr, T,
                           stream_of(pages)),
          "kv4_tables");
    if (!some) return {};
    return {slots, seq, pos, starts};
}

}  // namespace

PYBIND11_MODULE(mxfp4_ext, m) {
    m.doc() = "Compiled torch binding of libmxfp4_hip (gfx950)";
    auto lin = m.def_submodule("linear", "mxfp4_linear_ext surface");
    lin.attr("__name__") = "mxfp4_linear_ext";
    lin.def("forward", &forward, "x (M,K) half|bf16 -> fp16 round -> MXFP4 -> f32 (M,N)");
    auto dec = m.def_submodule("decode", "mxfp4_decode_ext surface");
    dec.attr("__name__") = "mxfp4_decode_ext";
    dec.def("prequant", &prequant, "bf16 (M,K) -> [xq (M,Kp/2) u8, xsc (M,Kp/32) u8]");
    dec.def("lin_pq", &lin_pq, "prequantized static MXFP4 linear -> f32 (M,N)");
    dec.def("moe_gateup", &moe_gateup, "grouped gate+up (2E*M weights) -> f32 (M*E,2N)");
    dec.def("moe_down", &moe_down, "fused silu(gate)*up, MXFP4, down -> f32 (M*E,N)");
    dec.def("moe_combine", &moe_combine, "out[m,c] = sum_e w[m,e]*yd[m*E+e,c]");
    dec.def("moe_gateup_tab", &moe_gateup_tab, "grouped gate+up from device pointer tables");
    dec.def("moe_down_tab", &moe_down_tab, "fused silu-down from device pointer tables");
    dec.def("attn_decode", &attn_decode, "decode attention over an E4M3 KV cache -> f32 (M,Hq,D)");
    dec.def("kv_write", &kv_write, "E4M3 KV write of M tokens at rows dpos+m");
    auto k4 = m.def_submodule("kv4", "the MXFP4 KV cache");
    k4.def("write", &kv4_write, py::arg("k"), py::arg("v"), py::arg("kq"), py::arg("ks"), py::arg("vq"), py::arg("vs"),
           py::arg("dpos"), py::arg("pages"), "k, v (B,M,Hkv,D) -> MXFP4 rows at dpos[b]+m");
    k4.def("read", &kv4_read, py::arg("kq"), py::arg("ks"), py::arg("vq"), py::arg("vs"), py::arg("n"), py::arg("start"),
           py::arg("pages"), py::arg("dtype"), "positions start[b] .. start[b]+n-1 -> [k, v] (B,n,Hkv,D)");
    k4.def("attn", &kv4_attn, py::arg("q"), py::arg("kq"), py::arg("ks"), py::arg("vq"), py::arg("vs"), py::arg("dpos"),
           py::arg("pages"), py::arg("dtype"), py::arg("window"), py::arg("sinks"), py::arg("tree"),
           "attention over the MXFP4 cache -> (B,M,Hq,D)");
    k4.def("attn_mx", &kv4_attn_mx, py::arg("q"), py::arg("kq"), py::arg("ks"), py::arg("vq"), py::arg("vs"), py::arg("dpos"),
           py::arg("pages"), py::arg("window"), py::arg("sinks"), py::arg("tree"), "attn as the MXFP4 rows of its bf16 rounding -> [oq, os]");
    k4.def("write_slots", &kv4_write_slots, "k, v (T,Hkv,D) -> MXFP4 rows at slots");
    k4.def("tree_masks", &kv4_tree_masks, "parents (B,M) -> [tree, depth]");
    k4.def("keep", &kv4_keep, "the accepted drafts' rows move together");
    k4.def("tables", &kv4_tables, "a batch's page table follows its lengths -> [slots, seq, pos, starts], or nothing");
}
