"""GPU tests of the decode step over the MXFP4 KV cache (DecodeStep(kv="mxfp4")) and of its write,
qk_norm_rope_kv4.

The step is compared layer by layer as tests/test_gpu_decode_step.py does, with that test's tolerances: both
sides hold the same cache bytes but for a row's few values whose fp32 sums round to another bf16, and that next
to a step of E2M1 (under 1e-5 of them); attention itself is held to its derived bound in test_gpu_kv4.py.
"""
import numpy as np
import pytest
import torch

from moe_fused_inference_amd import _lib, kv4
from moe_fused_inference_amd.decode_step import DecodeStep
from oracle import step as sref
from tests.gpu_helpers import DEV, assert_close, np_
from tests.test_gpu_decode_step import CFG, CTX, MAX_POS, tiny  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,M,Hq,Hkv,page,dpos", [
    (1, 1, 32, 4, 0, [7]), (1, 5, 8, 2, 0, [43]), (3, 2, 6, 3, 32, [-1, 30, 95]), (2, 33, 4, 4, 16, [40, -40])])
def test_qk_norm_rope_kv4(B, M, Hq, Hkv, page, dpos):
    """q's bits are qk_norm_rope_kv's, and the cache's those of kv4_write on the rows that it makes of k (as if
    they were q heads) and on bf16(v)."""
    D, lib, n_pages, P = 128, _lib.load(), (B * 3 if page else B), page or 48
    g = torch.Generator(device=DEV)
    g.manual_seed(B * 10 + M)
    qkv = torch.randn((B * M, (Hq + 2 * Hkv) * D), generator=g, device=DEV) * 3
    qw, kw = (1 + 0.1 * torch.randn((2, D), generator=g, device=DEV)).bfloat16()
    dp = torch.tensor(dpos, dtype=torch.int32, device=DEV)
    pages = torch.randperm(n_pages, generator=g, device=DEV).int().view(B, 3) if page else None
    if page and B > 2:
        pages[0, 0] = -1
    got, want = (kv4.empty_cache(n_pages, P, Hkv, D) for _ in range(2))
    q = torch.empty((B * M, Hq, D), dtype=torch.bfloat16, device=DEV)
    _lib.check(lib.mxfp4_qk_norm_rope_kv4(qkv.data_ptr(), qw.data_ptr(), kw.data_ptr(), 1e-6, 1e6, *[t.data_ptr() for t in got],
                                          None if pages is None else pages.data_ptr(), n_pages, P, 3 if page else 0, dp.data_ptr(),
                                          B, M, Hq, Hkv, D, q.data_ptr(), torch.cuda.current_stream().cuda_stream), "kv4")
    dummy = torch.empty((2, 16, Hq, D), dtype=torch.uint8, device=DEV)

    def rope(x, w, b, Hkv_):
        """The heads x (M, H, D) of sequence b through qk_norm_rope_kv's q side."""
        H = x.shape[1]
        y = torch.cat([x.reshape(M, H * D), torch.zeros((M, 2 * Hkv_ * D), device=DEV)], 1).contiguous()
        out = torch.empty((M, H, D), dtype=torch.bfloat16, device=DEV)
        at = dp[b:b + 1].contiguous()
        _lib.check(lib.mxfp4_qk_norm_rope_kv(y.data_ptr(), w.data_ptr(), w.data_ptr(), 1e-6, 1e6, at.data_ptr(), M, H, Hkv_, D,
                                             out.data_ptr(), dummy[0].data_ptr(), dummy[1].data_ptr(), 16, 0,
                                             torch.cuda.current_stream().cuda_stream), "rope")
        return out

    rows = qkv.view(B, M, Hq + 2 * Hkv, D)
    k = torch.stack([rope(rows[b, :, Hq:Hq + Hkv], kw, b, Hkv) for b in range(B)])
    kv4.kv4_write(k, rows[:, :, Hq + Hkv:].bfloat16(), want, dp, pages)
    for b in range(B):
        assert torch.equal(q.view(B, M, Hq, D)[b], rope(rows[b, :, :Hq], qw, b, Hkv))
    assert got.kq.any() and all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("M,steps,kw", [(1, 3, {}), (1, 2, dict(qkv_tail=False)), (1, 2, dict(fused_router=False)), (4, 2, {}),
                                        (16, 2, {})])   # 16 tokens are what the MoE takes
def test_decode_step(tiny, M, steps, kw):  # noqa: F811
    model, wnp = tiny
    st = DecodeStep(model, CFG, M=M, max_pos=MAX_POS, device=DEV, kv="mxfp4", **kw)
    st.fill_cache(CTX, seed=5)
    ids, pos = np.array([(37 * (i + 1)) % CFG.vocab for i in range(M)], np.int32), CTX
    st.set_state(ids, CTX)
    torch.cuda.synchronize()
    for i in range(steps):
        host, xs = [[np_(t).copy() for t in c] for c in st.kv4], []

        def hook(l, xa, moe):
            torch.cuda.synchronize()
            xs.append(np_((xa.float() + moe.bfloat16().float()).bfloat16().float()))

        st.run(on_layer=hook)
        torch.cuda.synchronize()
        logits, nxt, what = np_(st.b.logits), np_(st.b.ids), f"M={M} step {i}"
        assert int(np_(st.b.dpos)[0]) == pos + M
        tf_logits, tf_xs = sref.step_ref(wnp, CFG, ids, pos, host, [None] * CFG.n_layers, M == 1, x_teacher=xs, kv_codec=sref.KV4)
        for l in range(CFG.n_layers):
            assert_close(xs[l], tf_xs[l], 0.99999, 5e-3, what=f"{what} layer {l} residual (same input)")
            for got, want in zip(st.kv4[l], host[l]):
                got, rows = np_(got), slice(pos, pos + M)
                assert np.array_equal(got[:, :, :pos], want[:, :, :pos]) and not got[:, :, pos + M:].any()
                assert np.mean(got[:, :, rows] == want[:, :, rows]) >= 0.98, f"{what} layer {l}: the rows written"
        assert_close(logits, tf_logits, 0.9999, 1e-2, what=f"{what} logits (same input)")
        assert np.array_equal(nxt, sref.argmax_ref(logits)), what
        ids, pos = nxt.copy(), pos + M


@pytest.mark.parametrize("M", [1, 4])
def test_graph_replays_match_eager(tiny, M):  # noqa: F811
    model, _ = tiny
    seqs = []
    for graph in (False, True):
        st = DecodeStep(model, CFG, M=M, max_pos=MAX_POS, device=DEV, kv="mxfp4")
        st.fill_cache(CTX, seed=5)
        st.set_state(list(range(101, 101 + M)), CTX)
        seq, replay = [], None
        for i in range(4):
            if graph and i == 0:
                replay = st.capture().replay          # runs the first step
            elif graph:
                _ = torch.randn(1024, device=DEV).sum().item()
                replay()
            else:
                st.run()
            torch.cuda.synchronize()
            seq.append((st.b.logits.clone(), st.b.ids.clone()))
        seqs.append((seq, st.kv4))
    for (a, b), (c, d) in zip(seqs[0][0], seqs[1][0]):
        assert torch.equal(a, c) and torch.equal(b, d)
    assert all(torch.equal(x, y) for p, q in zip(seqs[0][1], seqs[1][1]) for x, y in zip(p, q))


def test_refusals(tiny):  # noqa: F811
    model, _ = tiny
    with pytest.raises(RuntimeError, match="kv must be"):
        DecodeStep(model, CFG, max_pos=MAX_POS, device=DEV, kv="int4")
    with pytest.raises(RuntimeError, match="multiple of 16"):
        DecodeStep(model, CFG, max_pos=100, device=DEV, kv="mxfp4")
