"""GPU tests of the decode step with a window over the MXFP4 KV cache (DecodeStep(kv="mxfp4", window=, sinks=)); the rest of
the step is tests/test_gpu_kv4_step.py's."""
import pytest
import torch

from moe_fused_inference_amd import kv4
from moe_fused_inference_amd.decode_step import DecodeStep
from tests.gpu_helpers import DEV
from tests.test_gpu_decode_step import CFG, CTX, MAX_POS, tiny  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,window,sinks", [(1, 1, 0), (1, 20, 4), (4, 33, 0), (4, 7, 40), (16, 16, 1)])
def test_decode_step(tiny, M, window, sinks):  # noqa: F811
    """Every layer's attention is attn_decode4_mx of the layer's q over its cache with that window, bit for bit."""
    model, _ = tiny
    st = DecodeStep(model, CFG, M=M, max_pos=MAX_POS, device=DEV, kv="mxfp4", window=window, sinks=sinks)
    st.fill_cache(CTX, seed=5)
    ids = [(37 * (i + 1)) % CFG.vocab for i in range(M)]
    st.set_state(ids, CTX)
    for i in range(2):
        pos, seen = torch.tensor([CTX + i * M], dtype=torch.int32, device=DEV), []

        def hook(l, xa, moe):
            oq, os_ = kv4.attn_decode4_mx(st.b.q[None], st.kv4[l], pos, window=window, sinks=sinks)
            none, _ = kv4.attn_decode4_mx(st.b.q[None], st.kv4[l], pos)
            assert torch.equal(st.b.aq, oq) and torch.equal(st.b.as_, os_), l
            assert not torch.equal(none, oq)
            seen.append(l)

        st.run(on_layer=hook)
        assert seen == list(range(CFG.n_layers)) and int(st.b.dpos) == CTX + (i + 1) * M and st.b.logits.isfinite().all()


def _logits(model, change=None, **kw):
    st = DecodeStep(model, CFG, M=2, max_pos=MAX_POS, device=DEV, kv="mxfp4", **kw)
    st.fill_cache(CTX, seed=5)
    for c in st.kv4:
        for t in c:
            if change:
                t[:, :, change] ^= 8          # a sign, or a code's bit
    st.set_state([101, 102], CTX)
    g = st.capture()                          # runs a step
    first = st.b.logits.clone()
    for _ in range(2):
        _ = torch.randn(1024, device=DEV).sum().item()
        g.replay()
    torch.cuda.synchronize()
    return first, st.b.logits.clone()


def test_what_a_window_hides_does_not_matter(tiny):  # noqa: F811
    """What is before the window and past the sinks may hold anything, in captured steps too; and what they see matters."""
    model, _ = tiny
    window, sinks = 12, 3
    want = _logits(model, window=window, sinks=sinks)
    hidden = slice(sinks, CTX - window + 1)
    assert all(torch.equal(a, b) for a, b in zip(want, _logits(model, hidden, window=window, sinks=sinks)))
    for seen in (slice(sinks - 1, sinks), slice(CTX - window + 1, CTX - window + 2)):
        assert not torch.equal(want[0], _logits(model, seen, window=window, sinks=sinks)[0])


def test_a_window_of_everything_is_none(tiny):  # noqa: F811
    model, _ = tiny
    want = _logits(model)
    for kw in (dict(window=MAX_POS), dict(window=2 ** 40, sinks=2 ** 40)):
        assert all(torch.equal(a, b) for a, b in zip(want, _logits(model, **kw)))


def test_refusals(tiny):  # noqa: F811
    model, _ = tiny
    for kw in (dict(window=8), dict(kv="mxfp4", window=0), dict(kv="mxfp4", window=-3), dict(kv="mxfp4", sinks=2), dict(kv="mxfp4", window=4, sinks=-1)):
        with pytest.raises(RuntimeError, match="window"):
            DecodeStep(model, CFG, max_pos=MAX_POS, device=DEV, **kw)
