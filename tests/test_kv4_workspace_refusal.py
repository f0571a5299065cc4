"""What attention over the MXFP4 cache says of a workspace that is too small, on the CPU: by addresses that are never read."""
import pytest

from moe_fused_inference_amd import _lib

P = 1 << 20


@pytest.mark.parametrize("window,sinks,tree", [(0, 0, None), (0, 0, P), (1024, 4, None), (1024, 4, P), (8192, 0, None)])
@pytest.mark.parametrize("given", [(P, 16), (None, 1 << 40), (P, -1)])
def test_the_function_that_says_its_size_is_named(window, sinks, tree, given):
    """By that function's own figure, and one byte less than it is refused."""
    lib, (ws, wsb) = _lib.load(), given
    if window:
        need, name = lib.mxfp4_attn_kv4_masked_workspace_size(8, 3, 8, 4, 128, 8192, window, sinks), "mxfp4_attn_kv4_masked_workspace_size"
    else:
        need, name = lib.mxfp4_attn_kv4_workspace_size(8, 3, 8, 4, 128, 8192), " mxfp4_attn_kv4_workspace_size"
    assert need > 16
    wsb = need - 1 if wsb == -1 else wsb
    rc = lib.mxfp4_attn_kv4_masked(P, 0, 8 * 128, P, P, P, P, None, 8, 8192, 0, P, window, sinks, tree, P, 2, None, None, 8, 3, 8, 4, 128, ws, wsb, None)
    said = lib.mxfp4_last_error().decode()
    assert rc == -1 and name in said and str(need) in said and f"of {wsb if ws else 0} bytes" in said, said
