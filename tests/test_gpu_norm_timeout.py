"""The row wait of the streaming norms, made to run out on the host's word: the limit is lowered to a few milliseconds and the row loads
are withheld.  The kernel returns by itself, stores nothing over a residual that is updated in place, leaves a record that names the wait,
the next call is refused until it has been read, and the launch after that is healthy."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ST_TIMEOUT_ROWS = 0x107


@pytest.mark.parametrize("post", [False, True], ids=["one norm", "two norms"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("n", [4096, 4000, 12288, 1155], ids=["exact", "partial", "wide", "any width"])
def test_a_row_wait_that_runs_out(n, norm, post):
    import aiter_b200 as ab

    g = torch.Generator().manual_seed(n)
    x, w = (torch.randn(*s, generator=g).bfloat16().cuda() for s in ((8200, n), (n,)))
    r = torch.randn(8200, n, generator=g).bfloat16().cuda()

    def call(res):
        return ab.gated_residual_norm(x, res, w, post_weight=w if post else None, norm=norm, residual_out=res)

    want_h = r.clone()
    want_y = call(want_h)[0]
    assert ab.device_status(0) == (0, 0, 0, 0)
    kept = r.clone()
    try:
        ab.debug_wait_control(0, limit_ns=3_000_000, withhold_scales=True)
        call(kept)
        torch.cuda.synchronize()  # returns: every CTA gave up after ~3 ms
        assert torch.equal(kept, r), "rows that never arrived were stored"
        launches = ab.launch_count()
        with pytest.raises(RuntimeError, match="gave up on a wait"):
            call(kept)
        assert ab.launch_count() == launches
    finally:
        ab.debug_wait_control(0)  # defaults: 1 s, nothing withheld
    assert ab.device_status(0)[0] == ST_TIMEOUT_ROWS
    assert ab.device_status(0) == (0, 0, 0, 0)
    y = call(kept)[0]
    assert torch.equal(y, want_y) and torch.equal(kept, want_h)
    assert ab.device_status(0) == (0, 0, 0, 0)
