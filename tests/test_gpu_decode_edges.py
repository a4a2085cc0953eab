"""Decoding steps where they can go wrong without a wrong formula: values that are not finite or very large, lengths
near the largest, streams and pages that are shared.

Tolerances as in the tests of the operators' formulas: u is the unit roundoff of the 16-bit type; an output is rounded
once, every softmax weight once, and f32 scores are off by at most 2^-20 sum |q k| scale."""

import pytest
from test_gpu_decode import Batch

pytestmark = pytest.mark.gpu


def _torch():
    import torch

    return torch


# ------------------------------------------------------------------ streams
@pytest.mark.parametrize("kw", [dict(q=(1,) * 30, own=(3000,) * 30, prefix=(4000,)), dict(q=(1, 2), own=(9000, 40))])
def test_a_step_made_beside_a_busy_default_stream(cuda_device, kw):
    """Nothing that a step starts from waits in the default stream: made, planned and used on another stream while that
    one is busy, it gives the same bits."""
    torch = _torch()
    from ripvec_b200.decode import DecodeStep

    b = Batch(seed=80, **kw)
    want = b.step.attend(b.cache, b.queries)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    torch.cuda._sleep(1_000_000_000)  # half a second of the default stream
    with torch.cuda.stream(side):
        step = DecodeStep(q_heads=b.hq, kv_heads=b.hkv, head_dim=b.d, page_size=b.page)
        step.plan(q_lens=b.q_lens, own_lens=b.own_lens, own_pages=b.own_pages, num_pages=b.cache.num_pages,
                  prefix_lens=b.prefix_lens, prefix_pages=b.prefix_pages)
        outs = [step.attend(b.cache, b.queries) for _ in range(3)]
    side.synchronize()
    assert not torch.cuda.default_stream().query()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
