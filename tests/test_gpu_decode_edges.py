"""Decoding steps where they can go wrong without a wrong formula: values that are not finite or very large, lengths
near the largest, streams and pages that are shared.

Tolerances as in the tests of the operators' formulas: u is the unit roundoff of the 16-bit type; an output is rounded
once, every softmax weight once, and f32 scores are off by at most 2^-20 sum |q k| scale."""

import math

import pytest
from test_gpu_decode import UNIT, Batch

pytestmark = pytest.mark.gpu


def _torch():
    import torch

    return torch


# ------------------------------------------------------------------ values
# (what the step is, and which kernels take it)
STEPS = [
    dict(q=(1, 1, 2), own=(5, 200, 64), prefix=(0,)),                            # few rows, one part
    dict(q=(1, 1), own=(6000, 3), prefix=(0,)),                                  # few rows, cut keys, join
    dict(q=(1, 1, 2), own=(5, 200, 64), prefix=(300,)),                          # few rows, shared prefix, join
    dict(q=(200,), own=(260,), prefix=(0,)),                                     # row tiles, whole
    dict(q=(70, 90), own=(70, 133), prefix=(300,), hq=12, hkv=4, d=64, page=32),  # row tiles behind a prefix
    dict(q=(150,), own=(6000,), prefix=(0,), page=128),                          # row tiles, cut keys, join
    dict(q=(1,) * 48, own=tuple(1 + 7 * i for i in range(48)), prefix=(3000,)),  # packed prefix, few-row own keys, join
    dict(q=(1, 1, 2), own=(5, 200, 64), prefix=(300,), hq=12, hkv=4, d=64, page=32),  # few rows of 64 values, join
]


def softmax64(b, scale, exact_scores=False):
    """out, its tolerance, lse and its tolerance by a softmax in 64 bits, NaN and infinities as they come: zeros and
    -inf for a row that sees no key.  exact_scores: the f32 scores have no error."""
    torch = _torch()
    g, u = b.hq // b.hkv, UNIT[b.act]
    out = torch.zeros(b.t, b.hq, b.d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full((b.t, b.hq), -math.inf, dtype=torch.float64, device="cuda")
    lse_tol = torch.zeros_like(lse)
    t0 = 0
    for i, n in enumerate(b.q_lens):
        k, v = (b.keys(x, i).repeat_interleave(g, 0) for x in (b.k, b.v))
        keys = k.shape[1]
        if n and keys:
            q = b.queries[t0:t0 + n].double().transpose(0, 1)
            at = torch.arange(keys, device="cuda")
            seen = at[None, :] <= keys - n + torch.arange(n, device="cuda")[:, None]
            assert seen.any(-1).all()
            s = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
            off = (q.abs() @ k.abs().transpose(1, 2)).masked_fill(~seen, 0).nan_to_num(0, 0, 0).amax(-1) * scale * 2.0 ** -20
            if exact_scores:
                off = off * 0
            p = s.softmax(-1)
            o, a = p @ v, p @ v.abs()
            e = u * o.abs() + (u + 2.0 ** -16 + 2 * off[..., None]) * a
            if b.act == "f16":
                e = e + 2.0 ** -25 * keys * v.abs().nan_to_num(0).max()
            out[t0:t0 + n], tol[t0:t0 + n] = o.transpose(0, 1), e.transpose(0, 1) + 1e-7
            l = s.logsumexp(-1)
            l = l.masked_fill(l == math.inf, math.nan)  # as its row is
            lse[t0:t0 + n] = l.T
            lse_tol[t0:t0 + n] = (off + 2.0 ** -20 * (1 + l.abs().nan_to_num(0, 0, 0))).T
        t0 += n
    return out, tol, lse, lse_tol


def agree(b, exact_scores=False):
    torch = _torch()
    scale = b.d ** -0.5
    lse = torch.full((b.t, b.hq), 7.0, device="cuda")
    got = b.step.attend(b.cache, b.queries, lse=lse)
    torch.cuda.synchronize()
    ref, tol, ref_lse, lse_tol = softmax64(b, scale, exact_scores)
    for name, x, r, e in (("out", got, ref, tol), ("lse", lse, ref_lse, lse_tol)):
        assert torch.equal(x.isnan(), r.isnan()), f"{name}: {int(x.isnan().sum())} NaN, expected {int(r.isnan().sum())}"
        low = r == -math.inf
        assert (x[low] == -math.inf).all(), name
        fine = r.isfinite()
        assert ((x.double() - r).abs()[fine] <= e[fine]).all(), name
    return got, ref


def slot(b, seq, key):
    """Page and slot of an own key of a sequence."""
    return b.own_pages[seq][key // b.page], key % b.page


@pytest.mark.parametrize("act", ["bf16", "f16"])
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_attend_keeps_nan(cuda_device, act, step):
    """NaN in a query, in a key or in a value that a row sees makes what a softmax makes of it, in every kernel and join."""
    for what in ("query", "own key", "last key", "prefix key", "value"):
        b = Batch(act=act, seed=40 + step, **STEPS[step])
        if what == "query":
            b.queries[0, 0, 5] = math.nan
            b.queries[b.t - 1] = math.nan
        elif what == "own key":  # one that all of the sequence's queries see
            p, s = slot(b, 0, 0)
            if b.q_lens[0] > 1 or b.own_lens[0] == 1:
                b.k[p, 0, s, 3] = math.nan
            else:
                b.k[p, :, s] = math.nan
        elif what == "last key":  # one that its last query sees
            p, s = slot(b, len(b.q_lens) - 1, b.own_lens[-1] - 1)
            b.k[p, 0, s, 0] = math.nan
        elif b.prefix_lens[0] == 0:
            continue
        elif what == "prefix key":
            b.k[b.prefix_pages[0][2 // b.page], 1, 2 % b.page, 1] = math.nan
        else:
            b.v[b.prefix_pages[0][0], 0, 1, 7] = math.nan
        got, ref = agree(b)
        assert ref.isnan().any()
        assert what != "last key" or ref.isfinite().any() or b.t == 1


@pytest.mark.parametrize("act", ["bf16", "f16"])
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_attend_with_infinite_scores(cuda_device, act, step):
    """Scores of -inf have no weight beside others, make NaN alone; a score of inf makes NaN."""
    torch = _torch()
    for what in ("one key", "prefix", "all"):
        b = Batch(act=act, seed=50 + step, **STEPS[step])
        if what == "one key":
            p, s = slot(b, 0, 0)
            b.k[p, :, s, 0] = math.inf  # scores of either sign
        else:
            b.queries[..., 0] = -1.0
            for pages, n in zip(b.prefix_pages + b.own_pages * (what == "all"), b.prefix_lens + b.own_lens * (what == "all")):
                for i, p in enumerate(pages):
                    b.k[p, :, : min(b.page, n - i * b.page), 0] = math.inf
        got, ref = agree(b)
        assert ref.isnan().all() if what == "all" else ref.isfinite().any()


@pytest.mark.parametrize("act,power", [("bf16", 10), ("bf16", 13), ("bf16", 15), ("bf16", 30), ("f16", 10),
                                       ("f16", 12), ("f16", 14), ("f16", 15)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_attend_with_large_scores(cuda_device, act, power, sign, step):
    """Scores far beyond the range of exponents, as keys of a type's largest or lowest values make them: all powers of
    two, so that the f32 scores are exact, and the weights are those of the largest score's keys alone."""
    torch = _torch()
    b = Batch(act=act, seed=60 + step, **STEPS[step])
    b.queries.fill_(sign * 2.0 ** power)
    for pages, n in zip(b.prefix_pages + b.own_pages, b.prefix_lens + b.own_lens):
        for i, p in enumerate(pages):
            fill = min(b.page, n - i * b.page)
            at = i * b.page + torch.arange(fill, device="cuda")
            size = torch.where(at % 7 == 4, 2.0 ** (power - 1), 2.0 ** power)
            b.k[p, :, :fill] = size[None, :, None].to(b.k.dtype)
    agree(b, exact_scores=True)


@pytest.mark.parametrize("act,power", [("bf16", 10), ("bf16", 13), ("bf16", 15), ("bf16", 30), ("bf16", 50), ("f16", 10),
                                       ("f16", 12), ("f16", 14), ("f16", 15)])
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_attend_with_large_inexact_scores(cuda_device, act, power, step):
    """As before with scores that the factor of the exponent rounds (1.5 times a power of two, and 0.75)."""
    torch = _torch()
    for sign in (1, -1):
        b = Batch(act=act, seed=90 + step, **STEPS[step])
        b.queries.fill_(sign * 2.0 ** power)
        for pages, n in zip(b.prefix_pages + b.own_pages, b.prefix_lens + b.own_lens):
            for i, p in enumerate(pages):
                fill = min(b.page, n - i * b.page)
                at = i * b.page + torch.arange(fill, device="cuda")
                size = torch.where(at % 7 == 4, 0.75 * 2.0 ** power, 1.5 * 2.0 ** power)
                b.k[p, :, :fill] = size[None, :, None].to(b.k.dtype)
        agree(b, exact_scores=True)


# ------------------------------------------------------------------ lengths
def test_attend_causal_limits_of_very_long_sequences(cuda_device):
    """Several row tiles of new tokens after 2^29 keys (pages may be read many times): each sees its own limit."""
    import numpy as np

    torch = _torch()
    from ripvec_b200.decode import DecodeStep, PagedCache

    past, n, ps, d = 2 ** 29, 300, 256, 64
    k = torch.zeros(3, 1, ps, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator(device="cuda").manual_seed(70)
    new_v = torch.randn(n, d, generator=g, device="cuda").to(k.dtype)
    k.view(3 * ps, d)[ps:ps + n, 0] = 320.0
    v.view(3 * ps, d)[ps:ps + n] = new_v
    q = torch.zeros(n, 1, d, dtype=k.dtype, device="cuda")
    q[..., 0] = 1.0  # scores 40 for the new tokens' keys, 0 for the others
    pages = np.zeros((1, past // ps + 2), np.int32)
    pages[0, -2:] = 1, 2
    step = DecodeStep(q_heads=1, kv_heads=1, head_dim=d, page_size=ps)
    step.plan(q_lens=[n], own_lens=[past + n], own_pages=pages, num_pages=3)
    got = step.attend(PagedCache(k, v), q)[:, 0].double()
    w = math.exp(40.0)
    count = torch.arange(1, n + 1, device="cuda", dtype=torch.float64)[:, None]
    ref, a = (x.double().cumsum(0) * w / (count * w + past) for x in (new_v, new_v.abs()))
    assert ((got - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -16) * a).all()


@pytest.mark.parametrize("causal", [True, False])
def test_attend_the_most_keys(cuda_device, causal):
    """2^30 keys, the most that a sequence may have: the last one counts."""
    import numpy as np

    torch = _torch()
    from ripvec_b200.decode import DecodeStep, PagedCache

    keys, ps, d = 2 ** 30, 256, 64
    k = torch.zeros(2, 1, ps, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    k[1, 0, -1, 0] = 320.0
    v[1, 0, -1] = torch.randn(d, generator=torch.Generator(device="cuda").manual_seed(71), device="cuda").to(k.dtype)
    q = torch.zeros(1, 1, d, dtype=k.dtype, device="cuda")
    q[..., 0] = 1.0  # a score of 40 for the last key, 0 for the others
    pages = np.zeros((1, keys // ps), np.int32)
    pages[0, -1] = 1
    step = DecodeStep(q_heads=1, kv_heads=1, head_dim=d, page_size=ps)
    step.plan(q_lens=[1], own_lens=[keys], own_pages=pages, num_pages=2, causal=causal)
    got = step.attend(PagedCache(k, v), q)[0, 0].double()
    w = math.exp(40.0)
    ref = v[1, 0, -1].double() * w / (w + keys - 1)
    assert ((got - ref).abs() <= (2.0 ** -7 + 2.0 ** -16) * ref.abs()).all()


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


@pytest.mark.parametrize("call", ["append", "attend", "norm", "norm 8 bit"])
def test_outputs_on_a_given_stream(cuda_device, call):
    """An output that a call makes itself is the given stream's memory: what the current stream still has to read is
    not written."""
    torch = _torch()
    from ripvec_b200.decode import rms_norm

    b = Batch(q=(1,) * 64, own=(40,) * 64, prefix=(100,), seed=71)
    cos, sin = torch.ones(200, 64, device="cuda"), torch.zeros(200, 64, device="cuda")
    kn = b.randn(b.t, b.hkv, b.d)
    x, w = b.randn(64, 4096), torch.ones(4096, device="cuda")
    side = torch.cuda.Stream()

    def run(stream):
        if call == "append":
            return (b.step.append(b.cache, b.queries, kn, kn, cos, sin, stream=stream),)
        if call == "attend":
            return (b.step.attend(b.cache, b.queries, stream=stream),)
        return rms_norm(x, w, out_8bit=call != "norm", stream=stream)

    want = [None if y is None else y.clone() for y in run(None)]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    kept = []
    for y in want:  # blocks that the current stream's next outputs of these sizes would get
        if y is not None:
            old = torch.zeros_like(y)
            kept.append((old, torch.ones_like(y)))
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)  # a fifth of a second
    for i, (old, copy) in enumerate(kept):
        copy.copy_(old)
        kept[i] = copy
    del old
    got = run(side.cuda_stream)
    side.synchronize()
    assert not torch.cuda.current_stream().query()  # the copies are still to come
    torch.cuda.synchronize()
    for y, z in zip(want, got):
        assert (y is None and z is None) or torch.equal(y.view(torch.uint8), z.view(torch.uint8))
    for copy in kept:
        assert (copy.view(torch.uint8) == 0).all()


@pytest.mark.parametrize("handle", [0, 1, 2])
def test_streams_without_an_object(cuda_device, handle):
    """The default stream by its two handles, and the calling thread's."""
    torch = _torch()
    from ripvec_b200.decode import rms_norm

    b = Batch(q=(1, 3), own=(40, 60), prefix=(100,), seed=76)
    x, w = b.randn(5, 256), torch.ones(256, device="cuda")
    for side in (torch.cuda.default_stream(), torch.cuda.Stream()):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = b.step.attend(b.cache, b.queries, stream=handle), *rms_norm(x, w, out_8bit=True, stream=handle)
        torch.cuda.synchronize()
        want = b.step.attend(b.cache, b.queries), *rms_norm(x, w, out_8bit=True)
        assert all(torch.equal(g.view(torch.uint8), e.view(torch.uint8)) for g, e in zip(got, want))


def test_one_handle_for_a_stream_of_each_thread(cuda_device):
    """cudaStreamPerThread is one handle and, in each host thread, another stream: a call waits for the step's earlier
    call of another thread."""
    import threading
    import time

    torch = _torch()
    b = Batch(q=(1,) * 30, own=(3000,) * 30, prefix=(4000,), seed=74)
    want = b.step.attend(b.cache, b.queries)
    outs = [torch.zeros_like(want) for _ in range(2)]
    done = [torch.cuda.Event() for _ in range(2)]
    torch.cuda.synchronize()
    queued, checked = threading.Event(), threading.Event()

    def first():
        with torch.cuda.stream(torch.cuda.ExternalStream(2)):
            torch.cuda._sleep(1_000_000_000)  # half a second
            b.step.attend(b.cache, b.queries, out=outs[0])
            done[0].record()
        queued.set()
        checked.wait(60)

    thread = threading.Thread(target=first)
    thread.start()
    assert queued.wait(60)
    with torch.cuda.stream(torch.cuda.ExternalStream(2)):
        b.step.attend(b.cache, b.queries, out=outs[1])
        done[1].record()
    time.sleep(0.1)
    late = done[1].query()
    busy = not done[0].query()
    checked.set()
    thread.join()
    torch.cuda.synchronize()
    assert busy and not late
    assert all(torch.equal(o, want) for o in outs)


def test_one_step_in_many_threads(cuda_device):
    """Threads that call one step, each on a stream of its own."""
    import threading

    torch = _torch()
    b = Batch(q=(1,) * 30, own=(300,) * 30, prefix=(4000,), seed=75)
    want = b.step.attend(b.cache, b.queries)
    torch.cuda.synchronize()
    wrong = []

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            outs = [b.step.attend(b.cache, b.queries) for _ in range(20)]
        stream.synchronize()
        wrong.extend(1 for o in outs if not torch.equal(o, want))

    threads = [threading.Thread(target=work) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------------------ refusals
def test_append_refuses_pages_that_others_read(cuda_device):
    """New tokens would overwrite keys that the step reads: a page among another sequence's earlier ones, or twice in a
    sequence's own list.  Without queries nothing is read, and pages that are only read may be shared."""
    torch = _torch()
    from ripvec_b200 import _lib as L

    b = Batch(q=(2, 1), own=(20, 40), prefix=(40,), seed=72)
    cos = torch.ones(100, 64, device="cuda")
    k = b.randn(3, 2, 128)
    (a0, a1), (b0, b1, b2) = b.own_pages

    def plan(pages, q_lens=(2, 1)):
        b.step.plan(q_lens=q_lens, own_lens=[20, 40], own_pages=pages, prefix_lens=[40], prefix_pages=b.prefix_pages,
                    num_pages=b.cache.num_pages)

    for pages in ([[a0, a1], [b0, a1, b2]], [[a1, a1], [b0, b1, b2]], [[a0, a1], [b2, b1, b2]], [[b2, a1], [b0, b1, b2]]):
        plan(pages)
        with pytest.raises(L.RvError):
            b.step.append(b.cache, b.queries, k, k, cos, cos)
        b.step.attend(b.cache, b.queries)
    plan([[a0, a1], [a0, b1, b2]])  # an earlier page that both read
    b.step.append(b.cache, b.queries, k, k, cos, cos)
    plan([[a0, a1], [a0, a1, b2]], q_lens=(2, 0))  # a sequence that rests
    b.step.append(b.cache, b.queries[:2], k[:2], k[:2], cos, cos)
    torch.cuda.synchronize()


def test_append_refuses_outputs_that_overlap(cuda_device):
    """As attend does: rotated queries of several tokens or heads in one place."""
    torch = _torch()
    from ripvec_b200 import _lib as L

    b = Batch(q=(2, 1), own=(20, 40), seed=73)
    cos = torch.ones(100, 64, device="cuda")
    k = b.randn(3, 2, 128)
    for shape in ((1, 8, 128), (3, 1, 128)):
        one = torch.zeros(shape, dtype=k.dtype, device="cuda").expand(3, 8, 128)
        with pytest.raises(L.RvError):
            b.step.append(b.cache, b.queries, k, k, cos, cos, q_out=one)
    torch.cuda.synchronize()
