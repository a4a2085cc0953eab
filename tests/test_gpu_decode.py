"""Decoder-side operators on the GPU (paged rotary append, shared-prefix attention, residual RMS norm)
against plain implementations in 64 bits.

Tolerances.  u is the unit roundoff of the 16-bit type (2^-8 bf16, 2^-11 f16).  Attention: the output is
rounded once (u |ref|), every softmax weight once (u sum p |v|, and 2^-25 each where f16 underflows), and
f32 scores are off by at most 2^-20 sum |q k| scale, which moves weights by as much.  Rotation: one
rounding (2^-25 where f16 underflows) and f32 products.  Norm: one rounding and f32 statistics; e4m3 codes half a step of 2^-3, or of
2^-9 below the normal range."""

import math

import pytest

pytestmark = pytest.mark.gpu

UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _torch():
    import torch

    return torch


def _dtype(name):
    torch = _torch()
    return torch.bfloat16 if name == "bf16" else torch.float16


class Batch:
    """Pools, page lists and a plan; unused slots of the pools hold NaN."""

    def __init__(self, *, act="bf16", hq=8, hkv=2, d=128, page=16, q=(1,), own=(1,), prefix=(0,), groups=None,
                 causal=True, seed=0, layout="head", std=2.0):
        torch = _torch()
        from ripvec_b200.decode import DecodeStep, PagedCache

        self.act, self.hq, self.hkv, self.d, self.page, self.causal = act, hq, hkv, d, page, causal
        self.q_lens, self.own_lens, self.prefix_lens = list(q), list(own), list(prefix)
        self.groups = [len(q)] if groups is None else list(groups)
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        dt = _dtype(act)
        need = [-(-n // page) for n in self.prefix_lens + self.own_lens]
        total = sum(need) + 2
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
        lists = []
        for k in need:
            lists.append(order[:k])
            order = order[k:]
        self.prefix_pages, self.own_pages = lists[:len(self.prefix_lens)], lists[len(self.prefix_lens):]
        shape = (total, hkv, page, d)
        if layout == "head":
            self.k, self.v = (torch.full(shape, math.nan, dtype=dt, device="cuda") for _ in range(2))
        else:  # token-major memory, wider rows than the head dim
            self.k, self.v = (torch.full((page, total, hkv, d + 8), math.nan, dtype=dt, device="cuda")[..., :d]
                              .permute(1, 2, 0, 3) for _ in range(2))
        for pages, n in zip(self.prefix_pages + self.own_pages, self.prefix_lens + self.own_lens):
            for pool in (self.k, self.v):
                for i, p in enumerate(pages):
                    fill = min(page, n - i * page)
                    pool[p, :, :fill] = self.randn(hkv, fill, d)
        self.t = sum(self.q_lens)
        self.queries = self.randn(self.t, hq, d, std=std)
        self.cache = PagedCache(self.k, self.v)
        self.step = DecodeStep(q_heads=hq, kv_heads=hkv, head_dim=d, page_size=page)
        self.step.plan(q_lens=self.q_lens, own_lens=self.own_lens, own_pages=self.own_pages, num_pages=total,
                       prefix_lens=self.prefix_lens, prefix_pages=self.prefix_pages, group_sizes=self.groups,
                       causal=causal)

    def randn(self, *shape, std=1.0):
        torch = _torch()
        return (torch.randn(*shape, generator=self.gen, device="cuda") * std).to(_dtype(self.act))

    def group_of(self, b):
        at = 0
        for g, n in enumerate(self.groups):
            at += n
            if b < at:
                return g

    def keys(self, pool, b):
        """[kv_heads, prefix + own, d] in f64."""
        torch = _torch()
        g = self.group_of(b)
        parts = [pool[p].transpose(0, 1) for p in self.prefix_pages[g]]
        pre = torch.cat(parts)[: self.prefix_lens[g]] if parts else pool[0, :, :0].transpose(0, 1)
        parts = [pool[p].transpose(0, 1) for p in self.own_pages[b]]
        own = torch.cat(parts)[: self.own_lens[b]] if parts else pool[0, :, :0].transpose(0, 1)
        return torch.cat((pre, own)).transpose(0, 1).double()

    def reference(self, scale):
        torch = _torch()
        g = self.hq // self.hkv
        out = torch.zeros(self.t, self.hq, self.d, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        lse = torch.full((self.t, self.hq), -math.inf, dtype=torch.float64, device="cuda")
        lse_tol = torch.zeros_like(lse)
        u = UNIT[self.act]
        t0 = 0
        for b, n in enumerate(self.q_lens):
            k, v = (self.keys(x, b).repeat_interleave(g, 0) for x in (self.k, self.v))
            keys, pre = k.shape[1], k.shape[1] - self.own_lens[b]
            if n and keys:
                q = self.queries[t0:t0 + n].double().transpose(0, 1)
                s = q @ k.transpose(1, 2) * scale
                off = (q.abs() @ k.abs().transpose(1, 2)).amax(-1) * scale * 2.0 ** -20
                if self.causal:
                    at = torch.arange(keys, device="cuda")
                    lim = pre + self.own_lens[b] - n + torch.arange(n, device="cuda")
                    s = s.masked_fill(at[None, :] > lim[:, None].clamp(min=pre - 1), -math.inf)
                m = s.amax(-1, keepdim=True)
                p = torch.where(m == -math.inf, torch.zeros_like(s), (s - m.clamp(min=-1e300)).exp())
                l = p.sum(-1, keepdim=True)
                p = p / l.clamp(min=1e-300)
                o = p @ v
                a = p @ v.abs()
                e = u * o.abs() + (u + 2 * off[..., None]) * a + 2.0 ** -25 * keys * (v.abs().max() if self.act == "f16" else 0)
                out[t0:t0 + n], tol[t0:t0 + n] = o.transpose(0, 1), e.transpose(0, 1) + 1e-7
                le = (m + l.log()).squeeze(-1)
                lse[t0:t0 + n] = le.T
                lse_tol[t0:t0 + n] = (off + 2.0 ** -20 * (1 + le.abs().nan_to_num(posinf=0))).T
            t0 += n
        return out, tol, lse, lse_tol

    def check(self, scale=None, out=None, queries=None, with_lse=True, stream=None):
        torch = _torch()
        lse = torch.full((self.t, self.hq), 7.0, device="cuda") if with_lse else None
        got = self.step.attend(self.cache, self.queries if queries is None else queries, out=out, lse=lse, scale=scale,
                               stream=stream)
        torch.cuda.synchronize()
        ref, tol, ref_lse, lse_tol = self.reference(self.d ** -0.5 if scale is None else scale)
        err = (got.double() - ref).abs()
        assert torch.isfinite(got).all()
        assert (err <= tol).all(), f"largest error over tolerance {(err / tol.clamp(min=1e-30)).max().item():.3g}"
        if with_lse:
            empty = ref_lse == -math.inf
            assert (lse[empty] == -math.inf).all()
            assert ((lse.double() - ref_lse).abs()[~empty] <= lse_tol[~empty]).all()
        return got


HEADS = [(12, 12, 64), (12, 4, 64), (8, 2, 128), (7, 1, 128), (16, 2, 128), (20, 1, 64), (32, 1, 128), (40, 8, 128),
         (1, 1, 64), (17, 1, 128)]


@pytest.mark.parametrize("act", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_attend_heads(cuda_device, act, hq, hkv, d):
    """Single tokens, short and long chunks of several sequences behind one prefix, every head layout."""
    Batch(act=act, hq=hq, hkv=hkv, d=d, page=32, q=(1, 1, 1, 1, 1), own=(1, 2, 65, 300, 32), prefix=(77,), seed=1).check()
    Batch(act=act, hq=hq, hkv=hkv, d=d, page=32, q=(3, 40, 129, 1), own=(3, 60, 129, 500), prefix=(200,), seed=2).check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("prefix", [0, 1, 15, 64, 127, 128, 129, 333, 1000])
def test_attend_prefix_lengths(cuda_device, page, prefix):
    own = (1, 17, 63, 64, 65, 127, 128, 129, 256, 257)
    Batch(page=page, q=(1,) * len(own), own=own, prefix=(prefix,), seed=prefix).check()
    Batch(page=page, q=(70, 5, 33), own=(70, 133, 161), prefix=(prefix,), act="f16", hq=12, hkv=4, d=64,
          seed=prefix).check()


@pytest.mark.parametrize("n", [1, 2, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 700])
def test_attend_one_prompt(cuda_device, n):
    """A causal prompt alone, at lengths around the tile sizes; and the same rows without the mask."""
    Batch(q=(n,), own=(n,), seed=n).check()
    Batch(q=(n,), own=(n,), hq=12, hkv=12, d=64, page=64, act="f16", seed=n).check()
    Batch(q=(n,), own=(n,), causal=False, hq=3, hkv=1, page=128, seed=n).check()


def test_attend_long_keys(cuda_device):
    """Long key ranges, which are split and joined: few rows, and many rows over a long prefix."""
    Batch(q=(1, 1), own=(20000, 3), page=64, hq=8, hkv=2, seed=3).check()
    Batch(q=(1,) * 48, own=tuple(1 + 7 * i for i in range(48)), prefix=(9000,), page=64, hq=28, hkv=4, seed=4).check()
    Batch(q=(1,) * 100, own=(1,) * 100, prefix=(5000,), page=16, hq=12, hkv=4, d=64, act="f16", seed=5).check()
    Batch(q=(150,), own=(6000,), page=128, seed=6).check()
    Batch(q=(1, 300, 1, 2), own=(1, 2300, 4000, 9), prefix=(3000,), page=32, seed=7).check()


def test_attend_middle_lengths_over_a_long_prefix(cuda_device):
    """Sequences of one to four row tiles over a prefix so long that they share its walk; beside longer and shorter ones."""
    Batch(q=(20,) * 5, own=(20, 21, 150, 83, 400), prefix=(4000,), page=64, seed=31).check()
    Batch(q=(1, 20, 30, 0, 250, 25, 300, 16), own=(1, 100, 30, 9, 250, 7, 310, 0), prefix=(9000,), page=128, seed=32).check()
    Batch(q=(20, 33, 17), own=(20, 5, 90), prefix=(5000,), causal=False, hq=28, hkv=4, seed=33).check()
    Batch(q=(70, 127, 129, 255, 64), own=(70, 300, 129, 0, 100), prefix=(12000,), hq=12, hkv=12, d=64, page=32, act="f16",
          seed=34).check()
    Batch(q=(17, 19, 40, 40, 18), own=(17, 30, 40, 41, 18), prefix=(6000, 100, 7000), groups=(2, 2, 1), page=256, seed=35).check()


def test_attend_groups(cuda_device):
    """Several prefixes in one step, some empty, some groups without sequences or tokens."""
    Batch(q=(1, 1, 5, 0, 1, 64), own=(4, 9, 5, 30, 0, 64), prefix=(130, 0, 64, 10), groups=(2, 0, 3, 1), seed=8).check()
    Batch(q=(1,) * 70, own=(1 + 5,) * 70, prefix=(300, 0, 40), groups=(33, 30, 7), hq=4, hkv=1, seed=9).check()


def test_attend_rows_that_see_nothing(cuda_device):
    """No key at all, and causal rows before the first key: zeros and a log-sum of -inf."""
    b = Batch(q=(1, 2, 1), own=(0, 0, 3), seed=10)
    got = b.check()
    assert (got[:3] == 0).all()
    for n, own in ((5, 2), (200, 3), (300, 130)):
        got = Batch(q=(n, 1), own=(own, 1), hq=4, hkv=1, seed=11).check()
        assert (got[: n - own] == 0).all() and (got[n - own:n] != 0).any()
    got = Batch(q=(40,) * 4, own=(0, 40, 0, 7), hq=4, hkv=1, seed=12, causal=False).check()
    assert (got[:40] == 0).all() and (got[80:120] == 0).all()


def test_attend_only_the_prefix(cuda_device):
    """Sequences without keys of their own read the shared memory alone."""
    Batch(q=(1, 33, 200, 4), own=(0, 0, 0, 0), prefix=(450,), seed=13).check()


@pytest.mark.parametrize("std,scale", [(30.0, None), (0.01, None), (2.0, 0.003), (2.0, 3.0)])
def test_attend_score_ranges(cuda_device, std, scale):
    """Softmaxes that one key decides, and nearly flat ones."""
    Batch(q=(1, 1, 60), own=(100, 300, 400), prefix=(500,), std=std, seed=14).check(scale=scale)
    Batch(q=(1, 1, 60), own=(100, 300, 400), prefix=(500,), std=std, act="f16", seed=15).check(scale=scale)


def test_attend_growing_scores(cuda_device):
    """Keys whose scores grow along the sequence move the running maximum in every tile."""
    torch = _torch()
    for q, own, prefix in (((1,), (1500,), 0), ((200,), (900,), 600), ((1,) * 40, (65,) * 40, 700)):
        b = Batch(q=q, own=own, prefix=(prefix,), seed=16)
        for pages in b.prefix_pages + b.own_pages:
            for i, p in enumerate(pages):
                b.k[p, ..., 0] = (0.5 * i * b.page / 16 + 0.02 * torch.arange(b.page, device="cuda")).to(b.k.dtype)
        b.queries[..., 0] = 8.0
        b.check()


def test_attend_strides(cuda_device):
    """Queries inside a packed projection, an output with gaps, pools in token-major order."""
    torch = _torch()
    for q, own, prefix in (((1, 1, 1), (5, 200, 64), 300), ((130, 3), (150, 3), 100)):
        b = Batch(q=q, own=own, prefix=(prefix,), layout="token", seed=17)
        wide = torch.zeros(b.t, b.hq * b.d + 3 * 64, dtype=b.queries.dtype, device="cuda")
        wide[:, 64: 64 + b.hq * b.d] = b.queries.reshape(b.t, -1)
        out = torch.full((b.t, b.hq + 1, 2 * b.d), 5.0, dtype=b.queries.dtype, device="cuda")
        view = out[:, 1:, b.d:]
        b.check(queries=wide[:, 64: 64 + b.hq * b.d].view(b.t, b.hq, b.d), out=view)
        assert (out[:, 0] == 5).all() and (out[:, :, : b.d] == 5).all()


def test_attend_without_lse_and_twice(cuda_device):
    """The same bits from every run of the same plan."""
    torch = _torch()
    b = Batch(q=(1, 1, 70, 1), own=(3000, 1, 100, 40), prefix=(2000,), seed=18)
    first = b.check(with_lse=False).clone()
    for _ in range(3):
        assert torch.equal(b.step.attend(b.cache, b.queries), first)


def test_attend_over_large_offsets(cuda_device):
    """Pages whose elements lie more than 2^31 elements into the pool."""
    torch = _torch()
    from ripvec_b200.decode import DecodeStep, PagedCache

    pages, hkv, ps, d = 2 ** 31 // (2 * 256 * 128) + 40, 2, 256, 128
    k = torch.empty(pages, hkv, ps, d, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    use = [pages - 1, 0, pages - 3, pages - 2, 5]
    g = torch.Generator(device="cuda").manual_seed(19)
    for p in use:
        k[p] = torch.randn(hkv, ps, d, generator=g, device="cuda").to(k.dtype)
        v[p] = torch.randn(hkv, ps, d, generator=g, device="cuda").to(k.dtype)
    small = PagedCache(k[use].contiguous(), v[use].contiguous())
    outs = []
    for cache, pre, own in ((PagedCache(k, v), use[:2], [[use[2]], use[3:5]]), (small, [0, 1], [[2], [3, 4]])):
        step = DecodeStep(q_heads=8, kv_heads=2, head_dim=d, page_size=ps)
        step.plan(q_lens=[1, 200], own_lens=[100, 400], own_pages=own, prefix_lens=[300], prefix_pages=[pre],
                  num_pages=cache.num_pages)
        q = torch.randn(201, 8, d, generator=torch.Generator(device="cuda").manual_seed(20), device="cuda").to(k.dtype)
        kn = q[:, :2] * 0.5
        cos, sin = torch.ones(700, 64, device="cuda"), torch.zeros(700, 64, device="cuda")
        step.append(cache, q, kn, kn, cos, sin)
        outs.append(step.attend(cache, q))
    assert torch.equal(outs[0], outs[1])


def test_streams(cuda_device):
    """A step used from several streams: each call waits for the step's earlier calls."""
    torch = _torch()
    b = Batch(q=(1,) * 30, own=(3000,) * 30, prefix=(4000,), seed=21)
    want = b.step.attend(b.cache, b.queries).clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(b.step.attend(b.cache, b.queries))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_graph_capture(cuda_device):
    """A captured layer replays on new queries."""
    torch = _torch()
    b = Batch(q=(1,) * 20, own=(90,) * 20, prefix=(700,), seed=22)
    cos, sin = torch.ones(1000, 64, device="cuda"), torch.zeros(1000, 64, device="cuda")
    kn, vn = b.randn(b.t, b.hkv, b.d), b.randn(b.t, b.hkv, b.d)
    out = torch.empty_like(b.queries)
    b.step.append(b.cache, None, kn, vn, cos, sin)
    b.step.attend(b.cache, b.queries, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.step.append(b.cache, None, kn, vn, cos, sin)
        b.step.attend(b.cache, b.queries, out=out)
    for k in range(2):
        kn.copy_(b.randn(b.t, b.hkv, b.d))
        b.queries.copy_(b.randn(b.t, b.hq, b.d))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, b.check())


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("act", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d,rot,interleaved", [(12, 12, 64, 64, False), (8, 2, 128, 128, False),
                                                      (7, 1, 128, 64, True), (4, 4, 64, 64, True), (3, 1, 64, 2, False),
                                                      (3, 1, 128, 18, True), (4, 2, 128, 0, False), (32, 8, 128, 32, False)])
def test_append_matches_the_rotation(cuda_device, act, hq, hkv, d, rot, interleaved):
    torch = _torch()
    for packed, layout in ((True, "head"), (False, "token")):
        b = Batch(act=act, hq=hq, hkv=hkv, d=d, page=16, q=(1, 33, 5, 0, 130), own=(1, 40, 500, 7, 130), prefix=(19, 300),
                  groups=(2, 3), layout=layout, seed=rot)
        positions = 300 + 500
        ang = torch.rand(positions, rot // 2, device="cuda", generator=b.gen) * 6.28
        cos, sin = ang.cos(), ang.sin()
        if packed:
            x = b.randn(b.t, (hq + 2 * hkv) * d)
            q, k, v = x[:, : hq * d].view(b.t, hq, d), x[:, hq * d:(hq + hkv) * d].view(b.t, hkv, d), x[:, (hq + hkv) * d:].view(b.t, hkv, d)
        else:
            q, k, v = (b.randn(h, b.t, d).transpose(0, 1) for h in (hq, hkv, hkv))
        before_k, before_v = b.k.clone(), b.v.clone()
        q_in = q.clone()
        got = b.step.append(b.cache, q, k, v, cos, sin, interleaved=interleaved)
        torch.cuda.synchronize()
        assert torch.equal(q, q_in)
        pos, page, slot = [], [], []
        for s, n in enumerate(b.q_lens):
            for i in range(n):
                place = b.own_lens[s] - n + i
                pos.append(b.prefix_lens[b.group_of(s)] + place)
                page.append(b.own_pages[s][place // b.page])
                slot.append(place % b.page)
        pos, page, slot = (torch.tensor(a, device="cuda") for a in (pos, page, slot))

        def turned(x):
            x = x.double()
            y, e = x.clone(), x.abs() * 0
            i0 = torch.arange(rot // 2, device="cuda") * (2 if interleaved else 1)
            i1 = i0 + (1 if interleaved else rot // 2)
            c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
            y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
            e[..., i0] = e[..., i1] = x[..., i0].abs() + x[..., i1].abs()
            return y, (UNIT[act] * y.abs() + (2.0 ** -25 if act == "f16" else 0)) * (e > 0) + 2.0 ** -22 * e

        for out, src in ((got, q_in), (b.k[page, :, slot], k)):
            ref, tol = turned(src)
            assert ((out.double() - ref).abs() <= tol).all()
        assert torch.equal(b.v[page, :, slot], v)
        before_k[page, :, slot] = b.k[page, :, slot]
        before_v[page, :, slot] = v
        for now, was in ((b.k, before_k), (b.v, before_v)):
            assert torch.equal(now.contiguous().view(torch.int16), was.contiguous().view(torch.int16))
        same = q.clone()  # in place, and keys and values alone
        b.step.append(b.cache, same, k, v, cos, sin, q_out=same, interleaved=interleaved)
        assert torch.equal(same, got.contiguous())
        k_now = b.k.clone()
        b.step.append(b.cache, None, k, v, cos, sin, interleaved=interleaved)
        assert torch.equal(k_now.view(torch.int16), b.k.clone().view(torch.int16))


def test_append_unaligned_rows(cuda_device):
    """Rows that do not start on 16 bytes go through the same call."""
    torch = _torch()
    b = Batch(hq=3, hkv=1, d=64, q=(20, 4), own=(20, 9), seed=23)
    ang = torch.rand(40, 32, device="cuda", generator=b.gen) * 6.28
    cos, sin = ang.cos(), ang.sin()
    x = b.randn(b.t, 5 * 64 + 3)
    q, k, v = x[:, 1:193].view(b.t, 3, 64), x[:, 193:257].view(b.t, 1, 64), x[:, 257:321].view(b.t, 1, 64)
    got = b.step.append(b.cache, q, k, v, cos, sin)
    kp, vp = b.k.clone(), b.v.clone()
    want = b.step.append(b.cache, q.clone(), k.clone(), v.clone(), cos, sin)
    assert torch.equal(got, want)
    assert torch.equal(kp.view(torch.int16), b.k.view(torch.int16)) and torch.equal(vp.view(torch.int16), b.v.view(torch.int16))


# ------------------------------------------------------------------ norm
def _norm_reference(x, residual, weight, eps):
    h = x.double() + (residual.double() if residual is not None else 0)
    return h, weight.double() * h / ((h * h).mean(-1, keepdim=True) + eps).sqrt()


@pytest.mark.parametrize("act", ["bf16", "f16"])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (1, 768), (3, 7), (5, 384), (64, 4096), (2, 4095), (300, 768), (7, 8192),
                                         (3, 16384), (2, 20001), (1, 65536), (2000, 128), (1000, 64), (5, 1000)])
@pytest.mark.parametrize("with_residual", [True, False])
def test_rms_norm(cuda_device, act, rows, hidden, with_residual):
    torch = _torch()
    from ripvec_b200.decode import rms_norm

    g = torch.Generator(device="cuda").manual_seed(rows * 31 + hidden)
    dt, u = _dtype(act), UNIT[act]
    x = torch.randn(rows, hidden, generator=g, device="cuda").to(dt)
    r = (torch.randn(rows, hidden, generator=g, device="cuda") * 4).to(dt) if with_residual else None
    w = 1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")
    x[-1] = 0
    if r is not None:
        r[-1] = 0  # a row of zeros
    h, y = _norm_reference(x, r, w, 1e-5)
    ro = torch.full_like(x, 9)
    out, scales = rms_norm(x, w, residual=r, residual_out=ro)
    assert scales is None
    assert ((out.double() - y).abs() <= (u + 1e-5) * y.abs() + 2.0 ** -25).all()
    assert ((ro.double() - h).abs() <= u * h.abs()).all()
    groups = [0] + [k for k in (32, 64, 128, 256) if hidden % k == 0]
    for group in groups:
        ro.fill_(9)
        codes, scales = rms_norm(x, w, residual=r, residual_out=ro, out_8bit=True, group=group)
        assert ((ro.double() - h).abs() <= u * h.abs()).all()
        yg = y.view(rows, -1, group or hidden)
        ref = yg.abs().amax(-1).clamp(min=1e-12) / 448
        assert ((scales.double() - ref).abs() <= 1e-5 * ref).all()
        s = scales.double()[..., None]
        got = codes.double().view_as(yg) * s
        assert ((got - yg).abs() <= (2.0 ** -4 + 2e-5) * yg.abs() + (2.0 ** -10 + 1e-5) * s).all()
        again = rms_norm(x, w, residual=r, out_8bit=True, group=group)[0]  # without the updated residual
        assert torch.equal(again.view(torch.uint8), codes.view(torch.uint8))


def test_rms_norm_strides_and_in_place(cuda_device):
    torch = _torch()
    from ripvec_b200.decode import rms_norm

    for hidden, off in ((768, 8), (768, 3), (4096, 16), (1001, 1)):
        wide = torch.randn(9, 2 * hidden + 32, device="cuda").to(torch.bfloat16)
        x, r = wide[:, off:off + hidden], wide[:, off + hidden:off + 2 * hidden]
        w = torch.rand(hidden, device="cuda") + 0.5
        want, _ = rms_norm(x.clone(), w, residual=r.clone())
        h, _ = _norm_reference(x, r, w, 1e-5)
        buf = torch.full((9, hidden + 24), 3.0, dtype=torch.bfloat16, device="cuda")
        got, _ = rms_norm(x, w, residual=r, residual_out=r, out=buf[:, 8:8 + hidden])
        assert torch.equal(got, want) and (buf[:, :8] == 3).all() and (buf[:, 8 + hidden:] == 3).all()
        assert torch.equal(r, h.to(torch.bfloat16))
        one = torch.randn(1, hidden, device="cuda").to(torch.bfloat16)  # one row broadcast to all
        got, _ = rms_norm(x, w, residual=one.expand(9, hidden))
        assert torch.equal(got, rms_norm(x, w, residual=one.expand(9, hidden).contiguous())[0])


# ------------------------------------------------------------------ refusals
def test_refusals(cuda_device):
    torch = _torch()
    from ripvec_b200 import _lib as L
    from ripvec_b200.decode import DecodeStep, PagedCache, rms_norm

    for kw in (dict(q_heads=6, kv_heads=4), dict(head_dim=96), dict(page_size=8), dict(page_size=48), dict(q_heads=0)):
        with pytest.raises(L.RvError):
            DecodeStep(**{**dict(q_heads=8, kv_heads=2, head_dim=128, page_size=16), **kw})
    b = Batch(q=(2, 1), own=(10, 20), prefix=(40,), seed=24)
    cos = torch.ones(60, 64, device="cuda")

    def plan(**kw):
        b.step.plan(**{**dict(q_lens=[2, 1], own_lens=[10, 20], own_pages=b.own_pages, prefix_lens=[40],
                              prefix_pages=b.prefix_pages, num_pages=b.cache.num_pages), **kw})

    bad = [dict(own_pages=[[0], [1]]), dict(own_pages=[[0], [1, b.cache.num_pages]]), dict(q_lens=[2]),
           dict(q_lens=[2, -1]), dict(own_pages=[[0], [1, -2]]), dict(prefix_lens=[40, 3]),
           dict(group_sizes=[1]), dict(prefix_pages=[[0, 1, 99999]]), dict(num_pages=1), dict(q_lens=[1.5, 1])]
    for kw in bad:
        with pytest.raises((L.RvError, ValueError)):
            plan(**kw)
        with pytest.raises((L.RvError, ValueError)):  # a failed plan leaves none
            b.step.attend(b.cache, b.queries)
        with pytest.raises((L.RvError, ValueError)):
            b.step.attend(b.cache, b.queries[:0])
    plan()
    k = b.randn(3, 2, 128)
    for args, kw in (((b.queries[:2], k, k, cos, cos), {}), ((b.queries, k.float(), k, cos, cos), {}),
                     ((b.queries, k, k[:, :1], cos, cos), {}), ((b.queries, k, k, cos[:30], cos[:30]), {}),
                     ((b.queries, k, k, cos, cos[:, :32]), {}), ((b.queries, k, k, cos.half(), cos.half()), {}),
                     ((b.queries, k.cpu(), k, cos, cos), {}), ((None, k, k, cos, cos), dict(q_out=b.queries))):
        with pytest.raises((L.RvError, ValueError)):
            b.step.append(b.cache, *args, **kw)
    shift = torch.zeros(3 * 8 * 128 + 8, dtype=b.queries.dtype, device="cuda")[1:3 * 8 * 128 + 1].view(3, 8, 128)
    for q, kw in ((b.queries[:1], {}), (b.queries.float(), {}), (shift, {}), (b.queries, dict(out=shift)),
                  (b.queries, dict(lse=torch.zeros(3, 7, device="cuda"))), (b.queries, dict(scale=0.0)),
                  (b.queries, dict(scale=-1.0)), (b.queries, dict(scale=math.inf)), (b.queries, dict(scale=math.nan))):
        with pytest.raises((L.RvError, ValueError)):
            b.step.attend(b.cache, q, **kw)
    with pytest.raises(L.RvError):  # fewer pages than the plan's
        b.step.attend(PagedCache(b.k[:1], b.v[:1]), b.queries)
    with pytest.raises((L.RvError, ValueError)):  # other head dim
        b.step.attend(PagedCache(b.k[..., :64], b.v[..., :64]), b.queries[..., :64].contiguous())
    # what cannot be appended can still be read
    for kw in (dict(own_lens=[1, 20], q_lens=[2, 1]), dict(own_pages=[[0], [1, 0]]),
               dict(own_pages=[[b.prefix_pages[0][0]], b.own_pages[1]])):
        plan(**kw)
        with pytest.raises(L.RvError):
            b.step.append(b.cache, b.queries, k, k, cos, cos)
        b.step.attend(b.cache, b.queries)
    for bad in ((b.k, b.v[:, :, :8]), (b.k.float(), b.v.float()), (b.k[0], b.v[0]), (b.k.cpu(), b.v.cpu()),
                (b.k, b.v.transpose(0, 1).contiguous().transpose(0, 1)), (b.k[..., ::2], b.v[..., ::2])):
        with pytest.raises(ValueError):
            PagedCache(*bad)
    x, w = torch.zeros(4, 256, dtype=torch.float16, device="cuda"), torch.ones(256, device="cuda")
    for args, kw in (((x.float(), w), {}), ((x, w.half()), {}), ((x, w[:5]), {}), ((x, w), dict(group=128)),
                     ((x, w), dict(out_8bit=True, group=100)), ((x, w), dict(residual=x[:2])), ((x, w), dict(eps=-1.0)),
                     ((x, w), dict(out_8bit=True, out=x)), ((x, w), dict(scales=w)), ((x[:, ::2], w[::2].contiguous()), {}),
                     ((x, w), dict(out=x[:1].expand(4, 256)))):
        with pytest.raises((L.RvError, ValueError)):
            rms_norm(*args, **kw)
    torch.cuda.synchronize()


def test_empty_calls(cuda_device):
    """No tokens, no sequences, no rows."""
    torch = _torch()
    from ripvec_b200.decode import rms_norm

    b = Batch(q=(0, 0), own=(5, 0), prefix=(9,), seed=25)
    assert b.step.attend(b.cache, b.queries).shape == (0, 8, 128)
    b.step.append(b.cache, b.queries, b.queries[:, :2], b.queries[:, :2], torch.ones(9, 64, device="cuda"), torch.ones(9, 64, device="cuda"))
    b.step.plan(q_lens=[], own_lens=[], own_pages=[], num_pages=3)
    assert b.step.attend(b.cache, b.queries).shape == (0, 8, 128)
    out, scales = rms_norm(torch.zeros(0, 256, dtype=torch.bfloat16, device="cuda"), torch.ones(256, device="cuda"), out_8bit=True)
    assert out.shape == (0, 256) and scales.shape == (0, 1)


# ------------------------------------------------------------------ together
def test_decoder_example(cuda_device):
    """The example decoder, a context read once and shared by answers that go on from it token by token, against
    the same network in f32 without a cache: cosine of every logits row at least 0.999, the bar of the encoder's
    embeddings in 16 bits."""
    import importlib.util
    from pathlib import Path

    torch = _torch()
    spec = importlib.util.spec_from_file_location("answer_over_context",
                                                  Path(__file__).resolve().parent.parent / "examples" / "answer_over_context.py")
    ex = importlib.util.module_from_spec(spec)
    import sys

    sys.modules[spec.name] = ex
    spec.loader.exec_module(ex)
    d = ex.Decoder(ex.DecoderSpec(pages=64), seed=3)
    s = d.spec
    g = torch.Generator(device="cuda").manual_seed(4)
    context = torch.randint(0, s.vocab, (300,), generator=g, device="cuda")
    answers = torch.randint(0, s.vocab, (5, 9), generator=g, device="cuda")

    def plain(ids):
        n = len(ids)
        x = d.embedding[ids].float()
        norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s.eps) * w  # noqa: E731
        see = torch.ones(n, n, device="cuda", dtype=torch.bool).tril()

        def turn(x):
            a, b = x.chunk(2, -1)
            c, si = d.cos[:n, None], d.sin[:n, None]
            return torch.cat((a * c - b * si, b * c + a * si), -1)

        for l in d.layers:
            q, k, v = (norm(x, l["norm1"]) @ l["qkv"].float().T).view(n, -1, s.head_dim).split((s.q_heads, s.kv_heads, s.kv_heads), 1)
            q, k = turn(q), turn(k)
            k, v = (y.repeat_interleave(s.q_heads // s.kv_heads, 1) for y in (k, v))
            p = (torch.einsum("ihd,jhd->hij", q, k) * s.head_dim ** -0.5).masked_fill(~see, -math.inf).softmax(-1)
            x = x + torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ l["o"].float().T
            gate, up = (norm(x, l["norm2"]) @ l["up"].float().T).chunk(2, -1)
            x = x + (torch.nn.functional.silu(gate) * up) @ l["down"].float().T
        return norm(x, d.norm) @ d.embedding.float().T

    want = torch.stack([plain(torch.cat((context, a)))[len(context):] for a in answers])
    read = d.read(context)
    pages = [d.take_pages(answers.shape[1]) for _ in answers]
    got, own = [], 0
    for new in (4, 1, 1, 1, 2):  # a prompt, single tokens, two at once
        ids = answers[:, own:own + new].reshape(-1)
        own += new
        d.step.plan(q_lens=[new] * 5, own_lens=[own] * 5, own_pages=pages, prefix_lens=[read["length"]],
                    prefix_pages=[read["pages"]], num_pages=s.pages)
        got.append(d.forward(ids).float().view(5, new, -1))
    got = torch.cat(got, 1)
    cos = torch.nn.functional.cosine_similarity(got.double(), want.double(), dim=-1)
    assert cos.min().item() >= 0.999, cos.min().item()
    out = d.answer(read, [a[:n] for a, n in zip(answers, (4, 1, 9, 2, 3))], 6)
    assert out.shape == (5, 6) and out.min() >= 0 and out.max() < s.vocab


def test_waits_that_run_out_are_reported(cuda_device):
    """The bounded-wait exits of both attention kernels: with the first signal of every CTA withheld and waits of
    about a millisecond, the launch ends, the step's next call reports it, and the one after is right again."""
    torch = _torch()
    from ripvec_b200 import _lib as L

    lib = L.lib()
    for kw in (dict(q=(1, 2), own=(300, 40), prefix=(0,)),            # few-row kernel
               dict(q=(200,), own=(260,), prefix=(300,)),             # tensor-core kernel
               dict(q=(1,) * 40, own=(70,) * 40, prefix=(900,))):     # both, and the join
        b = Batch(seed=26, **kw)
        b.check()
        assert lib.rv_debug_stall_attention(1, 2_000_000) == L.RV_OK
        try:
            b.step.attend(b.cache, b.queries)
            torch.cuda.synchronize()
        finally:
            lib.rv_debug_stall_attention(0, 0)
        with pytest.raises(L.RvError) as e:
            b.step.attend(b.cache, b.queries)
        assert e.value.code == L.RV_E_DEVICE
        b.check()


def test_long_forms_and_records_agree(cuda_device):
    """The C entries with one argument each give the bits of those with a record, which Python calls."""
    torch = _torch()
    from ripvec_b200 import _lib as L
    from ripvec_b200.decode import rms_norm

    b = Batch(q=[3, 1, 20], own=[9, 40, 20], prefix=[100], seed=5)
    lib, st = L.lib(), torch.cuda.current_stream().cuda_stream
    cos, sin = (torch.randn(200, 32, generator=b.gen, device="cuda") for _ in range(2))
    k, v = b.randn(b.t, b.hkv, b.d), b.randn(b.t, b.hkv, b.d)

    def at(t):
        return t.data_ptr(), t.stride(0), t.stride(1)

    turned = b.step.append(b.cache, b.queries, k, v, cos, sin, interleaved=True)
    pools = b.k.clone(), b.v.clone()
    b.k.fill_(0)
    b.v.fill_(0)
    again = torch.empty_like(turned)
    assert lib.rv_step_append(b.step._h, b.cache._ref, *at(b.queries), *at(k), *at(v), *at(again), cos.data_ptr(),
                              sin.data_ptr(), 200, 64, 1, st) == L.RV_OK
    assert torch.equal(turned, again)
    for pool, want in zip((b.k, b.v), pools):
        written = pool != 0
        assert written.any() and torch.equal(pool[written], want[written])
        pool.copy_(want)
    out = b.step.attend(b.cache, turned, scale=0.1)
    again = torch.empty_like(out)
    assert lib.rv_step_attend(b.step._h, b.cache._ref, *at(turned), *at(again), None, 0.1, st) == L.RV_OK
    assert torch.equal(out, again)
    x, w = b.randn(5, 256), torch.rand(256, generator=b.gen, device="cuda")
    y, scales = rms_norm(x, w, out_8bit=True, group=64)
    y2, s2 = torch.empty_like(y), torch.empty_like(scales)
    assert lib.rv_rms_norm(L.RV_DTYPE_BF16, x.data_ptr(), 256, None, 0, w.data_ptr(), None, 0, y2.data_ptr(), 256,
                           L.RV_DTYPE_E4M3, s2.data_ptr(), 64, 5, 256, 1e-5, st) == L.RV_OK
    assert torch.equal(y.view(torch.uint8), y2.view(torch.uint8)) and torch.equal(scales, s2)
