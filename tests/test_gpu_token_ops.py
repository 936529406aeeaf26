"""The token operators on the GPU against plain 64-bit implementations.

Tolerances come from the roundings, u = eps / 2 of the tensors' type:
- rotary: the output's own rounding u |y|, and (|a| + |b|) 2^-21 for sine and cosine of a
  fraction rounded to 32 bits (2 pi 2^-26), their own error (2^-23) and two products and a sum;
- attention: the output's rounding u |o|; weights rounded to the type before they meet the
  values, u max|v|; scores in 32 bits, off by at most e = 2^-20 (1 + the largest sum of
  |q k| scale and of the bias's terms), which moves the weighted mean by 2 e max|v|; and in
  fp16 weights below 2^-14, off by 2^-25 each with the largest weight at least 1.
"""
import importlib
import math

import pytest

from s2s_testlib import pkg

pytestmark = pytest.mark.gpu

try:
    import torch
except ImportError:  # collected without torch: the GPU run has it
    torch = None

HALVES = ["float16", "bfloat16"]


def binding():
    pkg()
    return importlib.import_module("swin2sr_b200.capi")


def unit(dtype):
    return torch.finfo(getattr(torch, dtype)).eps / 2


def heads(x):
    return binding().heads(x.data_ptr(), x.stride(0), x.stride(1), x.shape[1])


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------- rotary
def rotary_reference(plan, x, pos, inverse):
    """64 bits, on the CPU: (y, |a| + |b| of each value's pair)."""
    x = x.double()
    P = plan.pairs
    f = torch.tensor(list(plan.frequency[:P]), dtype=torch.float64)
    t = pos.double()[list(plan.axis[:P])].T * f * (-1 if inverse else 1)
    c, s = t.cos()[:, None], t.sin()[:, None]
    one = torch.arange(P) * 2 if plan.interleaved else torch.arange(P)
    other = one + 1 if plan.interleaved else one + P
    y, size = x.clone(), torch.zeros_like(x)
    a, b = x[..., one], x[..., other]
    y[..., one], y[..., other] = a * c - b * s, a * s + b * c
    size[..., one] = size[..., other] = a.abs() + b.abs()
    return y, size


def run_rotary(plan, dtype, tensors, pos, inverse=False, stream=None):
    C = binding()
    x = tensors[0][0]
    C.rotary(plan, dtype, x.shape[2], x.shape[0], pos.data_ptr(), pos.stride(0),
             [(heads(a), heads(b)) for a, b in tensors], inverse,
             (stream or torch.cuda.current_stream()).cuda_stream)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("tokens,qh,kh,dim,sections,interleaved,per_axis", [
    (1, 4, 2, 128, [64], False, False), (7, 6, 6, 32, [8, 8], False, True),
    (1000, 3, 1, 128, [16, 24, 24], False, False), (33, 2, 1, 80, [5, 7, 8], True, False),
    (33, 2, 1, 80, [5, 7, 8], False, False), (19, 1, 1, 256, [128], False, False),
    (5000, 5, 2, 64, [16, 16], True, True), (3, 1, 3, 31, [3], False, False),
    (3, 1, 3, 31, [3, 0, 4], True, False), (2500, 1, 1, 2, [1], False, False)])
def test_rotary(dtype, tokens, qh, kh, dim, sections, interleaved, per_axis):
    C = binding()
    plan = C.rotary_plan(sections, 10000.0, per_axis, interleaved)
    g = gen(tokens + dim)
    q = torch.randn(tokens, qh, dim, generator=g).to(getattr(torch, dtype))
    k = torch.randn(tokens, kh, dim, generator=g).to(getattr(torch, dtype))
    pos = torch.randint(-50, 5000000, (len(sections), tokens), generator=g, dtype=torch.int32)
    dq, dk, dpos = q.cuda(), k.cuda(), pos.cuda()
    for inverse in (False, True):
        yq, yk = torch.full_like(dq, 9.0), torch.full_like(dk, 9.0)
        run_rotary(plan, dtype, [(dq, yq), (dk, yk)], dpos, inverse)
        for x, y in ((q, yq), (k, yk)):
            want, size = rotary_reference(plan, x, pos, inverse)
            off = (y.cpu().double() - want).abs()
            assert (off <= unit(dtype) * want.abs() + size * 2.0 ** -21 + 1e-7 * (dtype == "float16")).all()
            assert torch.equal(y.cpu()[..., 2 * plan.pairs:], x[..., 2 * plan.pairs:])
    # in place: the same bits
    run_rotary(plan, dtype, [(dq, dq), (dk, dk)], dpos, True)
    assert torch.equal(dq, yq) and torch.equal(dk, yk)


def test_rotary_strides_far_positions_and_neighbours():
    """q and k as parts of one row per token, odd strides, positions at both ends of 32 bits;
    what lies between the rows stays as it was."""
    C = binding()
    plan = C.rotary_plan([8, 8])
    g = gen(3)
    for width in (3 * 4 * 32, 3 * 4 * 32 + 5):  # wide accesses, and a stride that allows none
        rows = torch.randn(40, width, generator=g).half()
        pos = torch.tensor([[-2 ** 31, 2 ** 31 - 1, 0, 1], [7, -9, 2 ** 30, -2 ** 30]],
                           dtype=torch.int32).repeat(1, 10).contiguous()
        d = rows.cuda()
        view = lambda r, part: r[:, :384].view(40, 4, 3, 32)[:, :, part] if width == 384 else \
            torch.as_strided(r, (40, 4, 32), (width, 96, 1), part * 32)  # noqa: E731
        run_rotary(plan, "float16", [(view(d, 0), view(d, 0)), (view(d, 1), view(d, 1))], pos.cuda())
        want = rows.clone().double()
        tol = torch.zeros_like(want)
        for part in (0, 1):
            y, size = rotary_reference(plan, view(rows, part), pos, False)
            view(want, part).copy_(y)
            # at 2^31 radians 53 bits leave 2^-21 of one in the turn count (two roundings) and
            # 2^-22 in the reference's angle: 2^-19 with the 2^-21 of the rest
            view(tol, part).copy_(unit("float16") * y.abs() + size * 2.0 ** -19 + 1e-7)
        assert ((d.cpu().double() - want).abs() <= tol).all()
        assert torch.equal(d.cpu()[:, 64:96], rows[:, 64:96])


def test_rotary_four_tensors_and_a_plan_by_hand():
    C = binding()
    plan = C.rotary_plan([4, 4])
    for p in range(8):
        plan.axis[p] = p % 2
        plan.frequency[p] = 0.3 * (p + 1)
    g = gen(5)
    xs = [torch.randn(21, h, 16, generator=g) for h in (1, 2, 3, 5)]
    pos = torch.randint(0, 1000, (2, 30), generator=g, dtype=torch.int32)
    dev = [x.cuda() for x in xs]
    out = [torch.empty_like(d) for d in dev]
    run_rotary(plan, "float32", list(zip(dev, out)), pos.cuda()[:, :21])
    for x, y in zip(xs, out):
        want, size = rotary_reference(plan, x, pos[:, :21], False)
        assert ((y.cpu().double() - want).abs() <= unit("float32") * want.abs() + size * 2.0 ** -21).all()


def test_rotary_inverse_is_the_gradient():
    """<turn(x), w> has the gradient turn back(w), also by differences of the 64-bit form."""
    C = binding()
    plan = C.rotary_plan([3, 5], interleaved=True)
    g = gen(8)
    x, w = torch.randn(2, 6, 2, 16, generator=g).unbind(0)
    pos = torch.randint(0, 99, (2, 6), generator=g, dtype=torch.int32)
    d, y = w.cuda(), torch.empty_like(w, device="cuda")
    run_rotary(plan, "float32", [(d, y)], pos.cuda(), True)
    step, got = 1e-4, y.cpu().double()
    for at in ((0, 0, 0), (3, 1, 7), (5, 0, 15)):
        e = torch.zeros_like(x, dtype=torch.float64)
        e[at] = step
        up, down = ((rotary_reference(plan, x.double() + s * e, pos, False)[0] * w).sum() for s in (1, -1))
        assert abs((up - down) / (2 * step) - got[at]) <= 1e-5


# ---------------------------------------------------------------------------- attention
@pytest.fixture(params=["mma", "tcgen05"])
def kernel(request, monkeypatch):
    """Each of the two attention kernels, whatever the sizes would choose."""
    monkeypatch.setenv("S2S_MASKED_ATTN", request.param)
    return request.param


class Problem:
    """Tensors of one call on the CPU, and what the definition says in 64 bits."""

    def __init__(self, dtype, dim, qh, kh, q_lens, kv_lens, causal=False, prefix=None, cap=0.0, axes=0,
                 seed=0, scale=None, sharp=1.5, far=0, tail=(0, 0), span=60):
        g = gen(seed + 100 * dim + len(q_lens))
        self.dtype, self.causal, self.prefix, self.cap, self.axes = dtype, causal, prefix, cap, axes
        self.q_lens, self.kv_lens = q_lens, kv_lens
        self.scale = dim ** -0.5 if scale is None else scale
        tq, tk = sum(q_lens) + tail[0], sum(kv_lens) + tail[1]
        t = getattr(torch, dtype)
        self.q = (sharp * torch.randn(tq, qh, dim, generator=g)).to(t)
        self.k = torch.randn(tk, kh, dim, generator=g).to(t)
        self.v = (torch.randn(tk, kh, dim, generator=g) + torch.randn(kh, dim, generator=g)).to(t)
        if axes:
            self.q_pos = (torch.randint(0, span, (axes, tq), generator=g) + far).to(torch.int32)
            self.kv_pos = (torch.randint(0, span, (axes, tk), generator=g) + far).to(torch.int32)
            self.slopes = torch.rand(axes, qh, generator=g) * torch.tensor([1.0, -0.3, 0.01])[:axes, None]

    def expected(self):
        """out, lse, and the bound on |out - got| and |lse - got| (NaN where no document is)."""
        u, nan = unit(self.dtype), float("nan")
        qh, group = self.q.shape[1], self.q.shape[1] // self.k.shape[1]
        out = torch.full(self.q.shape, nan, dtype=torch.float64)
        tol = torch.full(self.q.shape, nan, dtype=torch.float64)
        lse = torch.full((qh, self.q.shape[0]), nan, dtype=torch.float64)
        ltol = torch.full((qh, self.q.shape[0]), nan, dtype=torch.float64)
        a = b = 0
        for d, (nq, nk) in enumerate(zip(self.q_lens, self.kv_lens)):
            i, j = torch.arange(nq)[:, None], torch.arange(nk)[None]
            see = torch.ones(nq, nk, dtype=torch.bool)
            if self.causal:
                see = (j <= i + nk - nq) | (j < (self.prefix[d] if self.prefix else 0))
            for h in range(qh):
                q, k = self.q[a:a + nq, h].double(), self.k[b:b + nk, h // group].double()
                v = self.v[b:b + nk, h // group].double()
                z = q @ k.T * self.scale
                size = (q.abs() @ k.abs().T * self.scale)
                if self.cap:
                    z = self.cap * torch.tanh(z / self.cap)
                for x in range(self.axes):
                    far = (self.q_pos[x, a:a + nq, None].double() - self.kv_pos[x, None, b:b + nk].double()).abs()
                    z = z - self.slopes[x, h].double().abs() * far
                    size = size + self.slopes[x, h].abs() * far.max() if nk and nq else size
                z = torch.where(see, z, -math.inf)
                w = torch.logsumexp(z, 1)
                p = torch.where(see, torch.exp(z - w[:, None].clamp(min=-1e300)), 0.0)
                lse[h, a:a + nq] = w
                o = p @ torch.where(see.any(0)[:, None], v, 0.0)  # keys that no row sees may hold anything
                e = 2.0 ** -20 * (1 + torch.where(see, size, 0.0).amax(1)) if nk else torch.zeros(nq)
                big = torch.where(see.any(0)[:, None], v, 0.0).abs().max() if nk else 0.0
                out[a:a + nq, h] = o
                tiny = nk * 2.0 ** -25 if self.dtype == "float16" else 0.0
                tol[a:a + nq, h] = u * o.abs() + ((u + 2 * e + tiny) * big)[:, None]
                ltol[h, a:a + nq] = e + 2.0 ** -20
            a, b = a + nq, b + nk
        return out, lse, tol, ltol

    def run(self, q=None, k=None, v=None, offsets=True, stream=None, lse=True, out=None):
        C = binding()
        self.keep = keep = {n: x.cuda() for n, x in (("q", self.q), ("k", self.k), ("v", self.v))}
        q, k, v = (keep[n] if x is None else x for n, x in (("q", q), ("k", k), ("v", v)))
        out = torch.full(self.q.shape, 7.0, device="cuda", dtype=self.q.dtype) if out is None else out
        sums = torch.full((self.q.shape[1], self.q.shape[0]), 7.0, device="cuda") if lse else None

        def ints(x):
            return torch.tensor(x, dtype=torch.int32, device="cuda")

        more = {}
        if offsets:
            keep["qo"] = ints([sum(self.q_lens[:i]) for i in range(len(self.q_lens) + 1)])
            keep["ko"] = ints([sum(self.kv_lens[:i]) for i in range(len(self.kv_lens) + 1)])
            more.update(d_q_offsets=keep["qo"].data_ptr(), d_kv_offsets=keep["ko"].data_ptr())
        if self.prefix:
            keep["prefix"] = ints(self.prefix)
            more.update(d_prefix=keep["prefix"].data_ptr())
        if self.axes:
            for n in ("slopes", "q_pos", "kv_pos"):
                keep[n] = getattr(self, n).cuda()
                more["d_" + n] = keep[n].data_ptr()
        self.call = lambda stream: C.attention(
            self.dtype, self.q.shape[2], self.scale, heads(q), heads(k), heads(v), heads(out),
            self.q.shape[0], self.k.shape[0], len(self.q_lens), causal=self.causal, cap=self.cap,
            axes=self.axes, d_lse=sums.data_ptr() if lse else 0, stream=stream, **more)
        torch.cuda.synchronize()
        self.call((stream or torch.cuda.current_stream()).cuda_stream)
        return out, sums

    def check(self, out, lse=None, want=None):
        o, w, tol, ltol = want or self.expected()
        here = ~o.isnan()
        got = out.cpu().double()
        assert ((got - o).abs()[here] <= tol[here]).all(), float(((got - o).abs()[here] / tol[here]).max())
        assert (got[~here] == 7.0).all(), "rows of no document were written"
        if lse is not None:
            here, got = ~w.isnan(), lse.cpu().double()
            empty = w == -math.inf
            assert (got[empty] == -math.inf).all()
            assert (out.cpu().transpose(0, 1)[empty] == 0).all()
            at = here & ~empty
            assert ((got - w).abs()[at] <= ltol[at]).all()
            assert (got[~here] == 7.0).all()


ODD = [1, 0, 17, 64, 65, 128, 129, 255, 0, 300, 2]
CASES = {
    "one": (64, 2, 2, [1], [1], {}),
    "odd": (64, 2, 1, ODD, ODD, {}),
    "odd-causal": (128, 4, 2, ODD, ODD, dict(causal=True)),
    "odd-causal-bias": (32, 3, 3, ODD, ODD, dict(causal=True, axes=2)),
    "prefix": (64, 2, 2, ODD, ODD, dict(causal=True, prefix=[1, 0, 5, 70, 0, 128, 60, 1, 3, 200, -4])),
    "prefix-cap": (128, 8, 1, [40, 333, 7], [40, 333, 7], dict(causal=True, prefix=[3, 200, 7], cap=5.0)),
    "more-keys": (64, 2, 2, [5, 130, 33], [70, 700, 33], dict(causal=True, axes=1)),
    "more-queries": (64, 2, 2, [9, 200, 64, 300], [4, 30, 0, 290], dict(causal=True)),
    "no-keys": (64, 2, 2, [3, 5], [0, 0], {}),
    "some-keys": (64, 2, 1, [3, 5, 140], [0, 7, 0], dict(cap=2.0)),
    "dim8": (8, 2, 2, [100, 200], [100, 200], dict(axes=3)),
    "dim24": (24, 6, 3, [130], [257], {}),
    "dim40": (40, 2, 2, [65, 300], [65, 300], dict(causal=True, cap=30.0)),
    "dim80": (80, 2, 1, [400], [400], dict(axes=1)),
    "dim120": (120, 2, 2, [129], [1000], dict(cap=50.0)),
    "windows": (32, 6, 6, [64] * 30, [64] * 30, dict(axes=2)),
    "windows-odd": (32, 3, 3, [49] * 20, [49] * 20, {}),
    "single": (128, 8, 2, [1] * 6, [1, 100, 0, 1000, 5000, 64], dict(causal=True)),
    "single-cap": (64, 8, 8, [1] * 4, [3000, 2, 77, 129], dict(causal=True, cap=20.0, axes=1)),
    "single-one": (64, 4, 4, [1], [613], dict(causal=True)),
    "group40": (64, 40, 1, [2, 1], [300, 900], dict(causal=True)),
    "few": (128, 16, 2, [5], [6001], dict(causal=True, axes=1)),
    "few-prefix": (64, 4, 2, [30, 3], [20, 4000], dict(causal=True, prefix=[20, 4000])),
    "long": (128, 2, 1, [1500], [1500], dict(causal=True)),
    "long-cap-bias": (64, 2, 2, [1111, 600], [1111, 900], dict(causal=True, cap=30.0, axes=3, prefix=[100, 900])),
    "long-keys": (64, 1, 1, [300], [5000], {}),
    "sharp": (64, 2, 2, [700], [700], dict(causal=True, sharp=40.0)),
    "far-positions": (64, 2, 2, [300], [300], dict(axes=2, far=2 ** 31 - 100)),
}


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("name", list(CASES))
def test_attention(name, dtype, kernel):
    dim, qh, kh, q, kv, more = CASES[name]
    P = Problem(dtype, dim, qh, kh, q, kv, **more)
    out, lse = P.run()
    P.check(out, lse)
    again, _ = P.run(lse=False)  # the same bits, with and without the sums
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim,heads,q,kv,more", [
    (64, 8, [700, 1, 1500], [700, 1, 1500], dict(causal=True)),
    (128, 8, [900, 300], [1300, 300], dict(causal=True, cap=50.0, prefix=[700, 0])),
    (32, 10, [1000, 1000], [1000, 1100], dict(axes=2)),
    (128, 6, [1500], [1500], dict(causal=True, axes=1, sharp=6.0))])
def test_attention_of_the_size_for_the_large_kernel(dim, heads, q, kv, more, dtype):
    """Sizes for which the library chooses its tcgen05 kernel by itself."""
    P = Problem(dtype, dim, heads, heads // 2, q, kv, **more)
    P.check(*P.run())


@pytest.mark.parametrize("name", ["odd-causal", "windows", "single", "long", "long-cap-bias"])
def test_attention_masked_values_may_be_anything(name, kernel):
    """NaN and infinities behind the last document and at keys that a row does not see."""
    dim, qh, kh, q, kv, more = CASES[name]
    P = Problem("float16", dim, qh, kh, q, kv, tail=(3, 150), **more)
    end = sum(kv)
    want = P.expected()
    P.k[end:], P.v[end:] = float("nan"), float("inf")
    P.check(*P.run(), want=want)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n", [20, 300, 900])
def test_attention_hidden_values_of_the_own_document(n, dtype, kernel):
    """A NaN value in the middle of a causal document reaches the rows that see it, no other."""
    P = Problem(dtype, 64, 4, 2, [n], [n], causal=True)
    want = P.expected()
    bad = n // 2
    P.v[bad, 1, 5] = float("nan")
    P.v[bad + 3, 0, 0] = float("inf")
    out, lse = P.run()
    got = out.cpu()
    assert got[bad:, 2:, 5].isnan().all() and not got[:bad, 2:].isnan().any()
    assert (got[bad + 3:, :2, 0] == math.inf).all()
    assert ((got[:bad].double() - want[0][:bad]).abs() <= want[2][:bad]).all()
    clean = [c for c in range(64) if c not in (0, 5)]
    assert ((got[..., clean].double() - want[0][..., clean]).abs() <= want[2][..., clean]).all()
    here = (lse.cpu().double() - want[1]).abs() <= want[3]
    assert here.all()


@pytest.mark.parametrize("what", ["all", "channel", "first", "query"])
def test_attention_values_that_are_nan_for_good(what, kernel):
    """NaN wherever the definition has it and nowhere else, at the size where a row done again
    key after key would show in the time: all values, one channel, the first key, one query."""
    n = 3000
    P = Problem("bfloat16", 64, 4, 2, [n], [n], causal=True)
    want = P.expected()
    if what == "all":
        P.v[:] = float("nan")
    elif what == "channel":
        P.v[:, :, 7] = float("nan")
    elif what == "first":
        P.v[0] = float("nan")
    else:
        P.q[100] = float("nan")
    out, lse = P.run()
    got = out.cpu().double()
    nan = torch.zeros(n, 4, 64, dtype=torch.bool)
    if what in ("all", "first"):
        nan[:] = True
    elif what == "channel":
        nan[..., 7] = True
    else:
        nan[100] = True
    assert torch.equal(got.isnan(), nan)
    assert ((got - want[0]).abs() <= want[2])[~nan].all()
    rows = torch.arange(n) != (100 if what == "query" else -1)
    assert ((lse.cpu().double() - want[1]).abs() <= want[3])[:, rows].all()


@pytest.mark.parametrize("name", ["windows", "odd-causal", "single", "long"])
def test_attention_strides(name, kernel):
    """q, k, v as parts of one row per token and head, as [head][token] planes, and as rows
    with gaps; outputs into a plane, their neighbours untouched."""
    dim, qh, kh, q, kv, more = CASES[name]
    P = Problem("bfloat16", dim, qh, kh, q, kv, **more)
    plain, sums = P.run()
    t = P.q.dtype

    def plane(x):
        return x.cuda().transpose(0, 1).contiguous().transpose(0, 1)

    out = torch.full((qh, P.q.shape[0], dim), 7.0, device="cuda", dtype=t).transpose(0, 1)
    got, s = P.run(plane(P.q), plane(P.k), plane(P.v), out=out)
    assert torch.equal(got, plain) and torch.equal(s, sums)

    def gaps(x):
        wide = torch.full((x.shape[0], x.shape[1] + 1, dim + 24), float("nan"), device="cuda", dtype=t)
        wide[:, 1:, 8:8 + dim] = x.cuda()
        return wide, wide[:, 1:, 8:8 + dim]

    wide, out = gaps(torch.full_like(P.q, 7.0))
    got, s = P.run(gaps(P.q)[1], gaps(P.k)[1], gaps(P.v)[1], out=out)
    assert torch.equal(got, plain) and torch.equal(s, sums)
    assert wide[:, 0].isnan().all() and wide[..., :8].isnan().all() and wide[..., 8 + dim:].isnan().all()


def test_attention_on_the_library_qkv_rows(kernel):
    """The rows [token][head][q|k|v][dp] that the forward's QKV product writes."""
    P = Problem("float16", 32, 6, 6, [64] * 12, [64] * 12, axes=2)
    plain, _ = P.run()
    rows = torch.stack([P.q, P.k, P.v], 2).cuda()
    q, k, v = rows.unbind(2)
    got, _ = P.run(q, k, v)
    assert torch.equal(got, plain)


@pytest.mark.parametrize("q,kv,n", [(64, 64, 9), (1, 700, 5), (300, 310, 3), (20, 20, 1)])
def test_attention_documents_of_equal_length_need_no_offsets(q, kv, n, kernel):
    P = Problem("bfloat16", 64, 4, 2, [q] * n, [kv] * n, causal=True)
    with_offsets = P.run()
    without = P.run(offsets=False)
    P.check(*without)
    for a, b in zip(with_offsets, without):
        assert torch.equal(a, b)


@pytest.mark.parametrize("q,kv", [([70, 30], [70, 30]), ([1, 1], [300, 80]), ([600, 300], [600, 300])])
def test_attention_leaves_rows_behind_the_documents(q, kv, kernel):
    P = Problem("float16", 64, 2, 2, q, kv, tail=(90, 0))
    P.check(*P.run())


def test_attention_offsets_outside_the_tokens_stay_inside(kernel):
    """Offsets past the tokens, negative and falling ones: results mean nothing, but nothing
    outside the outputs is written."""
    C = binding()
    P = Problem("float16", 64, 2, 2, [40, 60], [40, 60], causal=True, axes=1)
    for off in ([0, 40, 1 << 30], [-5, 200, 100], [90, 10, 100], [2 ** 31 - 1, -2 ** 31, 0]):
        wide = torch.full((300, 2, 64), 7.0, device="cuda", dtype=torch.float16)
        P.run(out=wide[100:200])
        o = torch.tensor(off, dtype=torch.int32, device="cuda")
        P.keep["qo"].copy_(o)
        P.keep["ko"].copy_(o)
        P.call(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert (wide[:100] == 7).all() and (wide[200:] == 7).all()
    C.device_status(0)


@pytest.mark.parametrize("name", ["windows", "odd-causal-bias", "few", "long-cap-bias"])
def test_attention_in_streams_and_graphs(name, kernel):
    """Another stream; two calls at once; captured, replayed on changed inputs."""
    dim, qh, kh, q, kv, more = CASES[name]
    P, R = (Problem("bfloat16", dim, qh, kh, q, kv, seed=s, **more) for s in (0, 1))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    want, _ = P.run()
    other, _ = R.run()
    for _ in range(3):
        with torch.cuda.stream(a):
            x, _ = P.run(stream=a)
        with torch.cuda.stream(b):
            y, _ = R.run(stream=b)
        torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(y, other)
    out, _ = P.run(stream=a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=a):
        P.call(a.cuda_stream)
    for n in ("q", "k", "v") + (("slopes", "q_pos", "kv_pos") if P.axes else ()):
        P.keep[n].copy_(getattr(R, n))
    out.fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, other)


def test_a_refused_device_leaves_no_error_behind():
    C = binding()
    with pytest.raises(C.S2SError):
        C.device_status(99)
    x = torch.ones(4, device="cuda") + 1  # looks at the last error after its launch
    assert x.sum().item() == 8


def test_host_memory_is_refused():
    C = binding()
    P = Problem("float16", 64, 2, 2, [4], [4])
    with pytest.raises(C.S2SError, match="not device memory"):
        P.run(q=P.q)
    plan = C.rotary_plan([4])
    with pytest.raises(C.S2SError, match="not device memory"):
        run_rotary(plan, "float16", [(P.q, P.keep["q"])], torch.zeros(1, 4, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim,axes", [(32, 2), (64, 1), (64, 3), (128, 1), (128, 3)])
def test_attention_positions_far_apart_in_a_tile(dtype, dim, axes, kernel):
    """Neighbouring queries anywhere in 2^23, a key at each one's place and one beside it: distances
    are exact whatever the others' are. Tolerance: differences of positions below 2^24 are exact in 32
    bits, so a bias is off by 2^-23 of itself, and those that count (0 and a few slopes) are below 4;
    the products as in Problem; one rounding of the weights and one of the output."""
    n, g = 200, gen(dim + axes)
    P = Problem(dtype, dim, 2, 2, [n, n], [2 * n, 2 * n], axes=axes)
    P.slopes = 0.5 + torch.rand(axes, 2, generator=g)
    place = torch.randint(-2 ** 22, 2 ** 22, (axes, 2, n), generator=g)
    step = torch.randint(0, 2, (axes, 2, n), generator=g)
    P.q_pos = place.flatten(1).to(torch.int32)
    P.kv_pos = torch.cat([place, place + step], 2).flatten(1).to(torch.int32)
    out, lse, _, _ = P.expected()
    got, sums = P.run()
    size = (P.q.abs().double().amax((0, 1)) @ P.k.abs().double().amax((0, 1))) * P.scale
    e, u = 2.0 ** -20 * (1 + size + 4), unit(dtype)
    tiny = 2 * n * 2.0 ** -25 if dtype == "float16" else 0.0
    tol = u * out.abs() + (u + 2 * e + tiny) * P.v.abs().max()
    assert ((got.cpu().double() - out).abs() <= tol).all()
    assert ((sums.cpu().double() - lse).abs() <= e + 2.0 ** -20).all()


# ----------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", HALVES)
def test_rotary_then_attention(dtype, kernel):
    """Frames of two clips: q and k turned along time, height and width, then attended with
    the same positions for the bias, a prefix of each clip seen whole; one stream, and the
    whole run replayed as a graph."""
    C = binding()
    frames, rows, cols = [3, 5], 6, 7
    lens = [f * rows * cols for f in frames]
    pos = torch.cat([torch.stack(torch.meshgrid(torch.arange(f), torch.arange(rows), torch.arange(cols),
                                                indexing="ij")).flatten(1) for f in frames], 1).to(torch.int32)
    P = Problem(dtype, 64, 4, 2, lens, lens, causal=True, prefix=[42, 84], axes=3, cap=30.0)
    P.q_pos = P.kv_pos = pos
    plan = C.rotary_plan([8, 12, 12], per_axis=True)
    raw_q, raw_k = P.q, P.k
    turned_q, size_q = rotary_reference(plan, raw_q, pos, False)
    turned_k, size_k = rotary_reference(plan, raw_k, pos, False)
    dq, dk = raw_q.cuda(), raw_k.cuda()
    tq, tk = torch.empty_like(dq), torch.empty_like(dk)
    s = torch.cuda.Stream()
    dpos = pos.cuda()
    torch.cuda.synchronize()
    run_rotary(plan, dtype, [(dq, tq), (dk, tk)], dpos, stream=s)
    out, lse = P.run(tq, tk, stream=s)
    torch.cuda.synchronize()
    u = unit(dtype)
    assert ((tq.cpu().double() - turned_q).abs() <= u * turned_q.abs() + size_q * 2.0 ** -21 + 1e-7).all()
    assert ((tk.cpu().double() - turned_k).abs() <= u * turned_k.abs() + size_k * 2.0 ** -21 + 1e-7).all()
    P.q, P.k = tq.cpu(), tk.cpu()  # what attention was given
    P.check(out, lse)
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        run_rotary(plan, dtype, [(dq, tq), (dk, tk)], dpos, stream=s)
        P.call(s.cuda_stream)
    tq.zero_()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    C.device_status(0)
