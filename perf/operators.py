"""The attention operators over packed documents and their rotary positions, as measured work.

Two operators of the library on device tensors, each in a plain form (elementary torch
operations) and through the library's own calls (where `own` is true):

rotary     turns pairs of a head's values by angles that grow with a token's position along
           one of several axes (time, height, width);
attention  softmax attention over documents packed one behind another, with a cap on the
           scores, a bias that falls with the distance along the position axes, a causal
           mask and a prefix that every query sees.

A case names its lengths as text: "5,17,64x3" is documents of 5, 17, 64, 64 and 64 tokens.
"""
import importlib
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False  # true: run() makes the library's calls

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------ the cases
def attention_case(name, dtype, head_dim, heads, q, kv, causal=False, prefix="", cap=0.0, axes=0, grid=0, fused=False,
                   lse=False):
    """heads: "query heads/key heads"; grid: tokens in an image row (positions); fused: q, k and v are parts of one row
    per token, head by head; lse: the logarithm of each row's softmax sum is wanted too."""
    return {"name": name, "op": "attention", "dtype": dtype, "head_dim": head_dim, "heads": heads, "q": q, "kv": kv,
            "causal": causal, "prefix": prefix, "cap": cap, "axes": axes, "grid": grid, "fused": fused, "lse": lse}


def rotary_case(name, dtype, head_dim, heads, tokens, sections, start=0, interleaved=False, per_axis=False, grid=1,
                inverse=False):
    """sections: pairs of each position axis; start: the first token's position; per_axis: each axis has its own
    series of frequencies."""
    return {"name": name, "op": "rotary", "dtype": dtype, "head_dim": head_dim, "heads": heads, "tokens": tokens,
            "sections": sections, "start": start, "interleaved": interleaved, "per_axis": per_axis, "grid": grid,
            "inverse": inverse}


def listed():
    return [
        # the 31 x 41 windows of a padded 240 x 320 image, six heads of 30 in 32, biased by the distance in the window
        attention_case("windows", "float16", 32, "6/6", "64x1271", "64x1271", axes=2, grid=8, fused=True),
        # images of several sizes (56 x 56, 64 x 64, 40 x 48 and ragged ones) in one sequence, each on its own
        attention_case("images", "bfloat16", 64, "12/12", "3136,4096,1920,777,1,2501", "3136,4096,1920,777,1,2501", axes=2,
                       grid=56, fused=True),
        # one long sequence in order, queries sharing key heads
        attention_case("causal-long", "bfloat16", 128, "8/2", "16384", "16384", causal=True),
        # packed prompts behind prefixes that are seen whole, capped scores, and the sums that join shards
        attention_case("prefix-capped", "float16", 128, "16/4", "1531,2048,401,64,999", "1531,2048,401,64,999", causal=True,
                       prefix="300,0,401,10,500", cap=50.0, lse=True),
        # a few dozen rows over earlier frames: queries at the end of longer documents, three axes
        attention_case("frames", "bfloat16", 64, "16/8", "196,49,100", "6272,1813,900", causal=True, axes=3, grid=7, cap=30.0),
        # one new token of one short sequence: latency
        attention_case("single-small", "float16", 64, "8/8", "1", "613", causal=True),
        # one new token for each of 24 sequences of very different lengths
        attention_case("single-batch", "bfloat16", 128, "32/8", "1x24",
                       "8001,17,4096,12345,900,1,6000,2222,3333,5120,64,7777,9999,40,1500,10240,512,8192,311,2048,4444,7000,13000,1024",
                       causal=True, cap=50.0),
        # five tokens at the end of one long sequence, falling off with distance
        attention_case("few-long", "bfloat16", 128, "16/2", "5", "40001", causal=True, axes=1, lse=True),
        # two axes over the tokens of a padded 240 x 320 image, six heads of 32
        rotary_case("rotary-image", "float16", 32, "6/6", 81344, "8,8", grid=328, per_axis=True),
        # three axes over 16 frames of 56 x 56 tokens
        rotary_case("rotary-video", "bfloat16", 128, "16/4", 50176, "16,24,24", start=1000, grid=56),
        # one new token far along
        rotary_case("rotary-single", "bfloat16", 128, "32/8", 1, "64", start=123457),
        # a part of each head turned back, neighbouring pairs, 32 bits
        rotary_case("rotary-part", "float32", 80, "9/3", 4097, "5,7,8", start=77, grid=33, interleaved=True, inverse=True),
    ]


def log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["windows", "images", "causal", "prefix", "frames", "single", "few", "rotary", "rotary"])
    dtype = rng.choice(["float16", "bfloat16"])
    join = lambda v: ",".join(map(str, v))  # noqa: E731
    if kind == "rotary":
        dtype = rng.choice(["float16", "bfloat16", "float32"])
        dim = rng.choice([16, 32, 64, 80, 96, 128])
        pairs = rng.choice([dim // 2, dim // 2, dim // 4])
        axes = rng.randint(1, 3)
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4])
        most = max(2, 50176 * 128 * 20 // (dim * (heads + kv) * (2 if dtype == "float32" else 1)))
        case = rotary_case("", dtype, dim, "%d/%d" % (heads, kv), log_uniform(rng, 1, min(most, 100000)), join(sections),
                           start=log_uniform(rng, 1, 1000000), interleaved=rng.random() < 0.3, per_axis=rng.random() < 0.5,
                           grid=rng.randint(1, 400), inverse=rng.random() < 0.2)
    elif kind == "windows":
        side = rng.randint(4, 12)
        heads = rng.randint(1, 8)
        count = log_uniform(rng, 16, max(17, 81344 * 6 // (side * side * heads)))
        text = "%dx%d" % (side * side, count)
        case = attention_case("", dtype, rng.choice([16, 32, 32, 40, 64]), "%d/%d" % (heads, heads), text, text,
                              axes=rng.choice([0, 2]), grid=side, fused=rng.random() < 0.5)
    elif kind == "images":
        lens = [log_uniform(rng, 1, 4200) for _ in range(rng.randint(1, 7))]
        heads = rng.randint(2, 12)
        case = attention_case("", dtype, rng.choice([32, 48, 64, 96]), "%d/%d" % (heads, heads), join(lens), join(lens),
                              axes=rng.randint(0, 2), grid=rng.randint(8, 64), fused=rng.random() < 0.5, lse=rng.random() < 0.3)
    elif kind == "causal":
        n = log_uniform(rng, 300, 16000)
        kv = rng.choice([1, 2, 4])
        heads = kv * rng.choice([h for h in (1, 2, 4, 8) if h * kv <= 8])
        case = attention_case("", dtype, rng.choice([64, 80, 128]), "%d/%d" % (heads, kv), str(n), str(n), causal=True,
                              cap=rng.choice([0.0, 30.0]), axes=rng.randint(0, 1), lse=rng.random() < 0.3)
    elif kind == "prefix":
        lens = [log_uniform(rng, 1, 2300) for _ in range(rng.randint(1, 9))]
        kv = rng.choice([1, 2, 4])
        heads = kv * rng.choice([1, 2, 4])
        case = attention_case("", dtype, rng.choice([64, 128, 128]), "%d/%d" % (heads, kv), join(lens), join(lens), causal=True,
                              prefix=join([rng.randint(0, n) for n in lens]), cap=rng.choice([0.0, 20.0, 50.0]), lse=rng.random() < 0.5)
    elif kind == "frames":
        q = [log_uniform(rng, 17, 300) for _ in range(rng.randint(1, 5))]
        kv = rng.choice([2, 4, 8])
        case = attention_case("", dtype, rng.choice([32, 64, 128]), "%d/%d" % (kv * rng.choice([1, 2]), kv), join(q),
                              join([n * rng.randint(1, 30) for n in q]), causal=rng.random() < 0.7, axes=rng.randint(0, 3),
                              grid=rng.randint(3, 20), cap=rng.choice([0.0, 30.0]))
    else:
        count = 1 if kind == "few" else log_uniform(rng, 1, 32)
        q = [rng.randint(2, 16) if kind == "few" else 1 for _ in range(count)]
        k = [n + log_uniform(rng, 1, 40000 if kind == "few" else 13000) for n in q]
        kv = rng.choice([1, 2, 4, 8])
        case = attention_case("", dtype, rng.choice([64, 128, 128]), "%d/%d" % (kv * rng.choice([1, 4, 8]) if kv < 8 else 32, kv),
                              join(q), join(k), causal=True, cap=rng.choice([0.0, 50.0]), axes=rng.randint(0, 1), lse=rng.random() < 0.3)
    del case["name"]
    return case


# ------------------------------------------------------------------------- sizes and work
def numbers(text):
    """The numbers of "5,17,64x3"."""
    parts = [p.split("x") for p in text.split(",")] if text else []
    return [int(p[0]) for p in parts for _ in range(int(p[1]) if len(p) > 1 else 1)]


def two(heads):
    return tuple(int(h) for h in heads.split("/"))


def prefixes(case):
    return numbers(case["prefix"]) or [0] * len(numbers(case["q"]))


def seen(case):
    """Keys that all queries of all documents see, counted pair by pair."""
    total = 0
    for nq, nk, p in zip(numbers(case["q"]), numbers(case["kv"]), prefixes(case)):
        total += sum(min(nk, max(p, i + 1 + nk - nq, 0)) for i in range(nq)) if case["causal"] else nq * nk
    return total


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    qh, kh = two(case["heads"])
    d = case["head_dim"]
    if case["op"] == "rotary":
        n = case["tokens"] * (qh + kh)
        pairs = sum(numbers(case["sections"]))
        return {"bytes": 2 * n * d * size + 4 * case["tokens"] * len(numbers(case["sections"])), "flops": 6 * n * pairs}
    tq, tk = sum(numbers(case["q"])), sum(numbers(case["kv"]))
    io = 2 * tq * qh * d * size + 2 * tk * kh * d * size
    return {"bytes": io + 4 * case["axes"] * (tq + tk) + (4 * tq * qh if case["lse"] else 0), "flops": 4 * d * qh * seen(case)}


# ------------------------------------------------------------------------------ the inputs
def grid_positions(index, axes, grid):
    """Positions [axes, tokens] of the tokens `index` of an image (two axes) or of frames of 7 rows (three)."""
    rows = index // max(grid, 1)
    return torch.stack({1: [index], 2: [rows, index % max(grid, 1)], 3: [rows // 7, rows % 7, index % max(grid, 1)]}[axes])


def prepare(case, seed):
    rng = torch.Generator(device="cuda").manual_seed(seed)
    dtype, d, (qh, kh) = DTYPES[case["dtype"]], case["head_dim"], two(case["heads"])

    def normal(*shape):
        return torch.randn(*shape, generator=rng, device="cuda", dtype=torch.float32)

    if case["op"] == "rotary":
        sections = numbers(case["sections"])
        index = torch.arange(case["start"], case["start"] + case["tokens"], device="cuda")
        pos = grid_positions(index, len(sections), case["grid"]).to(torch.int32)
        rows = normal(case["tokens"], qh + kh, d).to(dtype)  # q and k heads of a token behind one another
        return {"case": case, "q": rows[:, :qh], "k": rows[:, qh:], "pos": pos, "sections": sections}

    qn, kn = numbers(case["q"]), numbers(case["kv"])
    tq, tk = sum(qn), sum(kn)
    if case["fused"]:
        rows = normal(tq, qh, 3, d).to(dtype)
        q, k, v = rows.unbind(2)
    else:
        q, k, v = normal(tq, qh, d).to(dtype), normal(tk, kh, d).to(dtype), normal(tk, kh, d).to(dtype)
    # queries that look for something, and values with a mean of their own in each channel
    q.mul_(1.5)
    v.add_(normal(v.shape[1], d).to(dtype))

    def offsets(n):
        return torch.tensor([0] + n, device="cuda").cumsum(0).to(torch.int32)

    state = {"case": case, "q": q, "k": k, "v": v, "q_offsets": offsets(qn), "kv_offsets": offsets(kn), "prefix": None,
             "slopes": None, "q_pos": None, "kv_pos": None, "scale": d ** -0.5}
    if case["prefix"]:
        state["prefix"] = torch.tensor(numbers(case["prefix"]), device="cuda", dtype=torch.int32)
    if case["axes"]:
        kv_index = torch.cat([torch.arange(n, device="cuda") for n in kn])
        q_index = torch.cat([torch.arange(b - a, b, device="cuda") for a, b in zip(qn, kn)])
        state["kv_pos"] = grid_positions(kv_index, case["axes"], case["grid"]).to(torch.int32)
        state["q_pos"] = grid_positions(q_index, case["axes"], case["grid"]).to(torch.int32)
        steps = torch.arange(1, qh + 1, device="cuda") * (-8.0 / qh)
        state["slopes"] = torch.exp2(steps)[None, :] * (1 + 0.1 * normal(case["axes"], qh).abs())
    return state


# --------------------------------------------------------------------------- one pass
def run(state):
    rotary = state["case"]["op"] == "rotary"
    if own:
        return own_rotary(state) if rotary else own_attention(state)
    return plain_rotary(state) if rotary else plain_attention(state)


def frequencies(sections, per_axis, base=10000.0):
    """Angle per unit of position, and the position axis, of each pair."""
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    at = [i for n in sections for i in range(n)] if per_axis else list(range(len(axis)))
    of = [sections[a] for a in axis] if per_axis else [len(axis)] * len(axis)
    return [base ** (-i / n) for i, n in zip(at, of)], axis


def plain_rotary(state):
    case = state["case"]
    freq, axis = frequencies(state["sections"], case["per_axis"])
    pairs = len(freq)
    # in 64 bits: a far position's angle has no room for its fraction in 32
    angle = state["pos"].double()[axis].T * torch.tensor(freq, device="cuda", dtype=torch.float64)
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if case["inverse"]:
        s = -s

    def turned(x):
        y = x.float()
        if case["interleaved"]:
            a, b = y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]
            z = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
        else:
            a, b = y[..., :pairs], y[..., pairs:2 * pairs]
            z = torch.cat([a * c - b * s, a * s + b * c], -1)
        return torch.cat([z, y[..., 2 * pairs:]], -1).to(x.dtype)

    return turned(state["q"]), turned(state["k"])


def plain_attention(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    qo, ko = state["q_offsets"].long(), state["kv_offsets"].long()
    nq, nk = qo.diff()[:, None], ko.diff()[:, None]
    # documents side by side, the short ones filled up: [documents, longest]
    i = torch.arange(max(numbers(case["q"])), device="cuda")[None]
    j = torch.arange(max(numbers(case["kv"])), device="cuda")[None]
    qrow, krow = (qo[:-1, None] + i).clamp(max=q.shape[0] - 1), (ko[:-1, None] + j).clamp(max=k.shape[0] - 1)
    group = q.shape[1] // k.shape[1]
    s = q.float()[qrow].unflatten(2, (k.shape[1], group)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [doc, kv head, group * i, d]
    s = torch.matmul(s, k.float()[krow].permute(0, 2, 3, 1)).unflatten(2, (group, -1)).flatten(1, 2)  # [doc, head, i, j]
    s *= state["scale"]
    if case["cap"]:
        s = s.div_(case["cap"]).tanh_().mul_(case["cap"])
    if case["axes"]:
        for axis in range(case["axes"]):
            far = (state["q_pos"][axis][qrow][:, :, None] - state["kv_pos"][axis][krow][:, None, :]).abs().float()
            s.addcmul_(state["slopes"][axis][None, :, None, None], far[:, None], value=-1)
    count = nk.expand(-1, i.shape[1])
    if case["causal"]:
        before = 0 if state["prefix"] is None else state["prefix"].long()[:, None]
        count = torch.minimum(nk, (i + 1 + nk - nq).clamp(min=0).clamp(min=before))
    s.masked_fill_((j[:, None] >= count[:, :, None])[:, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)  # rows that see nothing: a finite top
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    values = v.float()[krow].permute(0, 2, 1, 3)
    o = torch.matmul(p.unflatten(1, (k.shape[1], group)).flatten(2, 3), values).unflatten(2, (group, -1)).flatten(1, 2)
    o = torch.where(total > 0, o / total, 0.0).transpose(1, 2)  # [doc, i, head, d]
    here = i < nq
    out = torch.empty(q.shape, device="cuda", dtype=q.dtype)
    out[qrow[here]] = o[here].to(q.dtype)
    if not case["lse"]:
        return out
    lse = torch.empty(q.shape[1], q.shape[0], device="cuda")
    lse[:, qrow[here]] = (top + total.log())[..., 0].transpose(1, 2)[here].T
    return out, lse


def library():
    """The package (its folder's name is no identifier) and its binding."""
    if "swin2sr_b200" not in sys.modules:
        folder = Path(__file__).resolve().parents[1] / "swin2sr-rs_b200"
        spec = importlib.util.spec_from_file_location("swin2sr_b200", folder / "__init__.py", submodule_search_locations=[str(folder)])
        sys.modules["swin2sr_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["swin2sr_b200"])
    return importlib.import_module("swin2sr_b200.capi")


capi = None  # the binding, once it is used


def heads_of(x):
    return capi.heads(x.data_ptr(), x.stride(0), x.stride(1), x.shape[1])


def own_rotary(state):
    global capi
    capi = capi or library()
    case, q, k, pos = state["case"], state["q"], state["k"], state["pos"]
    if "plan" not in state:  # of the sections alone: a program makes it once
        state["plan"] = capi.rotary_plan(state["sections"], 10000.0, case["per_axis"], case["interleaved"])
    out_q, out_k = torch.empty(q.shape, device="cuda", dtype=q.dtype), torch.empty(k.shape, device="cuda", dtype=k.dtype)
    capi.rotary(state["plan"], case["dtype"], q.shape[2], q.shape[0], pos.data_ptr(), pos.stride(0),
                ((heads_of(q), heads_of(out_q)), (heads_of(k), heads_of(out_k))), case["inverse"],
                torch.cuda.current_stream().cuda_stream)
    return out_q, out_k


def own_attention(state):
    global capi
    capi = capi or library()
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    out = torch.empty(q.shape, device="cuda", dtype=q.dtype)
    lse = torch.empty(q.shape[1], q.shape[0], device="cuda") if case["lse"] else None
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    capi.attention(case["dtype"], q.shape[2], state["scale"], heads_of(q), heads_of(k), heads_of(v), heads_of(out), q.shape[0],
                   k.shape[0], documents=state["q_offsets"].shape[0] - 1, d_q_offsets=at(state["q_offsets"]),
                   d_kv_offsets=at(state["kv_offsets"]), causal=case["causal"], d_prefix=at(state["prefix"]), cap=case["cap"],
                   axes=case["axes"], d_slopes=at(state["slopes"]), d_q_pos=at(state["q_pos"]), d_kv_pos=at(state["kv_pos"]),
                   d_lse=at(lse), stream=torch.cuda.current_stream().cuda_stream)
    return out if lse is None else (out, lse)


# ------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    return exact_rotary(case, seed) if case["op"] == "rotary" else exact_attention(case, seed)


def exact_rotary(case, seed):
    """Pairs as complex numbers, multiplied by exp(i position frequency)."""
    state = prepare(case, seed)
    sections, sign = state["sections"], -1.0 if case["inverse"] else 1.0
    pairs, answers = sum(sections), []
    for x in (state["q"], state["k"]):
        y, first = x.double().clone(), 0
        for a, n in enumerate(sections):
            for m in range(n):
                p = first + m
                power = m / n if case["per_axis"] else p / pairs
                turn = torch.polar(torch.ones(case["tokens"], device="cuda", dtype=torch.float64),
                                   sign * state["pos"][a].double() * 10000.0 ** -power)[:, None]
                one, other = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + pairs)
                z = torch.complex(x[..., one].double(), x[..., other].double()) * turn
                y[..., one], y[..., other] = z.real, z.imag
            first += n
        answers.append(y)
    return tuple(answers)


def exact_attention(case, seed):
    """Document by document and head by head."""
    state = prepare(case, seed)
    q, k, v = state["q"], state["k"], state["v"]
    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    lse = torch.full((q.shape[1], q.shape[0]), -math.inf, device="cuda", dtype=torch.float64)
    lengths = list(zip(numbers(case["q"]), numbers(case["kv"]), prefixes(case)))
    alike = len(set(lengths)) == 1 and len(lengths) > 1  # documents of one size at once
    fold = len(lengths) if alike else 1
    qs = ks = 0
    for nq, nk, prefix in lengths[:1] if alike else lengths:
        shape = lambda t, n: t[:fold * n].reshape(fold, n, *t.shape[1:]) if alike else t[None]  # noqa: E731
        for h in range(q.shape[1]):
            g = h // group
            a = shape(q[:, h] if alike else q[qs:qs + nq, h], nq).double()
            b = shape(k[:, g] if alike else k[ks:ks + nk, g], nk).double()
            s = a @ b.mT * state["scale"]
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            for axis in range(case["axes"]):
                x = shape(state["q_pos"][axis] if alike else state["q_pos"][axis][qs:qs + nq], nq).double()
                y = shape(state["kv_pos"][axis] if alike else state["kv_pos"][axis][ks:ks + nk], nk).double()
                s -= state["slopes"][axis, h].double() * (x[..., :, None] - y[..., None, :]).abs()
            if case["causal"]:
                i, j = torch.arange(nq, device="cuda")[:, None], torch.arange(nk, device="cuda")[None]
                s = torch.where((j <= i + (nk - nq)) | (j < prefix), s, -math.inf)
            w = torch.logsumexp(s, -1)
            p = torch.where(w[..., None] > -math.inf, torch.exp(s - w[..., None]), 0.0)
            o = p @ shape(v[:, g] if alike else v[ks:ks + nk, g], nk).double()
            out[qs:qs + fold * nq, h] = o.flatten(0, 1)
            lse[h, qs:qs + fold * nq] = w.flatten()
        qs, ks = qs + nq, ks + nk
    return (out, lse) if case["lse"] else out
