"""Performance cases of the paged key-value cache: what a server of many sequences calls between the projections of a layer.

  append  rotary positions of one or several axes for q and k, and k and v written to their pages
  step    attention of one new token of every sequence over its pages
  prompt  attention of several new tokens of every sequence (a prompt, or a part of one behind a filled cache), causal

Rows are ragged: those of sequence i are `starts[i] .. starts[i + 1] - 1`, and its cache has `lens[i]` positions, the new ones
among them.  q, k and v are views of one tensor of rows, as a fused projection leaves them.  Pages are handed out in random order."""
from __future__ import annotations

import math

import torch

own = False
GPU = "cuda"
TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases
def _case(kind, seqs, new, past, heads, kv_heads, dim, page, act, pages, window=0, axes=1, interleaved=False):
    """`new` and `past`: the most new and earlier positions of a sequence; the others have between a quarter of that and all of it."""
    c = dict(kind=kind, seqs=seqs, new=new, past=past, heads=heads, kv_heads=kv_heads, dim=dim, page=page, act=act, pages=pages)
    if kind == "append":
        c.update(axes=axes, interleaved=interleaved)
    else:
        c.update(window=window)
    return c


def listed():
    return [
        # one conversation, one new token, the cache type of the Llama decoder: nothing but latency
        dict(_case("append", 1, 1, 299, 32, 8, 128, 16, "f32", "f32", interleaved=True), name="append_1_token_f32"),
        # a decode step of 64 conversations
        dict(_case("append", 64, 1, 4000, 32, 8, 128, 32, "bf16", "bf16"), name="append_64_sequences_bf16"),
        # prompts of text and pictures: three axes
        dict(_case("append", 4, 8192, 0, 32, 8, 128, 64, "f16", "f16", axes=3), name="append_prompts_3_axes_f16"),
        # one short conversation: the smallest call
        dict(_case("step", 1, 1, 299, 32, 8, 128, 16, "f32", "f32"), name="step_300_f32"),
        # a decode step of 32 conversations of ordinary length
        dict(_case("step", 32, 1, 2047, 32, 8, 128, 16, "f16", "f16"), name="step_32x2048_f16"),
        # one new token behind a very long document
        dict(_case("step", 1, 1, 131071, 32, 8, 128, 64, "bf16", "bf16"), name="step_131072_bf16"),
        # a large batch: f32 rows over f16 pages (the decoders' residual stream is f32), eight heads a KV head
        dict(_case("step", 64, 1, 8191, 64, 8, 128, 32, "f32", "f16"), name="step_64x8192_f32_f16"),
        # a short odd prompt of a small model
        dict(_case("prompt", 1, 77, 0, 8, 2, 64, 16, "f16", "f16"), name="prompt_77_f16"),
        # parts of prompts of eight conversations behind what they have cached
        dict(_case("prompt", 8, 512, 4001, 32, 8, 128, 16, "bf16", "bf16"), name="prompt_8x512_behind_4001_bf16"),
        # a long prompt from its start
        dict(_case("prompt", 1, 8192, 0, 32, 8, 128, 64, "f16", "f16"), name="prompt_8192_f16"),
        # a few tokens behind a very long document (a question about it): few rows, a long axis
        dict(_case("prompt", 1, 33, 65536, 32, 8, 128, 64, "f16", "f16"), name="prompt_33_behind_65536_f16"),
        # layers with a window, everything in f32
        dict(_case("prompt", 2, 2049, 500, 16, 4, 64, 32, "f32", "f32", window=1024), name="prompt_2x2049_window_f32"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "step", "step", "step", "prompt", "prompt", "prompt"])
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 4, 4, 5, 8])
    dim = rng.choice([64, 64, 96, 128, 128, 128, 256]) if kv * 256 <= 1024 else rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 64, 128])
    act, pages = rng.choice([("f32", "f32"), ("f16", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")])
    window = rng.choice([0, 0, 0, _spread(rng, 64, 4096)])
    if kind == "append":
        seqs = _spread(rng, 1, 64)
        new = rng.choice([1, _spread(rng, 1, 16384 // seqs)])
        return _case(kind, seqs, new, _spread(rng, 1, 8192 // seqs + 1), heads, kv, dim, page, act, pages, axes=rng.choice([1, 3]), interleaved=rng.choice([False, True]))
    if kind == "step":
        seqs = _spread(rng, 1, 64)
        return _case(kind, seqs, 1, _spread(rng, 1, min(65536, 262144 // seqs)), heads, kv, dim, page, act, pages, window)
    seqs = _spread(rng, 1, 8)
    new = _spread(rng, 2, 2048 // seqs)
    return _case(kind, seqs, new, rng.choice([0, _spread(rng, 1, 8192 // seqs)]), heads, kv, dim, page, act, pages, window)


def _lengths(case):
    """New and cached positions of every sequence: the first has the most, the others spread down to a quarter."""
    n, at = case["seqs"], range(case["seqs"])
    share = [1.0 - 0.75 * ((i * 0.6180339887498949) % 1.0) for i in at]
    new = [case["new"] if i == 0 else max(1, round(case["new"] * share[i])) for i in at]
    past = [case["past"] if i == 0 else round(case["past"] * share[n - i]) for i in at]
    return new, past


def _sections(case):
    pairs = case["dim"] // 2
    return [pairs] if case["axes"] == 1 else [pairs // 4, 3 * pairs // 8, pairs - pairs // 4 - 3 * pairs // 8]


# ---------------------------------------------------------------- inputs
def _generator(seed, *what):
    h = 1469598103934665603
    for ch in repr((int(seed),) + what).encode():
        h = (h ^ ch) * 1099511628211 % (1 << 62)
    return torch.Generator(device=GPU).manual_seed(h)


def prepare(case, seed):
    new, past = _lengths(case)
    n, d, page, hq, hkv = case["seqs"], case["dim"], case["page"], case["heads"], case["kv_heads"]
    g = _generator(seed, "inputs", case["kind"])
    act, kept = TYPE[case["act"]], TYPE[case["pages"]]
    lens = [a + b for a, b in zip(new, past)]
    need = [-(-x // page) for x in lens]
    cols, pages = max(need), sum(need) + 3
    starts = torch.tensor([0] + new, device=GPU).cumsum(0).to(torch.int32)
    tokens = sum(new)
    s = dict(case=case, starts=starts, lens=torch.tensor(lens, dtype=torch.int32, device=GPU), tokens=tokens, max_new=max(new), max_len=max(lens))
    order = torch.randperm(pages, generator=g, device=GPU).to(torch.int32)
    table = torch.zeros(n, cols, dtype=torch.int32, device=GPU)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c
    s["table"] = table
    # heads differ in how sharply they look, and a few channels of K are large
    rows = torch.randn(tokens, hq + 2 * hkv, d, generator=g, device=GPU)
    rows[:, :hq] *= torch.linspace(0.5, 2.0, hq, device=GPU)[:, None]
    s["rows"] = rows.to(act).view(tokens, (hq + 2 * hkv) * d)
    strong = torch.ones(d, device=GPU)
    strong[::37] = 3.0
    s["k"] = torch.randn(pages, hkv, page, d, generator=g, device=GPU).mul_(strong).to(kept)
    s["v"] = torch.randn(pages, hkv, page, d, generator=g, device=GPU).to(kept)
    s["out"] = torch.empty(tokens, hq, d, dtype=act, device=GPU)
    if case["kind"] == "append":
        reach = max(lens)
        f = 500000.0 ** (-2.0 * torch.arange(d // 2, device=GPU, dtype=torch.float64) / d)
        angle = torch.arange(reach, device=GPU, dtype=torch.float64)[:, None] * f
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["axes"] > 1:  # text has its position on every axis, a picture its rows and columns
            t = torch.arange(tokens, device=GPU) % reach
            s["positions"] = torch.stack([t, t // 2, torch.randint(0, reach, (tokens,), generator=g, device=GPU)]).to(torch.int32)
        else:
            s["positions"] = None
    if own:
        s["calls"] = _handles(s)
    return s


_devices = []


def _handles(s):
    """The framework's tensors over the same memory, and the cache and batch that a program keeps."""
    from kalosm_amd.fusor import Device, PagedBatch, PagedKvCache, RopeCache, Tensor

    if not _devices:
        _devices.append(Device.gpu(0))
    dev, case = _devices[0], s["case"]
    name = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16", torch.int32: "i32"}

    def over(t, shape=None, offset=0):
        return Tensor(dev, t.shape if shape is None else shape, name[t.dtype], ptr=t.data_ptr() + offset * t.element_size())

    n, hq, hkv, d = s["tokens"], case["heads"], case["kv_heads"], case["dim"]
    strides = ((hq + 2 * hkv) * d, d)
    h = dict(cache=PagedKvCache.over(over(s["k"]), over(s["v"])), strides=strides,
             batch=PagedBatch(over(s["lens"]), over(s["table"]), over(s["starts"]), tokens=n, max_new=s["max_new"], max_len=s["max_len"]),
             q=over(s["rows"], (n, hq, d)), out=over(s["out"]))
    if case["kind"] == "append":
        h.update(k=over(s["rows"], (n, hkv, d), hq * d), v=over(s["rows"], (n, hkv, d), (hq + hkv) * d), rope=RopeCache.from_parts(over(s["cos"]), over(s["sin"])),
                 positions=None if s["positions"] is None else over(s["positions"]), sections=None if case["axes"] == 1 else _sections(case))
    return h


# ---------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    if own:
        h = s["calls"]
        if case["kind"] == "append":
            h["rope"].forward_paged(h["q"], h["k"], h["v"], h["cache"], h["batch"], positions=h["positions"], sections=h["sections"],
                                    interleaved=case["interleaved"], strides=h["strides"], out=h["out"])
            return s["out"], s["k"], s["v"]
        h["q"].paged_attention(h["cache"], h["batch"], 1.0 / math.sqrt(case["dim"]), window=case["window"], strides=h["strides"], out=h["out"])
        return s["out"]
    return _plain_append(s) if case["kind"] == "append" else _plain_attention(s)


def _owners(s):
    """Sequence and position of every row."""
    row = torch.arange(s["tokens"], device=GPU, dtype=torch.int32)
    seq = torch.searchsorted(s["starts"], row, right=True) - 1
    return seq, (s["lens"][seq] - (s["starts"][seq + 1] - row)).long()


def _plain_append(s):
    case, n = s["case"], s["tokens"]
    hq, hkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    seq, pos = _owners(s)
    x = s["rows"].view(n, hq + 2 * hkv, d)
    if s["positions"] is None:
        c, sn = s["cos"][pos], s["sin"][pos]
    else:
        axis = torch.repeat_interleave(torch.arange(3, device=GPU), torch.tensor(_sections(case), device=GPU), output_size=d // 2)
        at, pair = s["positions"].long()[axis].T, torch.arange(d // 2, device=GPU)
        c, sn = s["cos"][at, pair], s["sin"][at, pair]
    c, sn = c[:, None], sn[:, None]
    r = x[:, :hq + hkv].float()
    if case["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)
    else:
        a, b = r[..., :d // 2], r[..., d // 2:]
        r = torch.cat([a * c - b * sn, a * sn + b * c], -1)
    where = s["table"][seq, pos // page].long()
    s["k"][where, :, pos % page] = r[:, hq:].to(s["k"].dtype)
    s["v"][where, :, pos % page] = x[:, hq + hkv:].to(s["v"].dtype)
    return r[:, :hq].to(x.dtype), s["k"], s["v"]


def _plain_attention(s):
    case, n = s["case"], s["tokens"]
    hq, hkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    seqs, new, group = case["seqs"], s["max_new"], hq // hkv
    cols = s["table"].shape[1]
    seq, pos = _owners(s)
    slot = torch.arange(n, device=GPU) - s["starts"][seq].long()
    q = torch.zeros(seqs, new, hkv, group, d, device=GPU)
    q[seq, slot] = s["rows"].view(n, hq + 2 * hkv, d)[:, :hq].float().view(n, hkv, group, d)
    at = torch.full((seqs, new), -1, device=GPU)
    at[seq, slot] = pos
    keys = torch.arange(cols * page, device=GPU)
    seen = (keys <= at[:, :, None]) & (keys < s["lens"][:, None, None])
    if case["window"]:
        seen &= keys > at[:, :, None] - case["window"]
    k = s["k"][s["table"].long()].transpose(1, 2).reshape(seqs, hkv, cols * page, d).float()
    v = s["v"][s["table"].long()].transpose(1, 2).reshape(seqs, hkv, cols * page, d).float()
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, hkv, group * new, d)
    score = (q @ k.transpose(2, 3)).view(seqs, hkv, group, new, cols * page).mul_(1.0 / math.sqrt(d))
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp_min(-3e38)
    w = score.exp_()
    total = w.sum(-1, keepdim=True)
    o = (w.view(seqs, hkv, group * new, cols * page) @ v).view(seqs, hkv, group, new, d) / total.clamp_min(1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(seqs, new, hq, d)[seq, slot].to(s["rows"].dtype)


# ---------------------------------------------------------------- what a pass cannot do without, and its exact result
def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    new, past = _lengths(case)
    hq, hkv, d, a, p = case["heads"], case["kv_heads"], case["dim"], _size(case["act"]), _size(case["pages"])
    rows = sum(new)
    if case["kind"] == "append":
        tables = (sum(new) if case["axes"] == 1 else sum(new) * case["axes"]) * 4 + rows * d * 4
        return {"bytes": rows * d * ((2 * hq + 2 * hkv) * a + 2 * hkv * p) + tables, "flops": 3.0 * rows * (hq + hkv) * d}
    w = case["window"]
    pairs = read = 0
    for m, b in zip(new, past):
        if not w:
            pairs, read = pairs + m * b + m * (m + 1) // 2, read + m + b
        else:
            short = max(0, min(m, w - b))  # rows that see everything before them
            pairs, read = pairs + short * b + short * (short + 1) // 2 + (m - short) * w, read + min(m + b, m + w - 1)
    return {"bytes": 2 * read * hkv * d * p + 2 * rows * hq * d * a, "flops": 4.0 * pairs * hq * d}


def exact(case, seed):
    s = prepare(case, seed)
    new, past = _lengths(case)
    hq, hkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group, table = hq // hkv, s["table"].tolist()
    x = s["rows"].double().view(-1, hq + 2 * hkv, d)
    if case["kind"] == "append":
        return _exact_append(s, case, new, past, x, table)
    out, r0 = torch.empty(s["tokens"], hq, d, dtype=torch.float64, device=GPU), 0
    for i, (m, b) in enumerate(zip(new, past)):
        held = table[i][:-(-(m + b) // page)]
        mine = torch.arange(b, b + m, device=GPU)[:, None]
        other = torch.arange(m + b, device=GPU)[None]
        hidden = other > mine
        if case["window"]:
            hidden = hidden | (mine - other >= case["window"])
        for h in range(hkv):
            k = s["k"][held, h].double().reshape(-1, d)[:m + b]
            v = s["v"][held, h].double().reshape(-1, d)[:m + b]
            for e in range(h * group, (h + 1) * group):
                p = torch.softmax((x[r0:r0 + m, e] @ k.t().contiguous() / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                out[r0:r0 + m, e] = p @ v
        r0 += m
    return out


def _exact_append(s, case, new, past, x, table):
    hq, hkv, d, page, half = case["heads"], case["kv_heads"], case["dim"], case["page"], case["dim"] // 2
    k, v = s["k"].double(), s["v"].double()
    position = torch.cat([torch.arange(b, b + m, device=GPU) for m, b in zip(new, past)])
    cos, sin = torch.empty(len(x), half, dtype=torch.float64, device=GPU), torch.empty(len(x), half, dtype=torch.float64, device=GPU)
    first = 0
    for a, many in enumerate(_sections(case)):
        at = position if s["positions"] is None else s["positions"][a].long()
        cos[:, first:first + many], sin[:, first:first + many] = s["cos"][at, first:first + many].double(), s["sin"][at, first:first + many].double()
        first += many
    turn = torch.complex(cos, sin)[:, None]
    y = x.clone()
    i0, i1 = (slice(0, d, 2), slice(1, d, 2)) if case["interleaved"] else (slice(0, half), slice(half, d))
    z = torch.complex(x[:, :hq + hkv, i0], x[:, :hq + hkv, i1]) * turn
    y[:, :hq + hkv, i0], y[:, :hq + hkv, i1] = z.real, z.imag
    r0 = 0
    for i, (m, b) in enumerate(zip(new, past)):
        for j in range(b // page, -(-(m + b) // page)):
            lo, hi = max(b, j * page), min(m + b, (j + 1) * page)
            rows = y[r0 + lo - b:r0 + hi - b]
            k[table[i][j], :, lo - j * page:hi - j * page] = rows[:, hq:hq + hkv].transpose(0, 1)
            v[table[i][j], :, lo - j * page:hi - j * page] = rows[:, hq + hkv:].transpose(0, 1)
        r0 += m
    return y[:, :hq], k, v
