"""Cases of the 8-bit operators of a decoder block: the quantized linear layer, the quantized
paged cache (write and read back) and the attention of new tokens over that cache.

``run`` computes a case in elementary torch operations, or with the framework's operators when
``own`` is set.  The formulas:

linear      s_t = max_k |x_tk| / 127,  c_tk = round(x_tk / s_t);  y_tn = act(s_t w_n sum_k c_tk W_kn + b_n)
cache       per token and kv head the same rule over the head's elements; reading back gives c * s
attention   token i of a sequence with `new` new tokens and `length` cached ones (the new ones
            among them) sees the keys 0 .. length - new + i:
            o = sum_j softmax_j(scale q.k_j) v_j,  0 where it sees none
"""
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

_ROOT = Path(__file__).resolve().parent.parent


def _package():
    if "wechat_tfcc_b200" not in sys.modules:
        spec = importlib.util.spec_from_file_location("__graft_entry__", _ROOT / "__graft_entry__.py")
        entry = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(entry)
        entry.load_package()
    return sys.modules["wechat_tfcc_b200"]


# ---------------------------------------------------------------------------------------------
# cases

# the largest case of each kind bounds what draw() may ask for
_LINEAR_FLOPS = 2 * 4096 * 4096 * 16384
_CACHE_VALUES = 16384 * 8 * 128
_ATTENTION_FLOPS = 4 * 128 * 32 * 4096 * 6144
_ATTENTION_BYTES = 300_000_000


def _linear(name, tokens, k, n, bias=True, gelu=False):
    return {"name": name, "kind": "linear", "tokens": tokens, "k": k, "n": n, "bias": bias, "gelu": gelu}


def _paged(name, kind, batch, heads, kv_heads, dim, page, new, past, mix=0, causal=True):
    """`new` / `past`: "lowest-highest" tokens of a sequence, spread by the number `mix`."""
    c = {"name": name, "kind": kind, "batch": batch, "kv_heads": kv_heads, "dim": dim, "page": page, "new": new,
         "past": past, "mix": mix}
    if kind == "attention":
        c.update(heads=heads, causal=causal)
    return c


def listed():
    return [
        # one token through a projection of the encoder's width: latency alone counts
        _linear("linear 1x768x768", 1, 768, 768),
        # a decode step of 16 sequences through a wide layer: the weights are the traffic
        _linear("linear 16x4096x16384", 16, 4096, 16384, gelu=True),
        # a batch of ragged prompts, widths that divide by nothing
        _linear("linear 777x1003x2050", 777, 1003, 2050, bias=False),
        # a chunk of a long prompt through a feed-forward layer
        _linear("linear 4096x4096x16384", 4096, 4096, 16384, gelu=True),
        # decode step: one token for each of 8 sequences
        _paged("cache 8x1, 8x128", "cache", 8, 8, 8, 128, 64, "1-1", "1-4000", mix=1),
        # ragged chunks over small pages
        _paged("cache 5 ragged, 12x64", "cache", 5, 12, 12, 64, 16, "3-1500", "0-700", mix=2),
        # prompts as they come in
        _paged("cache 16x1024, 8x128", "cache", 16, 8, 8, 128, 64, "1024-1024", "0-0"),
        # one short sequence at decode: latency
        _paged("decode 1x100, 12/12x64", "attention", 1, 12, 12, 64, 16, "1-1", "99-99"),
        # decode of a full batch of ragged lengths, grouped heads
        _paged("decode 32 ragged, 32/8x128", "attention", 32, 32, 8, 128, 64, "1-1", "100-8191", mix=3),
        # two long contexts: few rows, the keys' axis has to be shared out
        _paged("decode 2x65536, 64/8x128", "attention", 2, 64, 8, 128, 128, "1-1", "65535-65535"),
        # chunks and single tokens in one batch, some from an empty cache
        _paged("mixed 7 ragged, 12/12x64", "attention", 7, 12, 12, 64, 16, "1-900", "0-5000", mix=4),
        # a chunk of a long prompt
        _paged("chunk 4096 on 4096, 32/8x128", "attention", 1, 32, 8, 128, 64, "4096-4096", "4096-4096"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def _range(rng, lo, hi):
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return "%d-%d" % (a, b)


def draw(rng):
    while True:
        kind = rng.choice(["linear", "cache", "attention", "attention"])
        if kind == "linear":
            c = _linear("", _log(rng, 1, 4096), _log(rng, 64, 8192), _log(rng, 64, 16384), rng.random() < 0.5, rng.random() < 0.3)
            if rng.random() < 0.5:  # half of the layers have the widths that models have
                c["k"], c["n"] = max(64, c["k"] // 64 * 64), max(64, c["n"] // 64 * 64)
            fits = work(c)["flops"] <= _LINEAR_FLOPS
        else:
            dim = rng.choice([64, 128])
            kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
            heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
            page = rng.choice([8, 16, 32, 64, 128, 256])
            new = "1-1" if rng.random() < 0.4 else _range(rng, 1, 4096)
            past = rng.choice(["0-0", _range(rng, 1, 60000), _range(rng, 1, 8000)])
            c = _paged("", kind, _log(rng, 1, 48), heads, kv_heads, dim, page, new, past, rng.randrange(1000), rng.random() < 0.85)
            news, lengths = _lengths(c)
            if kind == "cache":
                fits = sum(news) * kv_heads * dim <= _CACHE_VALUES and sum(lengths) * kv_heads * dim <= 8 * _CACHE_VALUES
            else:
                w = work(c)
                padded = len(news) * max(news) * heads * max(lengths)  # scores of the plain form
                fits = w["flops"] <= _ATTENTION_FLOPS and w["bytes"] <= _ATTENTION_BYTES and padded <= 32 * 4096 * 8192
                fits = fits and len(news) * max(lengths) * kv_heads * dim <= 2 * 65536 * 8 * 128 * 4
        if fits:
            del c["name"]
            return c


def _lengths(case):
    """New tokens and cached tokens (the new ones among them) of every sequence."""
    rng = random.Random(case["mix"])
    lo, hi = (int(v) for v in case["new"].split("-"))
    plo, phi = (int(v) for v in case["past"].split("-"))
    news = [rng.randint(lo, hi) for _ in range(case["batch"])]
    return news, [n + rng.randint(plo, phi) for n in news]


def work(case):
    if case["kind"] == "linear":
        m, k, n = case["tokens"], case["k"], case["n"]
        return {"bytes": 4 * m * k + k * n + 4 * n + (4 * n if case["bias"] else 0) + 4 * m * n, "flops": 2 * m * k * n}
    news, lengths = _lengths(case)
    width = case["kv_heads"] * case["dim"]
    held = 2 * case["kv_heads"] * (case["dim"] + 4)  # bytes of a cached token, scales among them
    if case["kind"] == "cache":  # write and read back: values in, codes out and in, values out
        return {"bytes": sum(news) * (2 * 4 * width + 2 * held + 2 * 4 * width), "flops": 6 * 2 * sum(news) * width}
    seen = 0
    for new, length in zip(news, lengths):
        seen += new * length - (new * (new - 1) // 2 if case["causal"] else 0)
    return {"bytes": 2 * 4 * sum(news) * case["heads"] * case["dim"] + sum(lengths) * held,
            "flops": 4 * case["dim"] * case["heads"] * seen}


# ---------------------------------------------------------------------------------------------
# inputs


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    s = dict(case)
    if case["kind"] == "linear":
        m, k, n = case["tokens"], case["k"], case["n"]
        # activations with some channels larger than the others
        s["x"] = normal(m, k) * torch.exp(0.5 * normal(k))
        # weights quantized once per output channel, as they are kept; rows start on 16 bytes
        pitch = (n + 15) // 16 * 16
        w = torch.zeros(k, pitch, dtype=torch.int8, device=dev)
        w[:, :n] = (normal(k, n) * 36).round_().clamp_(-127, 127)
        s["w"] = w[:, :n]
        s["w_scales"] = torch.exp(0.3 * normal(n)) * (0.02 / 36)
        s["b"] = 0.1 * normal(n) if case["bias"] else None
        return s
    news, lengths = _lengths(case)
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    need = [(n + page - 1) // page for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, device=dev, generator=gen).to(torch.int32)
    table = torch.zeros(len(news), max(need), dtype=torch.int32, device=dev)
    first = 0
    for i, n in enumerate(need):
        table[i, :n] = order[first:first + n]
        first += n
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    s.update(table=table, starts=torch.tensor(starts, dtype=torch.int32, device=dev),
             lengths=torch.tensor(lengths, dtype=torch.int32, device=dev), rows=starts[-1], max_new=max(news),
             max_length=max(lengths))
    shape = (pages, kv, page, dim)
    if case["kind"] == "cache":
        s["k"] = normal(starts[-1], kv * dim) * torch.exp(0.5 * normal(kv * dim))
        s["v"] = normal(starts[-1], kv * dim)
        s["pool"] = [torch.zeros(shape, dtype=torch.int8, device=dev), torch.zeros(shape[:3], device=dev),
                     torch.zeros(shape, dtype=torch.int8, device=dev), torch.zeros(shape[:3], device=dev)]
        return s
    s["q"] = normal(starts[-1], case["heads"] * dim)
    s["scale"] = 1.0 / math.sqrt(dim)
    s["pool"] = []
    for _ in range(2):
        s["pool"].append((normal(*shape) * 42).round_().clamp_(-127, 127).to(torch.int8))
        s["pool"].append(torch.exp(0.25 * normal(*shape[:3])) / 42)
    return s


# ---------------------------------------------------------------------------------------------
# the operators


def run(state):
    if own:
        return _run_own(state)
    if state["kind"] == "linear":
        return _plain_linear(state)
    if state["kind"] == "cache":
        return _plain_cache(state)
    return _plain_attention(state)


def _run_own(s):
    pkg = _package()
    if s["kind"] == "linear":
        return pkg.quantization.linear(s["x"], s["w"], s["w_scales"], s["b"], activation="gelu" if s["gelu"] else None)
    cache = pkg.cache.PagedCache(*s["pool"])
    if s["kind"] == "cache":
        pkg.cache.append(cache, s["k"], s["v"], s["starts"], s["lengths"], s["table"])
        return pkg.cache.read(cache, s["starts"], s["lengths"], s["table"], s["rows"])
    return pkg.cache.attention(cache, s["q"], s["starts"], s["lengths"], s["table"], s["scale"], causal=s["causal"],
                               max_new=s["max_new"], max_length=s["max_length"])


def _quantized(x):
    """Codes (as floats) and scales of the last axis; the quotient in 64 bits decides ties."""
    scales = (x.abs().amax(-1, keepdim=True).double() / 127).float()
    codes = torch.round(x.double() / torch.where(scales > 0, scales, torch.ones_like(scales)).double())
    return codes.clamp_(-127, 127).float(), scales


def _plain_linear(s):
    codes, scales = _quantized(s["x"])
    y = (codes @ s["w"].float()) * scales * s["w_scales"]
    if s["b"] is not None:
        y = y + s["b"]
    if s["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * (1 / math.sqrt(2))))
    return y


def _places(s):
    """Page and slot of every new token, in the order of the rows."""
    starts = s["starts"].long()
    row = torch.arange(s["rows"], device=starts.device)
    seq = torch.searchsorted(starts[1:], row, right=True)
    new = starts[1:] - starts[:-1]
    pos = row - starts[seq] + (s["lengths"].long() - new)[seq]
    return s["table"][seq, pos // s["page"]].long(), pos % s["page"]


def _plain_cache(s):
    page, slot = _places(s)
    out = []
    for x, codes, scales in ((s["k"], s["pool"][0], s["pool"][1]), (s["v"], s["pool"][2], s["pool"][3])):
        c, m = _quantized(x.view(s["rows"], s["kv_heads"], s["dim"]))
        codes[page, :, slot] = c.to(torch.int8)
        scales[page, :, slot] = m[..., 0]
        back = codes[page, :, slot].float() * scales[page, :, slot][..., None]
        out.append(back.view(s["rows"], -1))
    return tuple(out)


def _plain_attention(s):
    dev = s["q"].device
    batch, kv, dim, heads, most, longest = s["batch"], s["kv_heads"], s["dim"], s["heads"], s["max_new"], s["max_length"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    # keys and values of every sequence, padded to the longest: [batch, kv_heads, longest, dim]
    at = torch.arange(longest, device=dev)
    held = at < lengths[:, None]
    page = s["table"][:, at // s["page"]].long()
    slot = (at % s["page"]).expand_as(page)
    k = s["pool"][0][page, :, slot].float() * s["pool"][1][page, :, slot][..., None]
    v = s["pool"][2][page, :, slot].float() * s["pool"][3][page, :, slot][..., None]
    k = torch.where(held[..., None, None], k, 0.0).permute(0, 2, 1, 3)
    v = torch.where(held[..., None, None], v, 0.0).permute(0, 2, 1, 3)
    # queries padded to the most new tokens: [batch, kv_heads, group * most, dim]
    i = torch.arange(most, device=dev)
    row = (starts[:-1, None] + i).clamp_(max=s["rows"] - 1)
    q = s["q"][row].view(batch, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, -1, dim)
    scores = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    sees = (lengths - new)[:, None] + i + 1 if s["causal"] else lengths[:, None].expand(batch, most)
    mask = (at < sees[..., None]) & held[:, None]
    mask = mask[:, None].expand(batch, heads // kv, most, longest).reshape(batch, 1, -1, longest)
    scores = scores.masked_fill_(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    o = o.view(batch, kv, heads // kv, most, dim).permute(0, 3, 1, 2, 4).reshape(batch, most, heads * dim)
    return o[i < new[:, None]]


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        x = s["x"].double()
        step = (x.abs().max(dim=1).values / 127).to(torch.float32).double()
        c = torch.round(x / step[:, None])
        y = torch.einsum("tk,kn,t,n->tn", c, s["w"].double(), step, s["w_scales"].double())
        if s["b"] is not None:
            y += s["b"].double()
        return torch.special.ndtr(y) * y if case["gelu"] else y
    news, lengths = _lengths(case)
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "cache":
        out = []
        for x in (s["k"], s["v"]):
            x = x.double().reshape(-1, dim)
            step = (x.abs().max(dim=1).values / 127).to(torch.float32).double()
            out.append((torch.round(x / step[:, None]) * step[:, None]).reshape(-1, kv * dim))
        return tuple(out)
    group = case["heads"] // kv
    out = torch.zeros(sum(news), case["heads"], dim, dtype=torch.float64, device=s["q"].device)
    q = s["q"].view(-1, case["heads"], dim)
    first = 0
    for b, (new, length) in enumerate(zip(news, lengths)):
        ids = s["table"][b, :(length + page - 1) // page].long()
        for h in range(kv):
            k = (s["pool"][0][ids, h].double() * s["pool"][1][ids, h].double()[..., None]).reshape(-1, dim)[:length]
            v = (s["pool"][2][ids, h].double() * s["pool"][3][ids, h].double()[..., None]).reshape(-1, dim)[:length]
            for lo in range(0, new, 512):
                hi = min(new, lo + 512)
                heads = slice(h * group, (h + 1) * group)
                t = torch.einsum("igd,jd->igj", q[first + lo:first + hi, heads].double(), k) * s["scale"]
                if case["causal"]:
                    last = torch.arange(lo, hi, device=t.device) + length - new
                    t.masked_fill_(torch.arange(length, device=t.device)[None, None] > last[:, None, None], -math.inf)
                out[first + lo:first + hi, heads] = torch.softmax(t, -1) @ v
        first += new
    return out.view(-1, case["heads"] * dim)
