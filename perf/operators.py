"""Measured cases of the attention and key/value-cache operators.

Four operators, each in its plain form (elementary torch operations in 32 bits,
rounded once) and as a call of the package's entry point:

* ``prompt``: softmax attention over whole prompts, packed or padded, causal or
  not, with grouped heads (``cta_b200.attention.prompt_attention``);
* ``train``:  the same with its gradients, as a training step takes them;
* ``cache``:  new keys and values quantised to e4m3, with one scale per token
  and head, as they are written into a paged cache, and read back
  (``cta_b200.ops.kv_cache_write`` / ``kv_cache_read``);
* ``paged``:  attention of the newest tokens of each sequence over such a cache
  (``cta_b200.ops.paged_attention``).
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0
#: a token whose largest magnitude is below this is quantised as if it were this
LEAST_MAX = 2.0**-100


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # three short prompts of an idle server: one launch's latency
        dict(name="prompt_short", op="prompt", packed=True, batch=3, low=1, high=90, heads=8, kv_heads=8, dim=64,
             causal=True, dtype="bf16"),
        # a prefill batch: ragged prompts packed without padding, grouped heads
        dict(name="prompt_ragged", op="prompt", packed=True, batch=24, low=16, high=2048, heads=32, kv_heads=8,
             dim=128, causal=True, dtype="bf16"),
        # the language model in its default type: a padded batch, causal
        dict(name="train_lm_fp32", op="train", packed=False, batch=4, low=300, high=512, heads=8, kv_heads=8, dim=64,
             causal=True, dtype="fp32"),
        # the classifier: a padded batch, every token sees every valid one
        dict(name="train_classifier", op="train", packed=False, batch=16, low=100, high=512, heads=8, kv_heads=8,
             dim=64, causal=False, dtype="bf16"),
        # the language model's benchmark block at its largest length
        dict(name="train_lm_long", op="train", packed=False, batch=1, low=16384, high=16384, heads=8, kv_heads=8,
             dim=64, causal=True, dtype="bf16"),
        # documents of different lengths packed into one row, grouped heads
        dict(name="train_packed", op="train", packed=True, batch=6, low=200, high=3000, heads=32, kv_heads=8, dim=128,
             causal=True, dtype="bf16"),
        # one decode step of one layer for a batch of 64: the cache write alone, latency
        dict(name="cache_step", op="cache", tokens=64, heads=8, dim=128, page=16, dtype="bf16"),
        # a prefill batch's keys and values
        dict(name="cache_prefill", op="cache", tokens=16384, heads=8, dim=128, page=64, dtype="bf16"),
        # one sequence, one new token: latency
        dict(name="decode_one", op="paged", batch=1, rows=1, low=777, high=777, heads=32, kv_heads=8, dim=128,
             page=16, cache="bf16", dtype="bf16"),
        # a decode step of a full batch over a 16-bit cache
        dict(name="decode_batch", op="paged", batch=64, rows=1, low=512, high=8192, heads=32, kv_heads=8, dim=128,
             page=16, cache="bf16", dtype="bf16"),
        # the same over an e4m3 cache
        dict(name="decode_batch_e4m3", op="paged", batch=64, rows=1, low=512, high=8192, heads=32, kv_heads=8,
             dim=128, page=64, cache="e4m3", dtype="bf16"),
        # chunks of long prompts over what the cache already holds of them
        dict(name="chunk", op="paged", batch=4, rows=512, low=1500, high=8192, heads=32, kv_heads=8, dim=128, page=64,
             cache="bf16", dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prompt", "train", "train", "cache", "paged", "paged"])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
    if op == "cache":
        return dict(op=op, tokens=_log(rng, 1, 16384), heads=rng.choice([1, 2, 4, 8]), dim=dim,
                    page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "fp16"]))
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4])
    if op == "paged":
        # rows: one token, a few speculated ones, a chunk
        rows = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 16, 512)])
        high = max(rows, _log(rng, 16, 8192))
        batch = max(1, min(_log(rng, 1, 64), 64 * 8192 // (high * min(rows, 16))))
        cache = rng.choice(["e4m3", "same"])
        dtype = rng.choice(["bf16", "fp16"])
        return dict(op=op, batch=batch, rows=rows, low=max(rows, high // rng.choice([1, 3, 12])), high=high,
                    heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]),
                    cache=dtype if cache == "same" else cache, dtype=dtype)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    high = _log(rng, 1, 1024 if dtype == "fp32" else 4096)
    # no more work than the largest listed case
    batch = max(1, min(_log(rng, 1, 24), (1 << 35) // (high * high * heads * dim)))
    return dict(op=op, packed=rng.random() < 0.5, batch=batch, low=max(1, high // rng.choice([1, 2, 8])), high=high,
                heads=heads, kv_heads=kv_heads, dim=dim, causal=rng.random() < 0.7, dtype=dtype)


def _lengths(case):
    """The sequences' lengths: a part of the case, the same for every seed."""
    rng = random.Random(case["batch"] * 1000003 + case["low"] * 8191 + case["high"])
    n = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    n[rng.randrange(len(n))] = case["high"]
    return n


def work(case):
    d = case["dim"]
    if case["op"] == "cache":
        # read k, v; write the codes and scales; read them back; write k, v
        n = 2 * case["tokens"] * case["heads"]
        return {"bytes": n * (2 * d + 2 * (d + 4) + 2 * d) + 2 * 8 * case["tokens"], "flops": 4 * n * d}
    lengths = _lengths(case)
    h, hk = case["heads"], case["kv_heads"]
    if case["op"] == "paged":
        rows = case["rows"]
        size = d + 4 if case["cache"] == "e4m3" else 2 * d
        pairs = sum(rows * n - rows * (rows - 1) // 2 for n in lengths)
        table = sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": 2 * hk * size * sum(lengths) + 4 * table + 2 * 2 * d * h * rows * len(lengths),
                "flops": 4 * d * h * pairs}
    size = 4 if case["dtype"] == "fp32" else 2
    rows = sum(lengths) if case["packed"] else case["high"] * case["batch"]
    if case["causal"]:
        pairs = sum(n * (n + 1) // 2 for n in lengths)
        # the padding's rows come back too, and see every valid key
        pairs += 0 if case["packed"] else sum((case["high"] - n) * n for n in lengths)
    else:
        pairs = sum(n * (n if case["packed"] else case["high"]) for n in lengths)
    once = rows * d * size
    if case["op"] == "prompt":
        return {"bytes": once * (2 * h + 2 * hk), "flops": 4 * d * h * pairs}
    return {"bytes": once * (4 * h + 4 * hk), "flops": 14 * d * h * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dt=dtype):
        return torch.randn(*shape, device=dev, dtype=torch.float32, generator=gen).to(dt)

    s = {"op": case["op"], "case": case, "dtype": dtype}
    d = case["dim"]
    if case["op"] == "cache":
        tokens, page, heads = case["tokens"], case["page"], case["heads"]
        pages = -(-tokens // page) + 3
        # tokens of a model differ in size by orders of magnitude
        size = torch.exp(1.5 * torch.randn(2, tokens, heads, 1, device=dev, generator=gen))
        s["k"], s["v"] = (normal(tokens, heads, d, dt=torch.float32) * x for x in size)
        s["k"], s["v"] = s["k"].to(dtype), s["v"].to(dtype)
        s["slots"] = torch.randperm(pages * page, device=dev, generator=gen)[:tokens].contiguous()
        for n in ("k", "v"):
            s[n + "_cache"] = torch.zeros(pages, page, heads, d, device=dev, dtype=torch.float8_e4m3fn)
            s[n + "_scale"] = torch.zeros(pages, heads, page, device=dev, dtype=torch.float32)
        return s
    h, hk = case["heads"], case["kv_heads"]
    lengths = _lengths(case)
    s["lengths"] = lengths
    s["scale"] = 1.0 / math.sqrt(d)
    starts = [0]
    if case["op"] == "paged":
        page, rows = case["page"], case["rows"]
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts) + 2
        order = torch.randperm(pages, device=dev, generator=gen).to(torch.int32)
        table = torch.zeros(len(lengths), max(counts), dtype=torch.int32, device=dev)
        where = torch.arange(max(counts), device=dev)
        n_pages = torch.tensor(counts, device=dev)
        first = torch.cumsum(n_pages, 0) - n_pages
        used = where[None, :] < n_pages[:, None]
        s["table"] = torch.where(used, order[(first[:, None] + where[None, :]).clamp(max=pages - 1)], table)
        s["seq_lens"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        s["cu"] = torch.arange(0, rows * len(lengths) + 1, rows, dtype=torch.int32, device=dev) if rows > 1 else None
        s["q"] = normal(rows * len(lengths), h, d)
        for n in ("k", "v"):
            x = normal(pages, page, hk, d)
            s[n + "_scale"] = None
            if case["cache"] == "e4m3":
                x, s[n + "_scale"] = _quantised(x)
                s[n + "_scale"] = s[n + "_scale"].transpose(1, 2).contiguous()
            s[n + "_cache"] = x
        return s
    if case["packed"]:
        for n in lengths:
            starts.append(starts[-1] + n)
        shape = (starts[-1],)
        s["cu"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        # the plan of the plain form: each row's sequence and place in it
        n = torch.tensor(lengths, device=dev)
        s["seq"] = torch.repeat_interleave(torch.arange(len(lengths), device=dev), n)
        s["place"] = torch.arange(starts[-1], device=dev) - s["cu"][:-1].long()[s["seq"]]
        s["mask"] = None
    else:
        shape = (case["batch"], case["high"])
        s["cu"] = None
        n = torch.tensor(lengths, device=dev)
        whole = min(lengths) == case["high"]
        s["mask"] = None if whole else (torch.arange(case["high"], device=dev)[None, :] < n[:, None])
    train = case["op"] == "train"
    for name, heads in (("q", h), ("k", hk), ("v", hk)):
        s[name] = normal(*shape, heads, d).requires_grad_(train)
    if train:
        s["grad"] = normal(*shape, h, d)
    return s


def _quantised(x):
    """e4m3 codes with one 32-bit scale per token and head."""
    x = x.float()
    most = x.abs().amax(dim=-1).clamp_min(LEAST_MAX)
    codes = (x * (E4M3_MAX / most)[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes, most / E4M3_MAX


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    return {"cache": _plain_cache, "paged": _plain_paged, "prompt": _plain_prompt, "train": _plain_train}[
        state["op"]](state)


def _own(s):
    root = os.path.join(os.getcwd(), "continuous-time-attention_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from cta_b200 import ops
    from cta_b200.attention import prompt_attention

    case = s["case"]
    if s["op"] == "cache":
        ops.kv_cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"],
                           v_scale=s["v_scale"])
        return ops.kv_cache_read(s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                 dtype=s["dtype"])
    if s["op"] == "paged":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"],
                                   cu_seqlens=s["cu"], max_rows=case["rows"], k_scale=s["k_scale"],
                                   v_scale=s["v_scale"])
    out = prompt_attention(s["q"], s["k"], s["v"], causal=case["causal"], key_mask=s["mask"], cu_seqlens=s["cu"])
    if s["op"] == "prompt":
        return out
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"]))


def _plain_cache(s):
    slots = s["slots"]
    at = (slots // s["case"]["page"], slice(None), slots % s["case"]["page"])
    back = []
    for n in ("k", "v"):
        codes, scale = _quantised(s[n])
        flat = s[n + "_cache"].view(torch.uint8).flatten(0, 1)
        flat[slots] = codes.view(torch.uint8)
        s[n + "_scale"][at] = scale
        read = flat[slots].view(torch.float8_e4m3fn).float() * s[n + "_scale"][at][..., None]
        back.append(read.to(s["dtype"]))
    return tuple(back)


def _weights(q, k, allowed):
    """softmax over the allowed keys; a row that is allowed none has no weights.
    q [B, Hk, rows, d] (scaled), k [B, Hk, keys, d], allowed broadcasts to [B, Hk, rows, keys]."""
    x = torch.matmul(q, k.transpose(-1, -2))
    x.masked_fill_(~allowed, float("-inf"))
    most = x.amax(dim=-1, keepdim=True)
    most.masked_fill_(most == float("-inf"), 0.0)
    x.sub_(most).exp_()
    total = x.sum(dim=-1, keepdim=True)
    return x.div_(total.masked_fill(total == 0, 1.0))


def _grouped(x, hk):
    """[B, L, H, d] -> [B, Hk, G * L, d]: the rows of the heads that share keys, one after another."""
    b, n, h, d = x.shape
    return x.reshape(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, h // hk * n, d)


def _ungrouped(x, h):
    b, hk, rows, d = x.shape
    g = h // hk
    return x.reshape(b, hk, g, rows // g, d).permute(0, 3, 1, 2, 4).reshape(b, rows // g, h, d)


def _padded(s, names):
    """The tensors as [B, Lmax, H, d] in 32 bits (zeros behind each sequence), and which keys are valid."""
    if s["cu"] is None:
        x = [s[n].detach().float() for n in names]
        valid = s["mask"] if s["mask"] is not None else torch.ones(x[0].shape[:2], dtype=torch.bool,
                                                                   device=x[0].device)
        return x, valid
    longest = s["case"]["high"]
    place = torch.arange(longest, device=s["cu"].device)
    n = (s["cu"][1:] - s["cu"][:-1])[:, None]
    valid = place[None, :] < n
    rows = (s["cu"][:-1, None].long() + place[None, :]).clamp(max=s["q"].shape[0] - 1)
    return [s[k].detach().float()[rows] * valid[:, :, None, None] for k in names], valid


def _packed(s, x):
    return x if s["cu"] is None else x[s["seq"], s["place"]]


def _allowed(s, valid):
    g = s["case"]["heads"] // s["case"]["kv_heads"]
    a = valid[:, None, None, :]
    if s["case"]["causal"]:
        n = valid.shape[1]
        i = torch.arange(n, device=valid.device)
        a = a & (i[None, :] <= i[:, None]).repeat(g, 1)[None, None]
    return a


def _plain_prompt(s):
    (q, k, v), valid = _padded(s, ("q", "k", "v"))
    h, hk = s["case"]["heads"], s["case"]["kv_heads"]
    w = _weights(_grouped(q, hk) * s["scale"], k.transpose(1, 2), _allowed(s, valid))
    return _packed(s, _ungrouped(torch.matmul(w, v.transpose(1, 2)), h)).to(s["dtype"])


def _plain_train(s):
    (q, k, v, grad), valid = _padded(s, ("q", "k", "v", "grad"))
    h, hk = s["case"]["heads"], s["case"]["kv_heads"]
    q, k, v, grad = _grouped(q, hk) * s["scale"], k.transpose(1, 2), v.transpose(1, 2), _grouped(grad, hk)
    w = _weights(q, k, _allowed(s, valid))
    out = torch.matmul(w, v)
    dv = torch.matmul(w.transpose(-1, -2), grad)
    dx = torch.matmul(grad, v.transpose(-1, -2))
    dx.sub_((grad * out).sum(dim=-1, keepdim=True)).mul_(w)
    dq = torch.matmul(dx, k) * s["scale"]
    dk = torch.matmul(dx.transpose(-1, -2), q)
    back = [_ungrouped(out, h), _ungrouped(dq, h), dk.transpose(1, 2), dv.transpose(1, 2)]
    return tuple(_packed(s, x).to(s["dtype"]) for x in back)


def _plain_paged(s):
    case = s["case"]
    h, hk, rows = case["heads"], case["kv_heads"], case["rows"]
    got = []
    for n in ("k", "v"):
        # the pages of each sequence, in order
        x = s[n + "_cache"]
        if s[n + "_scale"] is not None:
            x = x.view(torch.uint8)[s["table"].long()].view(torch.float8_e4m3fn).float()
            x = x * s[n + "_scale"][s["table"].long()].transpose(2, 3)[..., None]
        else:
            x = x[s["table"].long()].float()
        got.append(x.flatten(1, 2).transpose(1, 2))
    k, v = got
    q = s["q"].float().reshape(-1, rows, h, case["dim"])
    j = torch.arange(k.shape[2], device=q.device)
    last = s["seq_lens"][:, None] - rows + torch.arange(rows, device=q.device)[None, :]
    allowed = (j[None, None, :] <= last[:, :, None]).repeat(1, h // hk, 1)[:, None]
    w = _weights(_grouped(q, hk) * s["scale"], k, allowed)
    return _ungrouped(torch.matmul(w, v), h).reshape(-1, h, case["dim"]).to(s["dtype"])


# ---------------------------------------------------------------------------
# the definition, in 64 bits: sequence by sequence and head by head
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cache":
        both = []
        for n in ("k", "v"):
            x = s[n].double()
            most = torch.maximum(x.abs().max(dim=-1, keepdim=True).values, torch.tensor(LEAST_MAX).double().cuda())
            both.append(_nearest_e4m3(x * E4M3_MAX / most) * most / E4M3_MAX)
        return tuple(both)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    group = h // hk
    if case["op"] == "paged":
        rows, page = case["rows"], case["page"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lengths"]):
            pages = s["table"][b, : -(-n // page)].long()
            full = {}
            for x in ("k", "v"):
                c = s[x + "_cache"]
                if s[x + "_scale"] is None:
                    c = c[pages].double()
                else:
                    c = c.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
                    c = c * s[x + "_scale"][pages].double().transpose(1, 2)[..., None]
                full[x] = c.reshape(-1, hk, d)[:n]
            i = torch.arange(n - rows, n, device="cuda")
            see = torch.arange(n, device="cuda")[None, :] <= i[:, None]
            for a in range(h):
                q = s["q"][b * rows : (b + 1) * rows, a].double()
                w = _row_softmax(torch.einsum("id,jd->ij", q, full["k"][:, a // group]) / math.sqrt(d), see)
                out[b * rows : (b + 1) * rows, a] = w @ full["v"][:, a // group]
        return out
    names = ("q", "k", "v") + (("grad",) if case["op"] == "train" else ())
    x = {n: s[n].detach().double() for n in names}
    res = {n: torch.zeros_like(x["q" if n in ("o", "dq") else "k"]) for n in ("o", "dq", "dk", "dv")}
    begin = 0
    for b, n in enumerate(s["lengths"]):
        if case["packed"]:
            part = (slice(begin, begin + n),)
            begin += n
            rows = keys = n
        else:
            part, rows, keys = (b,), case["high"], n
        see = torch.ones(rows, keys, dtype=torch.bool, device="cuda")
        if case["causal"]:
            see = see.tril()
        for a in range(h):
            c = a // group
            q = x["q"][part][:, a]
            k, v = x["k"][part][:keys, c], x["v"][part][:keys, c]
            w = _row_softmax(q @ k.T / math.sqrt(d), see)
            o = w @ v
            res["o"][part][:, a] = o
            if case["op"] == "train":
                g = x["grad"][part][:, a]
                res["dv"][part][:keys, c] += w.T @ g
                dx = w * (g @ v.T - (g * o).sum(1, keepdim=True)) / math.sqrt(d)
                res["dq"][part][:, a] = dx @ k
                res["dk"][part][:keys, c] += dx.T @ q
    return res["o"] if case["op"] == "prompt" else (res["o"], res["dq"], res["dk"], res["dv"])


def _row_softmax(x, see):
    """Weights of each row over the keys it sees (at least one)."""
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    x = torch.exp(x - x.max(dim=1, keepdim=True).values)
    return x / x.sum(dim=1, keepdim=True)


def _nearest_e4m3(x):
    """x (64 bits, magnitude at most 448) rounded to 3 fraction bits, ties to even, exponents from -6."""
    size = x.abs().clamp_min(2.0**-6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    # log2 of a value just below a power of two may round up to it
    step = torch.where(size < step * 8, step / 2, step)
    return torch.round(x / step) * step
