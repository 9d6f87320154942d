"""Measured cases of window attention, shared prefixes and the rotated cache write.

Five operators, each in its plain form (elementary torch operations in 32 bits,
rounded once) and as a call of the package's entry point:

* ``prompt``: causal softmax attention over whole prompts, packed or padded, in
  which a row sees the last ``window`` tokens, itself included, and the first
  ``sinks`` ones (``cta_b200.attention.prompt_attention``);
* ``train``:  the same with its gradients, as a training step takes them;
* ``paged``:  attention of the newest tokens of each sequence over a paged cache
  under the same mask (``cta_b200.ops.paged_attention``);
* ``prefix``: attention of the newest tokens of a batch whose sequences all
  begin with the same long prefix, which lies in the cache once (the same
  entry point);
* ``rotate``: queries and new keys rotated by their positions, keys and values
  written into a paged cache (``cta_b200.ops.rotary_cache_write``), and read
  back where the cache holds e4m3.
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
        # three short prompts of an idle server, one of them longer than the window: one launch's latency
        dict(name="prompt_short", op="prompt", packed=True, batch=3, low=1, high=90, heads=8, kv_heads=8, dim=64,
             window=32, sinks=4, dtype="bf16"),
        # a prefill batch: ragged prompts packed without padding, grouped heads
        dict(name="prompt_ragged", op="prompt", packed=True, batch=12, low=16, high=4096, heads=32, kv_heads=8,
             dim=128, window=512, sinks=4, dtype="bf16"),
        # the language model in its default type: a padded batch, no sinks
        dict(name="train_lm_fp32", op="train", packed=False, batch=4, low=300, high=512, heads=8, kv_heads=8, dim=64,
             window=128, sinks=0, dtype="fp32"),
        # the language model's benchmark block at its largest length
        dict(name="train_lm_long", op="train", packed=False, batch=1, low=16384, high=16384, heads=8, kv_heads=8,
             dim=64, window=1024, sinks=4, dtype="bf16"),
        # documents of different lengths packed into one row, grouped heads, a window of an odd size
        dict(name="train_packed", op="train", packed=True, batch=6, low=200, high=5000, heads=32, kv_heads=8, dim=128,
             window=500, sinks=16, dtype="fp16"),
        # a decode step of a full batch over a 16-bit cache
        dict(name="decode_batch", op="paged", batch=64, rows=1, low=512, high=8192, heads=32, kv_heads=8, dim=128,
             page=16, window=1024, sinks=4, cache="bf16", dtype="bf16"),
        # chunks of long prompts over what an e4m3 cache already holds of them
        dict(name="chunk_e4m3", op="paged", batch=4, rows=512, low=1500, high=8192, heads=32, kv_heads=8, dim=128,
             page=64, window=1024, sinks=4, cache="e4m3", dtype="bf16"),
        # a few requests behind a system prompt: latency
        dict(name="prefix_few", op="prefix", batch=6, rows=1, prefix=2048, low=1, high=100, heads=32, kv_heads=8,
             dim=128, page=16, cache="bf16", dtype="bf16"),
        # a decode step of a full batch behind one long document
        dict(name="prefix_batch", op="prefix", batch=64, rows=1, prefix=8192, low=16, high=1024, heads=32, kv_heads=8,
             dim=128, page=16, cache="bf16", dtype="bf16"),
        # many samples of one longer prompt over an e4m3 cache
        dict(name="prefix_many_e4m3", op="prefix", batch=128, rows=1, prefix=16384, low=16, high=512, heads=32,
             kv_heads=8, dim=128, page=64, cache="e4m3", dtype="fp16"),
        # one decode step of one layer for a batch of 64: latency
        dict(name="rotate_step", op="rotate", tokens=64, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False,
             positions=32768, page=16, cache="bf16", dtype="bf16"),
        # a prefill batch into an e4m3 cache
        dict(name="rotate_prefill", op="rotate", tokens=16384, heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, positions=8192, page=64, cache="e4m3", dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prompt", "train", "train", "paged", "paged", "prefix", "prefix", "rotate"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    cache = rng.choice([dtype, "e4m3"])
    if op == "rotate":
        return dict(op=op, tokens=_log(rng, 1, 16384), heads=heads, kv_heads=kv_heads, dim=dim,
                    rotary=rng.choice([dim, dim, 16, dim // 32 * 16]), interleaved=rng.random() < 0.4,
                    positions=_log(rng, 64, 131072), page=page, cache=cache, dtype=dtype)
    if op == "prefix":
        rows = rng.choice([1, 1, 1, rng.randint(2, 4)])
        prefix = -(-_log(rng, 16, 16384) // page) * page
        high = max(rows, _log(rng, 1, 1024))
        batch = max(2, min(_log(rng, 2, 128), 128 * 16384 // (prefix + high)))
        return dict(op=op, batch=batch, rows=rows, prefix=prefix, low=max(rows, high // rng.choice([1, 3, 12])),
                    high=high, heads=heads, kv_heads=kv_heads, dim=dim, page=page, cache=cache, dtype=dtype)
    sinks = rng.choice([0, 0, 1, 4, 4, 16, 64, rng.randint(1, 300)])
    if op == "paged":
        # rows: one token, a few speculated ones, a chunk
        rows = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 16, 512)])
        high = max(rows, _log(rng, 16, 8192))
        batch = max(1, min(_log(rng, 1, 64), 64 * 8192 // (high * min(rows, 16))))
        return dict(op=op, batch=batch, rows=rows, low=max(rows, high // rng.choice([1, 3, 12])), high=high,
                    heads=heads, kv_heads=kv_heads, dim=dim, page=page, window=_log(rng, 1, 4096), sinks=sinks,
                    cache=cache, dtype=dtype)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    high = _log(rng, 1, 1024 if dtype == "fp32" else 4096)
    # no more work than the largest listed case
    batch = max(1, min(_log(rng, 1, 24), (1 << 35) // (high * high * heads * dim)))
    return dict(op=op, packed=rng.random() < 0.5, batch=batch, low=max(1, high // rng.choice([1, 2, 8])), high=high,
                heads=heads, kv_heads=kv_heads, dim=dim, window=_log(rng, 1, 2048), sinks=sinks, dtype=dtype)


def _lengths(case):
    """The sequences' lengths (behind the prefix, where there is one): a part of the case, the same for every seed."""
    rng = random.Random(case["batch"] * 1000003 + case["low"] * 8191 + case["high"])
    n = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    n[rng.randrange(len(n))] = case["high"]
    return n


def _padding(case):
    """Rows at the end of a rotated batch that fill it up and go nowhere."""
    return case["tokens"] // 16


def _seen(i, keys, window, sinks):
    """How many of `keys` keys the row at place i sees."""
    last = min(i, keys - 1)
    first = max(0, i - window + 1)
    return max(0, last - first + 1) + max(0, min(sinks, first, keys))


def work(case):
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "rotate":
        tokens, live = case["tokens"], case["tokens"] - _padding(case)
        size = 2 * d if case["cache"] != "e4m3" else d + 4
        once = tokens * 2 * d * 2 * h + live * 2 * hk * (2 * d + size) + tokens * (16 + 4 * case["rotary"])
        if case["cache"] == "e4m3":
            # read back: codes and scales, and both tensors written
            once += live * 2 * hk * size + tokens * 2 * hk * 2 * d
        return {"bytes": once, "flops": 3 * tokens * (h + hk) * case["rotary"]}
    lengths = _lengths(case)
    if case["op"] in ("paged", "prefix"):
        rows = case["rows"]
        size = d + 4 if case["cache"] == "e4m3" else 2 * d
        if case["op"] == "prefix":
            keys = case["prefix"] + sum(lengths)
            pairs = sum(rows * (case["prefix"] + n) - rows * (rows - 1) // 2 for n in lengths)
        else:
            w, s = case["window"], case["sinks"]
            keys = sum(min(n, w + rows - 1 + min(s, max(0, n - w - rows + 1))) for n in lengths)
            pairs = sum(_seen(i, n, w, s) for n in lengths for i in range(n - rows, n))
        return {"bytes": 2 * hk * size * keys + 4 * (keys // case["page"]) + 2 * 2 * d * h * rows * len(lengths),
                "flops": 4 * d * h * pairs}
    size = 4 if case["dtype"] == "fp32" else 2
    w, s = case["window"], case["sinks"]
    if case["packed"]:
        rows = sum(lengths)
        pairs = sum(_seen(i, n, w, s) for n in lengths for i in range(n))
    else:
        # the padding's rows come back too, and see what valid keys their windows reach
        rows = case["high"] * case["batch"]
        pairs = sum(_seen(i, n, w, s) for n in lengths for i in range(case["high"]))
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
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "rotate":
        return _prepare_rotate(s, case, gen, normal)
    lengths = _lengths(case)
    s["lengths"] = lengths
    s["scale"] = 1.0 / math.sqrt(d)
    if case["op"] in ("paged", "prefix"):
        page, rows, shared = case["page"], case["rows"], case.get("prefix", 0) // case["page"]
        counts = [-(-n // page) for n in lengths]
        pages = shared + sum(counts) + 2
        order = torch.randperm(pages, device=dev, generator=gen).to(torch.int32)
        where = torch.arange(max(counts), device=dev)
        n_pages = torch.tensor(counts, device=dev)
        first = shared + torch.cumsum(n_pages, 0) - n_pages
        used = where[None, :] < n_pages[:, None]
        table = torch.zeros(len(lengths), max(counts), dtype=torch.int32, device=dev)
        table = torch.where(used, order[(first[:, None] + where[None, :]).clamp(max=pages - 1)], table)
        if shared:
            table = torch.cat([order[:shared].expand(len(lengths), shared), table], dim=1).contiguous()
        s["table"] = table
        s["total"] = [shared * page + n for n in lengths]
        s["seq_lens"] = torch.tensor(s["total"], dtype=torch.int32, device=dev)
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
        starts = [0]
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


def _prepare_rotate(s, case, gen, normal):
    dev, d, page, tokens = gen.device, case["dim"], case["page"], case["tokens"]
    pages = -(-tokens // page) + 3
    # tokens of a model differ in size by orders of magnitude
    size = torch.exp(1.5 * torch.randn(2, tokens, case["kv_heads"], 1, device=dev, generator=gen))
    s["q"] = normal(tokens, case["heads"], d)
    s["k"], s["v"] = ((normal(tokens, case["kv_heads"], d, dt=torch.float32) * x).to(s["dtype"]) for x in size)
    s["live"] = tokens - _padding(case)
    s["slots"] = torch.randperm(pages * page, device=dev, generator=gen)[:tokens].contiguous()
    s["slots"][s["live"]:] = -1
    s["positions"] = torch.randint(0, case["positions"], (tokens,), device=dev, generator=gen)
    # the table of the model: cosines, then sines, of position / 10000^(2 i / rotary)
    half = case["rotary"] // 2
    turn = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
    angle = torch.arange(case["positions"], dtype=torch.float64, device=dev)[:, None] * turn[None, :]
    s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
    quantised = case["cache"] == "e4m3"
    for n in ("k", "v"):
        s[n + "_cache"] = torch.zeros(pages, page, case["kv_heads"], d, device=dev,
                                      dtype=torch.float8_e4m3fn if quantised else s["dtype"])
        s[n + "_scale"] = torch.zeros(pages, case["kv_heads"], page, device=dev) if quantised else None
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
    return {"prompt": _plain_prompt, "train": _plain_train, "paged": _plain_paged, "prefix": _plain_paged,
            "rotate": _plain_rotate}[state["op"]](state)


def _own(s):
    root = os.path.join(os.getcwd(), "continuous-time-attention_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from cta_b200 import ops
    from cta_b200.attention import prompt_attention

    case = s["case"]
    if s["op"] == "rotate":
        q = ops.rotary_cache_write(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["positions"],
                                   s["cos_sin"], interleaved=case["interleaved"], k_scale=s["k_scale"],
                                   v_scale=s["v_scale"])
        if s["k_scale"] is None:
            return q, s["k_cache"], s["v_cache"]
        return (q, *ops.kv_cache_read(s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"],
                                      v_scale=s["v_scale"], dtype=s["dtype"]))
    if s["op"] == "paged":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"],
                                   cu_seqlens=s["cu"], max_rows=case["rows"], k_scale=s["k_scale"],
                                   v_scale=s["v_scale"], window=case["window"], sinks=case["sinks"])
    if s["op"] == "prefix":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"],
                                   cu_seqlens=s["cu"], max_rows=case["rows"], k_scale=s["k_scale"],
                                   v_scale=s["v_scale"], shared_prefix=case["prefix"])
    out = prompt_attention(s["q"], s["k"], s["v"], causal=True, window=case["window"], sinks=case["sinks"],
                           key_mask=s["mask"], cu_seqlens=s["cu"])
    if s["op"] == "prompt":
        return out
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"]))


def _turned(x, cos, sin, interleaved):
    """x [T, heads, dim] in 32 bits, its first elements rotated pair by pair; cos, sin [T, 1, pairs]."""
    x = x.float()
    pairs = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0 : 2 * pairs : 2], x[..., 1 : 2 * pairs : 2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs : 2 * pairs]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., 2 * pairs :]], dim=-1)


def _plain_rotate(s):
    case = s["case"]
    cos, sin = s["cos_sin"][s["positions"]][:, None].chunk(2, dim=-1)
    q = _turned(s["q"], cos, sin, case["interleaved"]).to(s["dtype"])
    k = _turned(s["k"], cos, sin, case["interleaved"])
    slots = s["slots"][: s["live"]]
    at = (slots // case["page"], slice(None), slots % case["page"])
    back = []
    for n, x in (("k", k), ("v", s["v"])):
        if s["k_scale"] is None:
            s[n + "_cache"].flatten(0, 1)[slots] = x[: s["live"]].to(s["dtype"])
            continue
        codes, scale = _quantised(x[: s["live"]])
        flat = s[n + "_cache"].view(torch.uint8).flatten(0, 1)
        flat[slots] = codes.view(torch.uint8)
        s[n + "_scale"][at] = scale
        read = torch.zeros_like(x, dtype=s["dtype"])
        read[: s["live"]] = (flat[slots].view(torch.float8_e4m3fn).float() * s[n + "_scale"][at][..., None]).to(s["dtype"])
        back.append(read)
    return (q, *back) if back else (q, s["k_cache"], s["v_cache"])


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


def _in_reach(i, j, case):
    """Whether rows at places i see keys j."""
    return (j <= i) & ((j > i - case["window"]) | (j < case["sinks"]))


def _allowed(s, valid):
    g = s["case"]["heads"] // s["case"]["kv_heads"]
    i = torch.arange(valid.shape[1], device=valid.device)
    reach = _in_reach(i[:, None], i[None, :], s["case"]).repeat(g, 1)
    return valid[:, None, None, :] & reach[None, None]


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
    j = torch.arange(k.shape[2], device=q.device)[None, None, :]
    i = (s["seq_lens"][:, None] - rows + torch.arange(rows, device=q.device)[None, :])[:, :, None]
    allowed = (_in_reach(i, j, case) if case["op"] == "paged" else j <= i).repeat(1, h // hk, 1)[:, None]
    w = _weights(_grouped(q, hk) * s["scale"], k, allowed)
    return _ungrouped(torch.matmul(w, v), h).reshape(-1, h, case["dim"]).to(s["dtype"])


# ---------------------------------------------------------------------------
# the definition, in 64 bits: sequence by sequence and head by head
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(case, s)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    group = h // hk

    def reach(first, rows, keys):
        i = torch.arange(first, first + rows, device="cuda")[:, None]
        j = torch.arange(keys, device="cuda")[None, :]
        see = j <= i
        if "window" in case:
            see &= (i - j < case["window"]) | (j < case["sinks"])
        return see

    if case["op"] in ("paged", "prefix"):
        rows, page = case["rows"], case["page"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["total"]):
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
            see = reach(n - rows, rows, n).repeat(group, 1)
            for c in range(hk):
                q = s["q"][b * rows : (b + 1) * rows, c * group : (c + 1) * group].double()
                q = q.transpose(0, 1).reshape(group * rows, d)
                w = _row_softmax(q @ full["k"][:, c].T / math.sqrt(d), see) @ full["v"][:, c]
                out[b * rows : (b + 1) * rows, c * group : (c + 1) * group] = w.reshape(group, rows, d).transpose(0, 1)
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
        see = reach(0, rows, keys)
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
    """Weights of each row over the keys it sees; none where it sees none."""
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    most = x.max(dim=1, keepdim=True).values
    x = torch.exp(x - torch.where(torch.isinf(most), torch.zeros_like(most), most))
    total = x.sum(dim=1, keepdim=True)
    return x / torch.where(total == 0, torch.ones_like(total), total)


def _exact_rotate(case, s):
    pairs = case["rotary"] // 2
    table = s["cos_sin"].double()[s["positions"]]

    def turn(x):
        y = x.double().clone()
        for i in range(pairs):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + pairs)
            c, t = table[:, i, None], table[:, pairs + i, None]
            p, q = x[..., a].double(), x[..., b].double()
            y[..., a] = p * c - q * t
            y[..., b] = q * c + p * t
        return y

    live, page, both = s["live"], case["page"], []
    for n, x in (("k", turn(s["k"])), ("v", s["v"].double())):
        if case["cache"] == "e4m3":
            x[live:] = 0
            most = torch.maximum(x.abs().max(dim=-1, keepdim=True).values, torch.tensor(LEAST_MAX).double().cuda())
            both.append(_nearest_e4m3(x * E4M3_MAX / most) * most / E4M3_MAX)
        else:
            cache = torch.zeros(s[n + "_cache"].shape, dtype=torch.float64, device="cuda")
            slots = s["slots"][:live]
            cache[slots // page, slots % page] = x[:live]
            both.append(cache)
    return (turn(s["q"]), *both)


def _nearest_e4m3(x):
    """x (64 bits, magnitude at most 448) rounded to 3 fraction bits, ties to even, exponents from -6."""
    size = x.abs().clamp_min(2.0**-6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    # log2 of a value just below a power of two may round up to it
    step = torch.where(size < step * 8, step / 2, step)
    return torch.round(x / step) * step
