"""The operators of the 8-bit key/value cache, as cases that can be run and timed: the decode step, the prompt phase, the
read-back and the eviction by accumulated attention weight, each in a plain form (elementary torch operations) and through
fasterllama_amd.kv8.

The cache of one layer: K and V rows as 8-bit integers [B, H, L, D] with one float scale per block of `block` consecutive
rows and head, [B, H, L/block]; the rows of the block that is not full yet stay in fp16 in a tail [B, H, block, D] and are
quantised together when its last row arrives.  A stored value's rounding is part of the definition, since one step of it
decides about the next: a rotated key is fma(x0, c, -(x1 s)), fma(x1, c, x0 s) in 32 bits, then x -> fp16 (a non-finite value
becomes 0, a finite one is kept within +-65504); block scale = absmax/127 and integer = rint(x * (127/absmax)), each quotient
and product in 32 bits.  Attention reads the cache as it stands after the new rows are in.  Optionally every block gathers the softmax weight its rows receive, and the eviction keeps the
blocks that gathered most, beside the most recent ones.
"""
import math

import numpy as np
import torch

own = False  # True: run() goes through the framework's kernels

NEG = -3.4028234663852886e38  # what the reference driver's masks hold
FLOOR = -1e9                  # the softmax's maximum starts here


# ------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # The decode step.
        # The first configuration's heads: one short sequence in fp32, every launch counts; the step fills a block.
        {"name": "decode_b1_h4_d64_ctx128_f32", "op": "decode", "batch": 1, "heads": 4, "dim": 64, "block": 32, "total": 128,
         "rows": 127, "dtype": "f32", "ragged": False, "mask": False, "weights": False},
        # One long conversation, 7B heads: few heads, so the context has to be split.
        {"name": "decode_b1_h32_d128_ctx4083", "op": "decode", "batch": 1, "heads": 32, "dim": 128, "block": 64, "total": 4096,
         "rows": 4082, "dtype": "f16", "ragged": False, "mask": False, "weights": True},
        # The headline batch, 7B heads, under a mask row as a causal driver installs it, weights gathered.
        {"name": "decode_b64_h32_d128_ctx2041", "op": "decode", "batch": 64, "heads": 32, "dim": 128, "block": 64, "total": 2048,
         "rows": 2040, "dtype": "f16", "ragged": False, "mask": True, "weights": True},
        # 13B heads, sequences of very different lengths in one batch.
        {"name": "decode_b32_h40_d128_ragged4096", "op": "decode", "batch": 32, "heads": 40, "dim": 128, "block": 64, "total": 4096,
         "rows": 4090, "dtype": "f16", "ragged": True, "mask": False, "weights": False},
        # Odd everything: a head size that is no power of two, fp32 inputs, a long block, a masked window.
        {"name": "decode_b5_h7_d96_ctx777_f32", "op": "decode", "batch": 5, "heads": 7, "dim": 96, "block": 128, "total": 1024,
         "rows": 776, "dtype": "f32", "ragged": False, "mask": True, "weights": True},
        # The prompt phase.
        # A batch of prompts, 7B heads, causal.
        {"name": "prompt_b8_h32_d128_s1024", "op": "prompt", "batch": 8, "heads": 32, "dim": 128, "block": 64, "total": 1088,
         "seq": 1024, "start": 0, "dtype": "f16", "mask": True, "weight_queries": -1},
        # One long prompt, causal; the last queries' weights are gathered, for an eviction that follows.
        {"name": "prompt_b1_h32_d128_s4096", "op": "prompt", "batch": 1, "heads": 32, "dim": 128, "block": 64, "total": 4160,
         "seq": 4096, "start": 0, "dtype": "f16", "mask": True, "weight_queries": 64},
        # The second piece of a prompt, odd sizes, fp32, no mask, the weights of all its queries.
        {"name": "prompt_b3_h5_d96_s333_after77_f32", "op": "prompt", "batch": 3, "heads": 5, "dim": 96, "block": 32, "total": 448,
         "seq": 333, "start": 77, "dtype": "f32", "mask": False, "weight_queries": 0},
        # Reading the cache back, to move a sequence to another cache type: a batch of prompts, and a few odd rows.
        {"name": "read_b8_h32_d128_rows1024", "op": "read", "batch": 8, "heads": 32, "dim": 128, "block": 64, "total": 1088,
         "rows": 1024, "dtype": "f16", "ragged": False},
        {"name": "read_b2_h5_d96_rows77_f32", "op": "read", "batch": 2, "heads": 5, "dim": 96, "block": 32, "total": 128,
         "rows": 77, "dtype": "f32", "ragged": True},
        # The eviction: the headline batch cut to half its rows, and sequences of different lengths in an odd shape.
        {"name": "evict_b64_h32_d128_2048to1024", "op": "evict", "batch": 64, "heads": 32, "dim": 128, "block": 64, "total": 2048,
         "rows": 2048, "keep": 16, "recent": 4, "ragged": False},
        {"name": "evict_b3_h5_d96_ragged1500", "op": "evict", "batch": 3, "heads": 5, "dim": 96, "block": 32, "total": 1536,
         "rows": 1500, "keep": 17, "recent": 5, "ragged": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "read", "evict"])
    block = rng.choice([32, 64, 128])
    dim = rng.choice([32, 64, 96, 128] + ([256] if op != "prompt" else []))
    batch, heads = _log(rng, 1, 64), _log(rng, 1, 40)
    c = {"op": op, "batch": batch, "heads": heads, "dim": dim, "block": block}
    most = (1 << 28) // (batch * heads * dim)  # rows: at most half the headline cache
    if op == "prompt":
        fits = int(math.sqrt(3.0e10 / (batch * heads * dim)))
        seq = _log(rng, 1, max(2, min(3000, fits, most // 2)))
        start = rng.choice([0, 0, _log(rng, 1, max(2, min(2000, fits, most // 2)))])
        c.update(seq=seq, start=start, total=-(-(start + seq) // block) * block + block, dtype=rng.choice(["f16", "f32"]),
                 mask=rng.random() < 0.6, weight_queries=rng.choice([-1, 0, _log(rng, 1, 128)]))
        return c
    rows = _log(rng, 1, max(2, min(9000, most)))
    c.update(rows=rows, total=(rows // block + 1) * block, ragged=rng.random() < 0.4)
    if op == "evict":
        n = max(1, rows // block)
        keep = rng.randint(1, n)
        c.update(keep=keep, recent=rng.randint(0, keep))
    else:
        c["dtype"] = rng.choice(["f16", "f32"])
    if op == "decode":
        c.update(mask=rng.random() < 0.4, weights=rng.random() < 0.5)
    return c


# ------------------------------------------------------------------------------------------------------------ inputs

def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _table(rows, dim):
    """RoPE table [rows, dim]: cos and sin interleaved, angles in 64 bits."""
    w = torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"), -2.0 * torch.arange(dim // 2, device="cuda", dtype=torch.float64) / dim)
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * w
    return torch.stack([a.cos(), a.sin()], -1).reshape(rows, dim).float()


def _cache(case, g, weights):
    """A cache whose complete blocks hold quantised N(0,1) rows: what earlier steps left behind."""
    B, H, D, L, T = case["batch"], case["heads"], case["dim"], case["total"], case["block"]
    c = {}
    for name in ("k", "v"):
        x = torch.randn(B, H, L // T, T * D, generator=g, device="cuda", dtype=torch.float16)
        top = x.abs().amax(-1).float()
        q = x.float()
        q.mul_((127.0 / top)[..., None]).round_()
        c[name] = q.to(torch.int8).view(B, H, L, D)
        c[name + "_scale"] = top / 127.0
        del x, q
        c[name + "_tail"] = torch.randn(B, H, T, D, generator=g, device="cuda", dtype=torch.float16)
    c["weights"] = torch.rand(B, H, L // T, generator=g, device="cuda") if weights else None
    return c


def _lengths(case, seed):
    """Rows of each sequence; in the decode step of a ragged batch none of them fills its block (what a step that does leaves
    behind is in other cases)."""
    r, n = np.random.RandomState(seed % (1 << 31)), case["rows"]
    if not case["ragged"]:
        return np.full(case["batch"], n, np.int64)
    x = r.randint(0, n + 1, size=case["batch"])
    x[r.randint(case["batch"])] = n
    return x - ((x + 1) % case["block"] == 0) if case["op"] == "decode" else x


def prepare(case, seed):
    B, H, D, L, T, op = case["batch"], case["heads"], case["dim"], case["total"], case["block"], case["op"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    gathers = case.get("weights", False) or case.get("weight_queries", -1) >= 0 or op == "evict"
    s = {"case": case, "cache": _cache(case, g, gathers), "mask": None, "op": None}
    if op in ("decode", "prompt"):
        S = case.get("seq", 1)
        s["q"], s["k_new"], s["v_new"] = (torch.randn(B, S, H, D, generator=g, device="cuda").to(_dtype(case)) for _ in range(3))
        s["table"] = _table(L, D)
        if case["mask"]:
            j = torch.arange(L, device="cuda")
            s["mask"] = torch.where(j[None, :] > j[:, None], torch.tensor(NEG, device="cuda"), torch.tensor(0.0, device="cuda"))
            if op == "decode" and D == 96:  # a window as well, in the soft masks' value
                s["mask"] = torch.where(j[None, :] + 500 < j[:, None], torch.tensor(-1e5, device="cuda"), s["mask"])
    if op in ("decode", "read", "evict"):
        n = _lengths(case, seed)
        s["rows"] = torch.from_numpy(n).to("cuda")
        s["rows32"] = s["rows"].to(torch.int32)
        s["fills"] = op == "decode" and bool(((n + 1) % T == 0).any())
    if op == "evict":
        keep = case["keep"] * T
        s["to"] = {"k": torch.zeros(B, H, keep, D, dtype=torch.int8, device="cuda"), "v": torch.zeros(B, H, keep, D, dtype=torch.int8, device="cuda"),
                   "k_scale": torch.zeros(B, H, case["keep"], device="cuda"), "v_scale": torch.zeros(B, H, case["keep"], device="cuda"),
                   "k_tail": s["cache"]["k_tail"], "v_tail": s["cache"]["v_tail"], "weights": torch.zeros(B, H, case["keep"], device="cuda")}
    if own:  # the handle a program keeps: shapes and the workspace that goes with them
        from fasterllama_amd import kv8
        s["op"] = kv8.KV8Attention(B, H, D, L, dtype=_dtype(case) if "dtype" in case else torch.float16, block_len=T, max_seq_len=case.get("seq", 1))
        s["cache"] = kv8.KV8Cache.of(block_len=T, **s["cache"])
        if op == "evict":
            s["to"] = kv8.KV8Cache.of(block_len=T, **s["to"])
    return s


# -------------------------------------------------------------------------------------------------------- plain forms

def _rotate(x, table):
    """Interleaved pairs of [..., D] by the table rows [..., D]; the fused products' single rounding by way of 64 bits."""
    x = x.float()
    x0, x1, c, n = x[..., 0::2], x[..., 1::2], table[..., 0::2], table[..., 1::2]
    a, b = (x1 * n).double(), (x0 * n).double()
    return torch.stack([(x0.double() * c - a).float(), (x1.double() * c + b).float()], -1).flatten(-2)


def _stored(x):
    x = x.float()
    return torch.where(torch.isfinite(x), x, 0.0).clamp(-65504.0, 65504.0).to(torch.float16)


def _quantise(x):
    """[..., T, D] -> integers and scales [...]."""
    top = x.abs().amax((-1, -2)).double()  # quotients by way of 64 bits: a scalar's would be a product with its reciprocal
    inverse = torch.where(top > 0, 127.0 / top, 0.0).float()
    return (x.float() * inverse[..., None, None]).round().to(torch.int8), (top / 127.0).float()


def _values(c, name, T):
    B, H, L, D = c[name].shape
    return (c[name].view(B, H, L // T, T, D).float() * c[name + "_scale"][..., None, None])


def _with_tail(c, name, T, rows):
    """All rows of the cache as values [B, H, L, D]; `rows` [B] rows are in it."""
    x = _values(c, name, T)
    B, H, N, _, D = x.shape
    at = (rows // T).clamp(max=N - 1)
    open_ = ((rows % T) > 0)[:, None, None, None]
    i = torch.arange(B, device=x.device)
    x[i, :, at] = torch.where(open_, c[name + "_tail"].float(), x[i, :, at])
    return x.view(B, H, N * T, D)


def _softmax(s):
    top = s.amax(-1, keepdim=True).clamp(min=FLOOR)
    e = (s - top).exp()
    return e / e.sum(-1, keepdim=True)


def _decode(s):
    case, c, T, D = s["case"], s["cache"], s["case"]["block"], s["case"]["dim"]
    pos = s["rows"]
    B, H, L = c["k"].shape[:3]
    i, blk, off = torch.arange(B, device=pos.device), pos // T, pos % T
    row = s["table"][pos][:, None]
    q = _rotate(s["q"][:, 0], row)
    c["k_tail"][i, :, off] = _stored(_rotate(s["k_new"][:, 0], row))
    c["v_tail"][i, :, off] = _stored(s["v_new"][:, 0])
    full = (off == T - 1)[:, None]
    for name in ("k", "v"):
        ints, scale = _quantise(c[name + "_tail"])
        x, sc = c[name].view(B, H, L // T, T, D), c[name + "_scale"]
        x[i, :, blk] = torch.where(full[..., None, None], ints, x[i, :, blk])
        sc[i, :, blk] = torch.where(full, scale, sc[i, :, blk])
    k, v = _with_tail(c, "k", T, pos + 1), _with_tail(c, "v", T, pos + 1)
    w = (k * q[:, :, None]).sum(-1) * (1.0 / math.sqrt(D))
    if s["mask"] is not None:
        w = w + s["mask"][pos][:, None]
    p = _softmax(torch.where(torch.arange(L, device=pos.device) > pos[:, None, None], -math.inf, w))
    got = {"out": (p[..., None] * v).sum(2).reshape(B, H * D), "k_tail": c["k_tail"], "v_tail": c["v_tail"]}
    if c["weights"] is not None:
        n = torch.arange(L // T, device=pos.device)
        fresh = (n == blk[:, None]) & (off == 0)[:, None]
        c["weights"].copy_(torch.where(fresh[:, None], 0.0, c["weights"]) + p.view(B, H, L // T, T).sum(-1))
        got["weights"] = c["weights"]
    if s["fills"]:
        got["k"], got["v"] = _read(s, pos + 1)
    return got


def _prompt(s):
    case, c, T, D, S, P = s["case"], s["cache"], s["case"]["block"], s["case"]["dim"], s["case"]["seq"], s["case"]["start"]
    B, H, L = c["k"].shape[:3]
    table = s["table"][P:P + S][:, None]
    q = _rotate(s["q"], table).transpose(1, 2)
    first, end = P // T * T, P + S
    last = end // T * T  # rows at and behind it stay in the tail
    for name, new in (("k", _stored(_rotate(s["k_new"], table))), ("v", _stored(s["v_new"]))):
        x = torch.cat([c[name + "_tail"][:, :, :P - first], new.transpose(1, 2)], 2)
        n = last - first
        if n > 0:
            ints, scale = _quantise(x[:, :, :n].reshape(B, H, n // T, T, D))
            c[name][:, :, first:last] = ints.view(B, H, n, D)
            c[name + "_scale"][:, :, first // T:last // T] = scale
        c[name + "_tail"][:, :, :end - max(last, first)] = x[:, :, max(n, 0):]
    rows = torch.full((B,), end, device=q.device)
    k, v = (_with_tail(c, name, T, rows)[:, :, :end] for name in ("k", "v"))
    w = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    if s["mask"] is not None:
        w = w + s["mask"][P:end, :end]
    p = _softmax(w)
    got = {"out": torch.matmul(p, v)}
    if c["weights"] is not None:
        n = case["weight_queries"] or S
        per = torch.nn.functional.pad(p[:, :, -min(n, S):].sum(2), (0, -end % T)).view(B, H, -1, T).sum(-1)
        old = c["weights"][:, :, :per.shape[-1]]
        fresh = torch.arange(per.shape[-1], device=q.device) * T >= P
        old.copy_(torch.where(fresh, 0.0, old) + per)
        got["weights"] = c["weights"]
    got["k"], got["v"] = _read(s, rows)
    return got


def _read(s, rows):
    c, T = s["cache"], s["case"]["block"]
    n = s["case"]["rows"] + (s["case"]["op"] == "decode") if "rows" in s["case"] else s["case"]["start"] + s["case"]["seq"]
    keep = (torch.arange(n, device=rows.device) < rows[:, None])[:, None, :, None]
    return [torch.where(keep, _with_tail(c, name, T, rows)[:, :, :n], 0.0).to(_dtype(s["case"])) for name in ("k", "v")]


def _evict(s):
    case, c, to, T = s["case"], s["cache"], s["to"], s["case"]["block"]
    B, H, L, D = c["k"].shape
    K = case["keep"]
    n = (s["rows"] // T)[:, None, None]
    keep, i = n.clamp(max=K), torch.arange(L // T, device=c["k"].device)
    key = torch.where(i >= n - keep.clamp(max=case["recent"]), math.inf, c["weights"])
    key = torch.where(i >= n, -math.inf, key)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :K]
    there = torch.arange(K, device=order.device) < keep
    kept = torch.sort(torch.where(there, order, L), dim=-1).values
    at = torch.where(there, kept, 0)
    for name in ("k", "v"):
        x = torch.gather(c[name].view(B, H, L // T, T * D), 2, at[..., None].expand(-1, -1, -1, T * D))
        t = to[name].view(B, H, K, T * D)
        t.copy_(torch.where(there[..., None], x, t))
        to[name + "_scale"].copy_(torch.where(there, torch.gather(c[name + "_scale"], 2, at), to[name + "_scale"]))
    # the open block's weight moves behind the kept blocks where there is a place for it
    tail = (s["rows"] % T > 0)[:, None, None] & (torch.arange(K, device=order.device) == keep)
    old = torch.where(tail, torch.gather(c["weights"], 2, n.clamp(max=L // T - 1).expand(B, H, 1)), to["weights"])
    to["weights"].copy_(torch.where(there, torch.gather(c["weights"], 2, at), old))
    return {"kept": torch.where(there, kept, -1).to(torch.int32), "rows": (keep.flatten() * T + s["rows"] % T).to(torch.int32),
            **{name: to[name] for name in ("k", "v", "k_scale", "v_scale", "weights")}}


# --------------------------------------------------------------------------------------------------------------- run

def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "read":
            k, v = _read(state, state["rows"])
            return {"k": k, "v": v}
        return {"decode": _decode, "prompt": _prompt, "evict": _evict}[case["op"]](state)
    op, c = state["op"], state["cache"]
    if case["op"] == "decode":
        at = {"start_pos_per_seq": state["rows32"], "max_start_pos": case["rows"]} if case["ragged"] else {"start_pos": case["rows"]}
        got = {"out": op.decode(state["q"], state["k_new"], state["v_new"], c, state["table"], attn_mask=state["mask"], **at),
               "k_tail": c.k_tail, "v_tail": c.v_tail}
        if c.weights is not None:
            got["weights"] = c.weights
        if state["fills"]:
            got["k"], got["v"] = op.read(c, case["rows"] + 1, rows_per_seq=state["rows32"] + 1 if case["ragged"] else None)
        return got
    if case["op"] == "prompt":
        got = {"out": op.prefill(state["q"], state["k_new"], state["v_new"], c, state["table"], start_pos=case["start"],
                                 attn_mask=state["mask"], weight_queries=max(0, case["weight_queries"]))}
        if c.weights is not None:
            got["weights"] = c.weights
        got["k"], got["v"] = op.read(c, case["start"] + case["seq"])
        return got
    if case["op"] == "read":
        k, v = op.read(c, case["rows"], rows_per_seq=state["rows32"] if case["ragged"] else None)
        return {"k": k, "v": v}
    kept, rows = op.evict(c, case["keep"], case["recent"], case["rows"], rows_per_seq=state["rows32"] if case["ragged"] else None, into=state["to"])
    to = state["to"]
    return {"kept": kept, "rows": rows, "k": to.k, "v": to.v, "k_scale": to.k_scale, "v_scale": to.v_scale, "weights": to.weights}


# -------------------------------------------------------------------------------------------------------------- work

def work(case):
    B, H, D, T = case["batch"], case["heads"], case["dim"], case["block"]
    e = 2 if case.get("dtype") == "f16" else 4
    share = 0.5 if case.get("ragged") else 1.0  # lengths are even between nothing and the longest
    if case["op"] == "decode":
        rows = case["rows"] * share
        full = (case["rows"] + 1) % T == 0 and not case["ragged"]
        whole, open_ = (rows + 1) // T * T, (rows + 1) % T
        n = B * H * (2 * D * (whole + 2 * open_) + 8 * whole / T + 3 * D * e + 4 * D)
        n += B * H * 4 * D * T if full else 0                                         # the tail that is quantised
        n += B * H * 2 * (rows / T + 1) * 4 if case["weights"] else 0
        n += 2 * B * H * D * (case["rows"] + 1) * e if full else 0                    # read back
        return {"bytes": n + 4 * D * B, "flops": 4 * B * H * D * (rows + 1)}
    if case["op"] == "prompt":
        S, P = case["seq"], case["start"]
        pairs = S * (P + (S + 1) / 2) if case["mask"] else S * (P + S)
        n = B * H * (D * S * (3 * e + 4) + 2 * D * (P + S) * 2 + 8 * (P + S) / T) + 4 * D * S
        n += B * H * (2 * D * (P + S) * e)                                            # read back
        flops = 4 * B * H * D * pairs
        if case["weight_queries"] >= 0:
            W = min(case["weight_queries"] or S, S)
            n += B * H * 2 * (P + S) / T * 4
            flops += 2 * B * H * D * (W * (P + S - W / 2) if case["mask"] else W * (P + S))
        return {"bytes": n, "flops": flops}
    if case["op"] == "read":
        rows = case["rows"]
        return {"bytes": 2 * B * H * D * (rows * share + rows * e) + 8 * B * H * rows * share / T, "flops": 2 * B * H * D * rows * share}
    n = case["rows"] // T
    kept = min(case["keep"], n * share)
    return {"bytes": B * H * (2 * 2 * T * D * kept + 4 * n * share + 24 * kept), "flops": B * H * n * share}


# ------------------------------------------------------------------------------------------------------------- exact

def exact(case, seed):
    """What run() returns for these inputs, from the definition in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c, T, D, H = s["cache"], case["block"], case["dim"], case["heads"]
    if case["op"] == "evict":
        return _exact_evict(s)
    if case["op"] == "decode":
        starts, S = s["rows"].tolist(), 1
    elif case["op"] == "prompt":
        starts, S = [case["start"]] * case["batch"], case["seq"]
    else:
        starts, S = s["rows"].tolist(), 0
    kinds = ("out", "k", "v", "k_tail", "v_tail", "weights")
    got = {n: [] for n in kinds}
    n_read = case["rows"] + (case["op"] == "decode") if "rows" in case else case["start"] + case["seq"]
    table = torch.complex(s["table"][:, 0::2].double(), s["table"][:, 1::2].double()) if S else None

    def turn(x, P):  # [H, S, D] by complex products
        z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], D // 2, 2).contiguous())
        return torch.view_as_real(z * table[P:P + x.shape[1]]).flatten(-2)

    def stored_key(x, P):  # the definition's roundings to 32 bits, each of a value in 64
        p, t = x.double().unflatten(-1, (-1, 2)), table[P:P + x.shape[1]]
        even, odd = p[..., 0], p[..., 1]
        sub, add = (odd * t.imag).float().double(), (even * t.imag).float().double()
        return torch.stack([even * t.real - sub, odd * t.real + add], -1).float().double().flatten(-2)

    def half(x):
        return x.nan_to_num(nan=0.0, posinf=0.0, neginf=0.0).clamp(-65504.0, 65504.0).to(torch.float16).double()

    for b, P in enumerate(starts):
        end, val, tails = P + S, {}, {}
        for name in ("k", "v"):
            x = c[name][b].double() * c[name + "_scale"][b].double().repeat_interleave(T, -1)[..., None]
            tail = c[name + "_tail"][b].double().clone()
            x = x[:, :max(end, 1)].clone()
            lo = P // T * T
            x[:, lo:P] = tail[:, :P - lo]
            if S:
                new = s[name + "_new"][b].transpose(0, 1)
                x[:, P:end] = half(stored_key(new, P) if name == "k" else new.double())
                for t in range(lo, end, T):
                    if t + T > end:
                        tail[:, :end - t] = x[:, t:end]
                        continue
                    if case["op"] == "decode":
                        tail[:, :] = x[:, t:t + T]
                    most = x[:, t:t + T].abs().amax((-1, -2), keepdim=True)
                    per_unit = (127.0 / torch.where(most > 0, most, 1.0)).float().double()
                    x[:, t:t + T] = (x[:, t:t + T] * per_unit).float().double().round() * (most / 127.0).float().double()
            val[name], tails[name] = x, tail
        pad = torch.zeros(H, n_read - end, D, dtype=torch.float64, device="cuda")
        for name in ("k", "v"):
            if case["op"] != "decode" or s["fills"]:
                got[name].append(torch.cat([val[name][:, :end], pad], 1).to(torch.float32 if case["dtype"] == "f32" else torch.float16).cpu())
            if case["op"] == "decode":
                got[name + "_tail"].append(tails[name].to(torch.float16).cpu())
        if not S:
            continue
        q = turn(s["q"][b].transpose(0, 1), P)
        W = (case["weight_queries"] or S) if case["op"] == "prompt" else 1
        per = torch.zeros(H, -(-c["k"].shape[2] // T) * T, dtype=torch.float64, device="cuda")
        outs = []
        for a in range(0, S, 512):
            z = torch.matmul(q[:, a:a + 512], val["k"].transpose(-1, -2).contiguous()) / math.sqrt(D)
            if s["mask"] is not None:
                z += s["mask"][P + a:P + min(a + 512, S), :end].double()
            z = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=FLOOR))
            z /= z.sum(-1, keepdim=True)
            outs.append(torch.matmul(z, val["v"]))
            here = z[:, max(0, S - W - a):] if c["weights"] is not None else z[:, :0]
            per[:, :end] += here.sum(1)
        out = torch.cat(outs, 1)
        got["out"].append((out if case["op"] == "prompt" else out.reshape(H * D)).cpu())
        if c["weights"] is not None:
            old = c["weights"][b].double().clone()
            old[:, -(-P // T):-(-end // T)] = 0.0
            got["weights"].append((old + per.view(H, -1, T).sum(-1)).cpu())
    return {n: torch.stack(v) for n, v in got.items() if v}


def _exact_evict(s):
    case, T = s["case"], s["case"]["block"]
    n, K = s["rows"].cpu().numpy() // T, case["keep"]
    w = s["cache"]["weights"].double().cpu().numpy()
    sc = {name: s["cache"][name].double().cpu().numpy() for name in ("k_scale", "v_scale")}
    to = {name: np.zeros((case["batch"], case["heads"], K)) for name in ("k_scale", "v_scale", "weights")}
    for b in range(case["batch"]):
        keep = min(K, int(n[b]))
        sure = min(case["recent"], keep)
        for h in range(case["heads"]):
            cand = w[b, h, :n[b] - sure]
            best = np.lexsort((np.arange(cand.size), -cand))[:keep - sure]
            kept = np.concatenate([np.sort(best), np.arange(n[b] - sure, n[b])]).astype(np.int64)
            for name in sc:
                to[name][b, h, :keep] = sc[name][b, h, kept]
            to["weights"][b, h, :keep] = w[b, h, kept]
            if keep < K and int(s["rows"][b]) % T:
                to["weights"][b, h, keep] = w[b, h, n[b]]
    return {name: torch.from_numpy(x) for name, x in to.items()}
