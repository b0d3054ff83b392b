"""The operators of a served batch, as cases to measure: what one step over
paged KV caches does beside its model's own launches.

Kinds of case:

- ``plan``: block tables and slot maps made on the device from the requests'
  lengths (``paged.PagePlan``).
- ``store``: a step's q, k and v rows turned by RoPE, k and v stored into the
  paged pools at the plan's slots (``paged.PagedStore``).
- ``attend``: attention of one new token a request over its pages
  (``paged.PagedAttend``).
- ``quantize``: a matrix to 4-bit microscaled values and back
  (``mx4.Quantize``, ``mx4.Dequantize``).
- ``linear``: rows quantised and multiplied with kept 4-bit weights
  (``mx4.Quantize``, ``mx4.Gemm``).

The plain forms are elementary torch operations in 32 bits, rounded once at
the end.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

NONE = -1            # 0xFFFFFFFF, as the int32 tensors hold it
HEAD_ROOM = 3        # free blocks taken before the step, so that the list does not start at its first

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# The cases ------------------------------------------------------------------------


def listed():
    return [
        # One decode step of a few conversations: the smallest call.
        {"name": "plan-8", "kind": "plan", "requests": 8, "longest": 4095, "chunk": 1, "block": 16, "spare": 0},
        # A busy server's step: most requests decode a token, some are in a
        # chunk of their prompt, the step padded to its fixed token count.
        {"name": "plan-1500-chunked", "kind": "plan", "requests": 1500, "longest": 8000, "chunk": 512, "block": 16,
         "spare": 777},
        # A decode step's rows of the 1B model's heads, f32 as its GEMM makes them.
        {"name": "store-8", "kind": "store", "tokens": 8, "heads": 32, "kv_heads": 8, "head_dim": 64, "block": 64,
         "type": "f32", "cache": "f16", "rotated": 32},
        # Chunks of several prompts, an odd number of tokens, bf16 rows, half of each head turned.
        {"name": "store-8191-bf16", "kind": "store", "tokens": 8191, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "block": 16, "type": "bf16", "cache": "bf16", "rotated": 32},
        # Many short conversations, an odd group of query heads.
        {"name": "attend-41x700", "kind": "attend", "requests": 41, "longest": 700, "heads": 28, "kv_heads": 4,
         "head_dim": 64, "block": 16, "cache": "f16", "window": 0},
        # One very long document: only a split over its length fills the card.
        {"name": "attend-1x131072", "kind": "attend", "requests": 1, "longest": 131072, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "block": 64, "cache": "f16", "window": 0},
        # A large ragged batch, long and short together.
        {"name": "attend-64x16384-bf16", "kind": "attend", "requests": 64, "longest": 16384, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 16, "cache": "bf16", "window": 0},
        # A few rows of activations of a ragged width.
        {"name": "quantize-9x1000", "kind": "quantize", "rows": 9, "k": 1000, "type": "f32"},
        # A large layer's weights.
        {"name": "quantize-8192x8192", "kind": "quantize", "rows": 8192, "k": 8192, "type": "bf16"},
        # A decode step of eight rows through the 1B model's gate projection: the weights' stream.
        {"name": "linear-8x8192x2048", "kind": "linear", "m": 8, "n": 8192, "k": 2048, "type": "f32", "out": "f32"},
        # A short prompt through a layer of ragged sizes.
        {"name": "linear-100x5000x3080", "kind": "linear", "m": 100, "n": 5000, "k": 3080, "type": "bf16",
         "out": "bf16"},
        # The 1B prefill's rows (4 x 2048) through its gate projection.
        {"name": "linear-8192x8192x2048", "kind": "linear", "m": 8192, "n": 8192, "k": 2048, "type": "f16",
         "out": "f16"},
    ]


def _log(rng, lo, hi):
    """A whole number of lo .. hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["plan", "store", "attend", "attend", "quantize", "linear", "linear"])
    if kind == "plan":
        n = _log(rng, 1, 4096)
        return {"kind": kind, "requests": n, "longest": _log(rng, 1, 8192), "chunk": _log(rng, 1, 1 + 200000 // n // 4),
                "block": rng.choice([8, 16, 16, 24, 64, 128]), "spare": rng.choice([0, _log(rng, 1, 1000)])}
    if kind == "store":
        d = rng.choice([64, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        t = rng.choice(["f32", "f16", "bf16"])
        return {"kind": kind, "tokens": _log(rng, 1, 8191 * 128 // d), "heads": kv * rng.randint(1, 4), "kv_heads": kv,
                "head_dim": d, "block": rng.choice([8, 16, 24, 64]), "type": t,
                "cache": t if t != "f32" else rng.choice(["f16", "bf16"]), "rotated": rng.choice([0, d // 4, d // 2])}
    if kind == "attend":
        d = rng.choice([64, 64, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8, 8])
        n = _log(rng, 1, 200)
        longest = _log(rng, 16, min(131072, 64 * 16384 * 8 * 128 // (n * kv * d)))
        return {"kind": kind, "requests": n, "longest": longest, "heads": kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]),
                "kv_heads": kv, "head_dim": d, "block": rng.choice([8, 16, 16, 24, 64, 128]),
                "cache": rng.choice(["f16", "bf16"]), "window": rng.choice([0, 0, 0, _log(rng, 8, 4096)])}
    if kind == "quantize":
        rows = _log(rng, 1, 8192)
        return {"kind": kind, "rows": rows, "k": _log(rng, 8, 8192), "type": rng.choice(["f32", "f16", "bf16"])}
    m, n = _log(rng, 1, 8192), _log(rng, 16, 16384)
    k = _log(rng, 32, min(16384, max(32, 8192 * 8192 * 2048 // (m * n))))
    return {"kind": kind, "m": m, "n": n, "k": k, "type": rng.choice(["f32", "f16", "bf16"]),
            "out": rng.choice(["f32", "f16", "bf16"])}


# What a program has in hand --------------------------------------------------------


class _Framework:
    """The device, opened once a process."""

    device = None


def _device():
    if _Framework.device is None:
        from furykernel_amd import runtime
        torch.cuda.init()
        _Framework.device = runtime.Device(0)
    return _Framework.device


class _Owner:
    """Gives back what a state holds, once neither the state nor any view of
    its buffers is left."""

    def __init__(self):
        self.held = []

    def __del__(self):
        if self.held:
            torch.cuda.synchronize()
        for b in self.held:
            b.free()


class _Span:
    """Device memory as torch takes it; a tensor over it keeps its owner."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (int(ptr), False),
                                         "strides": None, "version": 2}


_VIEWS = {torch.float32: ("<f4", None), torch.float16: ("<f2", None), torch.bfloat16: ("<i2", torch.bfloat16),
          torch.int32: ("<i4", None), torch.uint8: ("|u1", None)}


class _Memory:
    """Buffers of the framework's, each with a tensor over the same memory."""

    def __init__(self):
        self.owner = _Owner()

    def empty(self, shape, dtype):
        typestr, as_type = _VIEWS[dtype]
        size = math.prod(shape) * dtype.itemsize
        buf = _device().alloc(max(size, 16))
        self.owner.held.append(buf)
        t = torch.as_tensor(_Span(self.owner, buf.ptr, shape, typestr), device="cuda")
        return buf, (t if as_type is None else t.view(as_type))

    def put(self, tensor):
        buf, view = self.empty(tuple(tensor.shape), tensor.dtype)
        view.copy_(tensor)
        return buf, view


class _State:
    """A pass (`go`) and what it needs; it returns its outputs."""

    def __init__(self, go):
        self.go = go


def prepare(case, seed):
    made = _INPUTS[case["kind"]](case, int(seed))
    go = (_OWN if own else _PLAIN)[case["kind"]](case, made)
    torch.cuda.synchronize()
    return _State(go)


def run(state):
    return state.go()


def exact(case, seed):
    """What `run` returns, from the definitions in binary64 (whole numbers in
    the host's integers), on the same inputs."""
    return _EXACT[case["kind"]](case, _INPUTS[case["kind"]](case, int(seed)))


def work(case):
    return _WORK[case["kind"]](case)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)


def _rng(seed):
    return np.random.default_rng(int(seed) * 2 + 1)


def _normal(gen, dims, dtype, std=1.0):
    return (torch.randn(dims, generator=gen, device="cuda") * std).to(dtype)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _lengths(rng, n, longest):
    """Lengths spread over the logarithm up to the longest, the longest
    among them."""
    low = max(1.0, longest / 16)
    x = np.exp(rng.uniform(math.log(low), math.log(longest), n)) if longest > 1 else np.ones(n)
    x = np.clip(np.rint(x), 1, longest).astype(np.int64)
    x[rng.integers(n)] = longest
    return x


# plan: block tables and slot maps ------------------------------------------------------


def _plan_sizes(case):
    """The step's counts, the same for every seed: requests that have
    finished add nothing, one in eight is in a chunk of its prompt."""
    n, chunk = case["requests"], case["chunk"]
    rng = np.random.default_rng(n * 7 + chunk)
    fresh = np.ones(n, np.int64)
    if chunk > 1:
        kind = rng.integers(0, 8, n)
        fresh[kind == 0] = rng.integers(1, chunk + 1, int((kind == 0).sum()))
        fresh[kind == 1] = 0
    table_len = -(-(case["longest"] + chunk) // case["block"])
    return fresh, table_len, int(fresh.sum()) + case["spare"]


def _plan_inputs(case, seed):
    rng = _rng(seed)
    n, block = case["requests"], case["block"]
    fresh, table_len, tokens = _plan_sizes(case)
    fresh = rng.permutation(fresh)
    cached = _lengths(rng, n, case["longest"])
    cached[rng.random(n) < 0.05] = 0
    held = -(-cached // block)
    need = -(-(cached + fresh) // block) - held
    blocks = int(held.sum() + need.sum()) + HEAD_ROOM + 5
    order = rng.permutation(blocks)
    table = np.zeros((n, table_len), np.int64)
    at = 0
    for r in range(n):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    ints = {k: _cuda(v.astype(np.int32)) for k, v in (("cached", cached), ("fresh", fresh), ("table", table),
                                                      ("free", np.concatenate([order[:HEAD_ROOM], order[at:]])),
                                                      ("head", np.array([HEAD_ROOM])))}
    return {**ints, "tokens": tokens}


def _plan_plain(case, s):
    block, n, tokens = case["block"], case["requests"], s["tokens"]
    table_len = s["table"].shape[1]
    spans = torch.arange(tokens, device="cuda")
    pages = torch.arange(table_len, device="cuda")[None]

    def go():
        cached, fresh, free, head = (s[k].long() for k in ("cached", "fresh", "free", "head"))
        table = s["table"]
        total = cached + fresh
        ends = fresh.cumsum(0)
        starts = torch.cat([ends.new_zeros(1), ends])
        held = (cached + block - 1) // block
        fits = (total <= table_len * block) & (ends <= tokens)
        need = torch.where(fits, (total + block - 1) // block - held, 0)
        after = need.cumsum(0)
        fits = fits & ((need == 0) | (after <= free.numel() - head))
        taken = torch.where(fits & (need > 0), after, 0).max()
        first = head + after - need
        mine = fits[:, None] & (pages >= held[:, None]) & (pages < (held + need)[:, None])
        new = free[(first[:, None] + pages - held[:, None]).clamp(0, free.numel() - 1)]
        table = torch.where(mine, new.int(), table)
        r = torch.searchsorted(ends, spans, right=True)
        live = r < n
        rc = r.clamp(max=n - 1)
        pos = torch.where(live, cached[rc] + spans - starts[rc], 0)
        page = (pos // block).clamp(max=table_len - 1)
        slots = torch.where(live & fits[rc], table[rc, page].long() * block + pos % block, NONE)
        owner = torch.where(live, r, NONE)
        counts = torch.stack([ends[-1], taken, (~fits).sum(), head[0] + taken])
        return {"table": table, "lengths": torch.where(fits, total, cached).int(), "starts": starts.int(),
                "slots": slots.int(), "positions": pos.int(), "owner": owner.int(), "counts": counts.int()}

    return go


def _plan_own(case, s):
    from furykernel_amd import paged
    mem = _Memory()
    n, tokens = case["requests"], s["tokens"]
    ins = {k: mem.put(s[k]) for k in ("cached", "fresh", "free", "head", "table")}
    outs = {"lengths": mem.empty((n,), torch.int32), "starts": mem.empty((n + 1,), torch.int32),
            "slots": mem.empty((tokens,), torch.int32), "positions": mem.empty((tokens,), torch.int32),
            "owner": mem.empty((tokens,), torch.int32), "counts": mem.empty((4,), torch.int32)}
    op = paged.PagePlan(_device(), **{k: b for k, (b, _) in (ins | outs).items()}, requests=n, tokens=tokens,
                        table_len=s["table"].shape[1], block_size=case["block"], free_len=s["free"].numel())
    views = {"table": ins["table"][1], **{k: v for k, (_, v) in outs.items()}}

    def go():
        op.enqueue()
        return views

    return go


def _plan_exact(case, s):
    """The definition, a request at a time."""
    block, n, tokens = case["block"], case["requests"], s["tokens"]
    cached, fresh, free, table = (s[k].cpu().numpy().astype(np.int64) for k in ("cached", "fresh", "free", "table"))
    head = int(s["head"])
    slots, pos, owner = np.full(tokens, NONE), np.zeros(tokens, np.int64), np.full(tokens, NONE)
    lengths, starts = cached.copy(), np.zeros(n + 1, np.int64)
    wanted = taken = refused = 0
    for r in range(n):
        c, f = int(cached[r]), int(fresh[r])
        first, last = int(starts[r]), int(starts[r]) + f
        starts[r + 1] = last
        held, pages = -(-c // block), -(-(c + f) // block)
        ok = pages <= table.shape[1] and last <= tokens
        if ok and pages > held:
            wanted += pages - held
            ok = wanted <= len(free) - head
            if ok:
                table[r, held:pages] = free[head + wanted - (pages - held):head + wanted]
                taken = wanted
        t = np.arange(first, min(last, tokens))
        p = c + t - first
        owner[t], pos[t] = r, p
        if ok:
            lengths[r] = c + f
            slots[t] = table[r, p // block] * block + p % block
        else:
            refused += 1
    counts = np.array([starts[-1], taken, refused, head + taken])
    return {k: _cuda(v.astype(np.int32)) for k, v in (
        ("table", table), ("lengths", lengths), ("starts", starts), ("slots", slots), ("positions", pos),
        ("owner", owner), ("counts", counts))}


def _plan_work(case):
    fresh, table_len, tokens = _plan_sizes(case)
    n = case["requests"]
    # lengths in and out, each token's slot, position and owner, each page the tokens touch
    return {"bytes": 4 * (4 * n + 3 * tokens + 2 * int((fresh // case["block"] + 1).sum())), "flops": 4 * tokens}


# store: rows into the pools -------------------------------------------------------------


def _store_inputs(case, seed):
    gen, rng = _generator(seed), _rng(seed)
    T, h, kv, d, block = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    blocks = -(-T // block) + 4
    slots = rng.permutation(blocks * block)[:T]
    slots[rng.random(T) < 0.02] = NONE           # a padded step's rows
    rotated, rows = case["rotated"], 4096
    pos = rng.integers(0, rows, T)
    freq = 10000.0 ** (-2.0 * np.arange(rotated) / d)
    angle = (np.arange(rows)[:, None] * freq.astype(np.float32)).astype(np.float32).astype(np.float64)
    rope = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    cache = _TYPES[case["cache"]]
    return {"qkv": _normal(gen, (T, (h + 2 * kv) * d), _TYPES[case["type"]]), "slots": _cuda(slots.astype(np.int32)),
            "positions": _cuda(pos.astype(np.int32)), "rope": _cuda(rope),
            "qr": _normal(gen, (T, h, d), cache), "k": _normal(gen, (blocks, kv, block, d), cache),
            "v": _normal(gen, (blocks, kv, block, d), cache)}


def _store_rows(case, s, dtype):
    """q, k, v as [tokens, heads, d], q and k turned, in `dtype`."""
    h, kv, d, n = case["heads"], case["kv_heads"], case["head_dim"], case["rotated"]
    x = s["qkv"].to(dtype)
    q, k, v = (t.unflatten(1, (-1, d)) for t in x.split([h * d, kv * d, kv * d], 1))
    c, sn = (t[:, None] for t in s["rope"][s["positions"].long()].to(dtype).unbind(-1))

    def turn(t):
        half = d // 2
        a, b = t[..., :n], t[..., half:half + n]
        return torch.cat([a * c - b * sn, t[..., n:half], b * c + a * sn, t[..., half + n:]], -1)

    return turn(q), turn(k), v


def _store_plain(case, s):
    block, kv = case["block"], case["kv_heads"]
    heads = torch.arange(kv, device="cuda")[None]
    # rows without a slot go to a block past the pool's, which is no output
    qr, blocks = s["qr"].clone(), s["k"].shape[0]
    pools = [torch.cat([s[i], s[i][:1]]) for i in "kv"]

    def go():
        q, k, v = _store_rows(case, s, torch.float32)
        slot = s["slots"].long()
        live = slot >= 0
        qr.copy_(torch.where(live[:, None, None], q.to(qr.dtype), qr))
        at = torch.where(live, slot // block, blocks)[:, None]
        for pool, x in zip(pools, (k, v)):
            pool[at, heads, (slot % block)[:, None]] = x.to(pool.dtype)
        return {"qr": qr, "k": pools[0][:blocks], "v": pools[1][:blocks]}

    return go


def _store_own(case, s):
    from furykernel_amd import paged
    mem = _Memory()
    T, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    b = {k: mem.put(s[k]) for k in ("qkv", "slots", "positions", "qr", "k", "v")}
    rope = mem.put(s["rope"])[0] if case["rotated"] else None
    op = paged.PagedStore(_device(), q=b["qkv"][0], k=b["qkv"][0], v=b["qkv"][0], k_offset=h * d,
                          v_offset=(h + kv) * d, q_stride=(h + 2 * kv) * d, k_stride=(h + 2 * kv) * d,
                          v_stride=(h + 2 * kv) * d, slots=b["slots"][0], positions=b["positions"][0], rope=rope,
                          rope_rows=s["rope"].shape[0], rotated=case["rotated"], qr=b["qr"][0], kpool=b["k"][0],
                          vpool=b["v"][0], tokens=T, heads=h, kv_heads=kv, head_dim=d, block_size=case["block"],
                          blocks=s["k"].shape[0], rows_type=case["type"], cache=case["cache"])
    views = {k: b[k][1] for k in ("qr", "k", "v")}

    def go():
        op.enqueue()
        return views

    return go


def _store_exact(case, s):
    q, k, v = _store_rows(case, s, torch.float64)
    out = {"qr": s["qr"].double(), "k": s["k"].double(), "v": s["v"].double()}
    slot = s["slots"].long()
    live = (slot >= 0).nonzero()[:, 0]
    out["qr"][live] = q[live]
    for name, x in (("k", k), ("v", v)):
        rows = out[name].transpose(1, 2).reshape(-1, *x.shape[1:])     # [slots, kv heads, d]
        rows[slot[live]] = x[live]
        out[name] = rows.view(out[name].shape[0], case["block"], *x.shape[1:]).transpose(1, 2).contiguous()
    return out


def _store_work(case):
    T, d = case["tokens"], case["head_dim"]
    wide = 4 if case["type"] == "f32" else 2
    e = (case["heads"] + 2 * case["kv_heads"]) * d
    return {"bytes": T * (e * (wide + 2) + 8 + 8 * case["rotated"]),
            "flops": T * 6 * case["rotated"] * (case["heads"] + case["kv_heads"])}


# attend: one token a request over its pages ------------------------------------------------


def _attend_lengths(case):
    rng = np.random.default_rng(case["requests"] * 31 + case["longest"])
    return _lengths(rng, case["requests"], case["longest"])


def _attend_inputs(case, seed):
    gen, rng = _generator(seed), _rng(seed)
    n, h, kv, d, block = (case[k] for k in ("requests", "heads", "kv_heads", "head_dim", "block"))
    lengths = rng.permutation(_attend_lengths(case))
    pages = -(-lengths // block)
    blocks = int(pages.sum()) + 3
    order = rng.permutation(blocks)
    table = np.zeros((n, -(-case["longest"] // block)), np.int32)
    at = 0
    for r in range(n):
        table[r, :pages[r]] = order[at:at + pages[r]]
        at += pages[r]
    t = _TYPES[case["cache"]]
    return {"q": _normal(gen, (n, h, d), t), "k": _normal(gen, (blocks, kv, block, d), t),
            "v": _normal(gen, (blocks, kv, block, d), t), "table": _cuda(table),
            "lengths": _cuda(lengths.astype(np.int32))}


def _scale(case):
    return 1.0 / math.sqrt(case["head_dim"])


def _attend_plain(case, s):
    n, h, kv, d, block = (case[k] for k in ("requests", "heads", "kv_heads", "head_dim", "block"))
    pages = s["table"].shape[1]
    keys = torch.arange(pages * block, device="cuda")[None]
    step = max(1, int((1 << 28) // (pages * block * kv * d)))   # requests at once: 1 GB of keys in 32 bits

    def go():
        out = []
        for r0 in range(0, n, step):
            rows = slice(r0, min(n, r0 + step))
            at = s["table"][rows].long()
            length = s["lengths"][rows].long()[:, None]

            def gather(pool):   # [requests, kv heads, keys, d]
                return pool[at].transpose(1, 2).flatten(2, 3).float()

            q = s["q"][rows].float().unflatten(1, (kv, h // kv))
            score = torch.matmul(q, gather(s["k"]).transpose(2, 3).contiguous()) * _scale(case)
            live = keys < length
            if case["window"]:
                live &= keys >= length - case["window"]
            score = score.masked_fill(~live[:, None, None], -math.inf)
            e = (score - score.amax(-1, keepdim=True)).exp()
            v = gather(s["v"]).masked_fill(~live[:, None, :, None], 0.0)
            o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
            out.append(o.flatten(1, 2).to(s["q"].dtype))
        return out[0] if len(out) == 1 else torch.cat(out)

    return go


def _attend_own(case, s):
    from furykernel_amd import paged
    mem = _Memory()
    b = {k: mem.put(s[k])[0] for k in ("q", "k", "v", "table", "lengths")}
    out, view = mem.empty(tuple(s["q"].shape), s["q"].dtype)
    sizes = dict(requests=case["requests"], heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                 block_size=case["block"], blocks=s["k"].shape[0], table_len=s["table"].shape[1])
    workspace, _ = mem.empty((paged.attend_workspace(**sizes),), torch.uint8)
    op = paged.PagedAttend(_device(), q=b["q"], kpool=b["k"], vpool=b["v"], table=b["table"], lengths=b["lengths"],
                           out=out, workspace=workspace, scale=_scale(case), window=case["window"],
                           cache=case["cache"], **sizes)

    def go():
        op.enqueue()
        return view

    return go


def _attend_exact(case, s):
    kv, d, block = case["kv_heads"], case["head_dim"], case["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, length in enumerate(s["lengths"].tolist()):
        first = max(0, length - case["window"]) if case["window"] else 0
        at = torch.arange(first, length, device="cuda")
        page, within = s["table"][r].long()[at // block], at % block
        for g in range(kv):
            k, v = s["k"][page, g, within].double(), s["v"][page, g, within].double()
            heads = slice(g * case["heads"] // kv, (g + 1) * case["heads"] // kv)
            p = torch.softmax(s["q"][r, heads].double() @ k.t() * _scale(case), -1)
            out[r, heads] = p @ v
    return out


def _attend_work(case):
    keys = _attend_lengths(case)
    if case["window"]:
        keys = np.minimum(keys, case["window"])
    keys = int(keys.sum())
    n, h, kv, d = (case[k] for k in ("requests", "heads", "kv_heads", "head_dim"))
    return {"bytes": 4 * keys * kv * d + 4 * n * h * d + 4 * n + 4 * (keys // case["block"]), "flops": 4 * keys * h * d}


# quantize: 4-bit microscaled values ---------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _matrix(gen, rows, k, dtype):
    """Normals with some columns far larger, as activations and weights have."""
    x = torch.randn((rows, k), generator=gen, device="cuda")
    gain = torch.where(torch.rand((k,), generator=gen, device="cuda") < 0.02, 20.0, 1.0)
    return (x * gain).to(dtype)


def _quantize_inputs(case, seed):
    return {"x": _matrix(_generator(seed), case["rows"], case["k"], _TYPES[case["type"]])}


def _mx4_plain(x):
    """(codes' values over their scales, the scales) of blocks of 32 of the
    rows, in 32 bits: [rows, blocks, 32] and [rows, blocks, 1]."""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))
    big = x.abs().amax(-1, keepdim=True)
    # frexp: big = m 2^e with m in [1/2, 1), so floor(log2 big) = e - 1
    exp = (torch.frexp(big)[1] - 3).clamp(-127, 127)
    scale = torch.ldexp(torch.ones_like(big), exp)
    scale = torch.where(big == 0, 1.0, scale)
    y = (x / scale).abs()
    # to the nearest value, ties to the even code
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp(max=6.0)
    return torch.copysign(y, x), scale


def _quantize_plain(case, s):
    k, dtype = case["k"], s["x"].dtype

    def go():
        codes, scale = _mx4_plain(s["x"])
        return {"values": (codes * scale).flatten(1)[:, :k].to(dtype), "scales": scale[..., 0]}

    return go


def _quantize_own(case, s):
    from furykernel_amd import mx4
    mem = _Memory()
    rows, k, t = case["rows"], case["k"], case["type"]
    x, _ = mem.put(s["x"])
    y, values = mem.empty((rows, k), s["x"].dtype)
    scales, scale_view = mem.empty((rows, -(-k // 32)), torch.float32)
    held = mx4.Mx4Matrix(_device(), rows, k)
    mem.owner.held.append(held)
    quantize = mx4.Quantize(_device(), x, held, x_type=t)
    back = mx4.Dequantize(_device(), held, y, y_type=t, scales=scales)

    def go():
        quantize.enqueue()
        back.enqueue()
        return {"values": values, "scales": scale_view}

    return go


def _mx4_exact(x):
    """The values and scales from the definition: the largest power of two
    in the block over e2m1's largest power of two (4); the nearest of its
    magnitudes, halfway cases to the even code."""
    x = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))
    big = x.abs().amax(-1, keepdim=True)
    scale = torch.where(big > 0, torch.exp2(torch.floor(torch.log2(torch.where(big > 0, big, 1.0))) - 2), 1.0)
    y = (x / scale).abs()
    code = torch.zeros_like(y)
    for i in range(7):
        mid = (_E2M1[i] + _E2M1[i + 1]) / 2
        code += (y > mid if i % 2 == 0 else y >= mid).double()
    grid = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")
    return torch.copysign(grid[code.long()], x) * scale, scale[..., 0]


def _quantize_exact(case, s):
    out, scales = [], []
    for rows in s["x"].split(1024):
        v, sc = _mx4_exact(rows)
        out.append(v.flatten(1)[:, :case["k"]])
        scales.append(sc)
    return {"values": torch.cat(out), "scales": torch.cat(scales)}


def _quantize_work(case):
    n, wide = case["rows"] * case["k"], 4 if case["type"] == "f32" else 2
    blocks = case["rows"] * -(-case["k"] // 32)
    # the values read, codes and scales written and read, the values and scales written
    return {"bytes": 2 * n * wide + n + 6 * blocks, "flops": 4 * n}


# linear: rows times 4-bit weights ------------------------------------------------------------


def _linear_inputs(case, seed):
    gen = _generator(seed)
    return {"x": _matrix(gen, case["m"], case["k"], _TYPES[case["type"]]),
            "w": _normal(gen, (case["n"], case["k"]), torch.bfloat16, case["k"] ** -0.5)}


def _linear_plain(case, s):
    out = _TYPES[case["out"]]
    codes, scale = _mx4_plain(s["w"])            # kept by the program: signs and codes a byte, scales
    grid = torch.tensor(_E2M1, device="cuda")
    kept = (torch.searchsorted(grid, codes.abs().contiguous()) + 8 * codes.signbit()).to(torch.uint8)
    signed = torch.cat([grid, -grid])

    def go():
        xc, xs = _mx4_plain(s["x"])
        w = signed[kept.int()] * scale
        return torch.matmul((xc * xs).flatten(1), w.flatten(1).t()).to(out)

    return go


def _linear_own(case, s):
    from furykernel_amd import mx4
    mem = _Memory()
    dev, m, n, k = _device(), case["m"], case["n"], case["k"]
    x, _ = mem.put(s["x"])
    y, view = mem.empty((m, n), _TYPES[case["out"]])
    weights, rows = mx4.Mx4Matrix(dev, n, k), mx4.Mx4Matrix(dev, m, k)
    mem.owner.held += [weights, rows]
    w, _ = mem.put(s["w"])
    torch.cuda.synchronize()
    mx4.Quantize(dev, w, weights, x_type="bf16").enqueue()
    quantize = mx4.Quantize(dev, x, rows, x_type=case["type"])
    product = mx4.Gemm(dev, rows, weights, y, c_type=case["out"])

    def go():
        quantize.enqueue()
        product.enqueue()
        return view

    return go


def _linear_exact(case, s):
    w = _mx4_exact(s["w"])[0].flatten(1)
    out = [_mx4_exact(x)[0].flatten(1) @ w.t() for x in s["x"].split(1024)]
    return torch.cat(out)


def _linear_work(case):
    m, n, k = case["m"], case["n"], case["k"]
    wide = {"f32": 4, "f16": 2, "bf16": 2}
    return {"bytes": m * k * wide[case["type"]] + n * k // 2 + n * k // 32 + m * n * wide[case["out"]],
            "flops": 2 * m * n * k}


_INPUTS = {"plan": _plan_inputs, "store": _store_inputs, "attend": _attend_inputs, "quantize": _quantize_inputs,
           "linear": _linear_inputs}
_PLAIN = {"plan": _plan_plain, "store": _store_plain, "attend": _attend_plain, "quantize": _quantize_plain,
          "linear": _linear_plain}
_OWN = {"plan": _plan_own, "store": _store_own, "attend": _attend_own, "quantize": _quantize_own,
        "linear": _linear_own}
_EXACT = {"plan": _plan_exact, "store": _store_exact, "attend": _attend_exact, "quantize": _quantize_exact,
          "linear": _linear_exact}
_WORK = {"plan": _plan_work, "store": _store_work, "attend": _attend_work, "quantize": _quantize_work,
         "linear": _linear_work}
