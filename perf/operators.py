"""What the operators of a decoder layer that reads a bounded or a shared context are measured on.

* ``linear``: ``activation(x @ w + bias) + residual``, the projections around attention and the feed-forward block, with what
  follows the product in its epilogue.
* ``window_prefill`` / ``window_decode``: attention in which a query sees the last ``window`` keys up to its own and the first
  ``sinks`` keys of its request; prompts over packed keys or a token table, single tokens over a paged cache.
* ``shared_decode``: single-token attention of a batch whose requests all begin with the same pages of the cache.

``run`` computes them in plain torch operations in 32 bits, or, with ``own``, calls the compiled operators.  Lengths are part of a
case (its number ``lengths`` seeds them), values come from the seed.
"""

from __future__ import annotations

import contextlib
import io
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HQ, HKV, D = 32, 8, 128
G = HQ // HKV


def listed():
    return [
        # the smallest projection: four sequences' next tokens through an output projection, into the residual stream
        dict(name="linear_decode_small", op="linear", dtype="bf16", M=4, N=4096, K=4096, act="none", residual=True),
        # the up-projection of one decode step of sixteen sequences: one pass over the weight
        dict(name="linear_decode_gelu", op="linear", dtype="f16", M=16, N=11008, K=4096, act="gelu_tanh", residual=False),
        # a packed batch of prompts of odd total length through an output projection
        dict(name="linear_ragged_residual", op="linear", dtype="f16", M=1237, N=4104, K=4096, act="none", residual=True),
        # the up-projection of a long prompt
        dict(name="linear_prompt_gelu", op="linear", dtype="bf16", M=4096, N=14336, K=4096, act="gelu_tanh", residual=False),
        # the smallest prompt: one request of a few tokens, no more than the window
        dict(name="window_prefill_small", op="window_prefill", dtype="bf16", table=False, window=1024, sinks=4, batch=1, shortest=37,
             longest=37, prefix=0, lengths=1),
        # packed prompts of unlike lengths, most of them many windows long
        dict(name="window_prefill_prompts", op="window_prefill", dtype="bf16", table=False, window=1024, sinks=4, batch=6, shortest=100,
             longest=8192, prefix=0, lengths=2),
        # chunks of prompts behind a cached part, through a token table, a window that is no multiple of anything
        dict(name="window_prefill_chunks", op="window_prefill", dtype="f16", table=True, window=1500, sinks=0, batch=8, shortest=200,
             longest=512, prefix=12000, lengths=3),
        # one sequence's next token over a token table: latency
        dict(name="window_decode_one", op="window_decode", dtype="bf16", page=1, window=1000, sinks=4, batch=1, shortest=9000,
             longest=9000, lengths=4),
        # a server's batch over pages of 64 tokens
        dict(name="window_decode_batch", op="window_decode", dtype="f16", page=64, window=4096, sinks=64, batch=64, shortest=300,
             longest=32000, lengths=5),
        # a handful of requests behind a short system prompt, over a token table
        dict(name="shared_decode_few", op="shared_decode", dtype="bf16", page=1, prefix=1000, batch=7, shortest=1, longest=200, lengths=6),
        # a server's batch behind a long document
        dict(name="shared_decode_batch", op="shared_decode", dtype="f16", page=64, prefix=8192, batch=64, shortest=20, longest=1024,
             lengths=7),
        # many short conversations behind a very long one
        dict(name="shared_decode_many", op="shared_decode", dtype="bf16", page=64, prefix=32768, batch=200, shortest=1, longest=700,
             lengths=8),
    ]


def _spread(rng, low, high, step=1):
    """A whole number of ``low`` .. ``high``, even over the logarithm, rounded to a multiple of ``step``."""
    n = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(step, min(high // step * step, round(n / step) * step))


def draw(rng):
    case = _draw(rng)
    while True:                                               # no more work than the largest listed cases
        cost = work(case)
        if cost["flops"] <= 4.8e11 and cost["bytes"] <= 1.02e9:
            return case
        shrunk = "M" if case["op"] == "linear" else "batch" if case["batch"] > 1 else "longest"
        case[shrunk] = case[shrunk] * 2 // 3


def _draw(rng):
    kind = rng.choice(["linear", "linear", "window_prefill", "window_decode", "shared_decode", "shared_decode"])
    dtype = rng.choice(["f16", "bf16"])
    seed = rng.randrange(1 << 20)
    if kind == "linear":
        few = rng.random() < 0.4
        return dict(op=kind, dtype=dtype, M=_spread(rng, 1, 64) if few else _spread(rng, 65, 4096), N=_spread(rng, 512, 14336, 8),
                    K=_spread(rng, 512, 4096, 256 if few else 8), act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    residual=rng.random() < 0.5)
    if kind == "window_prefill":
        longest = _spread(rng, 16, 8192)
        return dict(op=kind, dtype=dtype, table=rng.random() < 0.5, window=_spread(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 40]),
                    batch=_spread(rng, 1, 6), shortest=max(1, longest // 32), longest=longest, prefix=rng.choice([0, 100, 8000]),
                    lengths=seed)
    if kind == "window_decode":
        longest = _spread(rng, 16, 32000)
        return dict(op=kind, dtype=dtype, page=rng.choice([1, 64]), window=_spread(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 100]),
                    batch=_spread(rng, 1, 64), shortest=max(1, longest // 32), longest=longest, lengths=seed)
    longest = _spread(rng, 1, 1024)
    page = rng.choice([1, 64])
    return dict(op=kind, dtype=dtype, page=page, prefix=_spread(rng, 64, 32768, page), batch=_spread(rng, 1, 200),
                shortest=max(1, longest // 32), longest=longest, lengths=seed)


# ------------------------------------------------------------------------------- lengths
def _lengths(case):
    """``(query tokens, keys)`` of every request; of a shared prefix, keys are the request's own."""
    rng = random.Random(case["lengths"])
    new = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    if case["op"] != "window_prefill":
        return [1] * len(new), new
    return new, [n + rng.randint(case["prefix"] // 2, case["prefix"]) for n in new]


def _bounds(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------- the compiled operators
_KERNELS: dict = {}          # a program compiles an operator once and keeps it


def _operator(case):
    """What a program compiles for a case: one kernel for all batches of the same operator."""
    if case["op"] == "linear":
        return tuple(case[k] for k in ("op", "dtype", "M", "N", "K", "act", "residual"))
    if case["op"] == "window_prefill":
        return tuple(case[k] for k in ("op", "dtype", "table", "window", "sinks"))
    if case["op"] == "window_decode":
        return tuple(case[k] for k in ("op", "dtype", "page", "window", "sinks"))
    return tuple(case[k] for k in ("op", "dtype", "page"))


def _compile(case):
    import cleave_amd
    import cleave_amd.lang as cl
    from cleave_amd import examples
    from cleave_amd.pipeline import EvalConfig, ScheduleConfig

    dtype = {"f16": cl.f16, "bf16": cl.bf16}[case["dtype"]]
    if case["op"] == "linear":
        fn = examples.linear_op(None if case["act"] == "none" else case["act"], residual=case["residual"])
        split = cl.Split("K", (4, 8)) if case["M"] <= 64 else False
        return cleave_amd.compile(fn, shapes={k: case[k] for k in "MNK"}, dtype=dtype, preset="fast", split=split, cache_kernels=False,
                                  schedule=ScheduleConfig(topk=6, split_k=getattr(split, "factors", ())),
                                  eval=EvalConfig(warmup=3, iters=30, max_parallel=0))
    config = dict(schedule=ScheduleConfig(topk=1), max_workloads=3)
    if case["op"] == "window_prefill":
        fn = examples.prefill_op(HQ, HKV, D, ragged=not case["table"], dtype=dtype, window=case["window"], sinks=case["sinks"])
        mix = cl.workloads.causal_prefill(batch=(1, 4), q_len=(8, 2048), prefix=(0, 500))
        return cleave_amd.compile(fn, workloads=mix, **config)
    if case["op"] == "window_decode":
        fn = examples.paged_decode_op(HQ, HKV, D, case["page"], dtype=dtype, window=case["window"], sinks=case["sinks"])
        mix = cl.workloads.paged_decode(batch=(1, 32), kv_len=(256, 8192), samples=2)
        return cleave_amd.compile(fn, split=cl.Split("kv_len", (8,)), workloads=mix, **config)
    fn = examples.shared_prefix_decode_op(HQ, HKV, D, case["page"], dtype=dtype)
    mix = cl.workloads.paged_decode(batch=(1, 32), kv_len=(16, 512), samples=2, prefix=2048)
    return cleave_amd.compile(fn, workloads=mix, **config)


def _kernel(case):
    key = _operator(case)
    if key not in _KERNELS:
        with contextlib.redirect_stdout(io.StringIO()):
            _KERNELS[key] = _compile(case)
    return _KERNELS[key]


# ------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """The tensors of one call, in the operator's order."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(scale, *shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(scale)

    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        args = [normal(1.0, M, K), normal(K ** -0.5, K, N), normal(0.5, 1, N)]
        return args + [normal(1.0, M, N)] if case["residual"] else args
    new, keys = _lengths(case)
    scale = D ** -0.5
    if case["op"] == "window_prefill":
        rows, total = sum(new), sum(keys)
        q = normal(1.0, rows, HQ, D)
        if not case["table"]:
            return [q, normal(1.0, total, HKV, D), normal(1.0, total, HKV, D), _int32(_bounds(new)), _int32(_bounds(keys)), scale]
        pool = total + total // 4 + 16
        table = torch.randperm(pool, generator=gen, device="cuda")[:total].to(torch.int32)
        return [q, normal(1.0, pool, 1, HKV, D), normal(1.0, pool, 1, HKV, D), _int32(_bounds(new)), _int32(_bounds(keys)), table, scale]
    page = case["page"]
    pages = [-(-n // page) for n in keys]
    first = case.get("prefix", 0) // page                    # pages of the shared beginning (whole ones)
    pool = first + sum(pages) + sum(pages) // 4 + 16
    table = torch.randperm(pool, generator=gen, device="cuda")[:first + sum(pages)].to(torch.int32)
    args = [normal(1.0, case["batch"], HQ, D), normal(1.0, pool, page, HKV, D), normal(1.0, pool, page, HKV, D)]
    if case["op"] == "shared_decode":
        args.append(table[:first].clone())
    args += [_int32(_bounds(pages)), table[first:].clone()]
    if page > 1:
        args.append(_int32([n - (p - 1) * page for n, p in zip(keys, pages)]))
    return args + [scale]


def prepare(case, seed):
    state = {"case": case, "args": _inputs(case, seed), "options": {}}
    if case["op"] == "window_decode":
        state["options"] = {"longest": max(-(-n // case["page"]) for n in _lengths(case)[1])}    # a serving loop knows it
    if own:
        state["kernel"] = _kernel(case)
    return state


# ------------------------------------------------------------------------------- the plain form
def _activated(x, act):
    if act == "relu":
        return x.clamp_min(0)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh((2 / math.pi) ** 0.5 * (x + 0.044715 * x * x * x)))
    return x


def _attend(q, k, v, scale, visible=None):
    """Heads of ``q`` (heads, rows, d) over ``k``, ``v`` (kv heads, keys, d) in 32 bits: values and base-2 log-sum-exp."""
    heads, rows, d = q.shape
    kv = k.shape[0]
    scores = torch.bmm(q.reshape(kv, heads // kv * rows, d), k.transpose(1, 2).contiguous()).mul_(scale)
    scores = scores.reshape(kv, heads // kv, rows, -1)
    if visible is not None:
        scores = scores.masked_fill_(~visible, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = torch.bmm(weights.reshape(kv, -1, weights.shape[-1]), v).reshape(heads, rows, d) / total.reshape(heads, rows, 1)
    return out, ((top + torch.log(total)) / math.log(2.0)).reshape(heads, rows)


def _rows_of(cache, ids, keys):
    """Token rows ``keys`` tokens long of the pages ``ids`` -> (kv heads, keys, d) in 32 bits."""
    return cache[ids.long()].reshape(-1, *cache.shape[2:])[:keys].float().transpose(0, 1).contiguous()


def _plain(state):
    case, args = state["case"], state["args"]
    if case["op"] == "linear":
        x, w, bias = args[:3]
        y = _activated(x.float() @ w.float() + bias.float(), case["act"])
        return (y + args[3].float() if case["residual"] else y).to(x.dtype)
    new, keys = _lengths(case)
    q = args[0]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    if case["op"] == "window_prefill":
        at_q, at_k = _bounds(new), _bounds(keys)
        for b, (n, m) in enumerate(zip(new, keys)):
            if case["table"]:
                ids = args[5][at_k[b]:at_k[b + 1]]
                k, v = _rows_of(args[1], ids, m), _rows_of(args[2], ids, m)
            else:
                k, v = (t[at_k[b]:at_k[b + 1]].float().transpose(0, 1).contiguous() for t in args[1:3])
            for lo in range(0, n, 1024):                     # (a block of queries reads its own windows' keys and the first ones)
                hi = min(n, lo + 1024)
                pos = torch.arange(m - n + lo, m - n + hi, device=q.device)[:, None]
                start = max(0, m - n + lo - case["window"] + 1)
                seen = torch.cat([torch.arange(min(case["sinks"], start), device=q.device), torch.arange(start, m - n + hi, device=q.device)])
                visible = (seen <= pos) & ((seen > pos - case["window"]) | (seen < case["sinks"]))
                rows = slice(at_q[b] + lo, at_q[b] + hi)
                o, s = _attend(q[rows].float().transpose(0, 1).contiguous(), k[:, seen].contiguous(), v[:, seen].contiguous(), args[-1],
                               visible)
                out[rows], lse[rows] = o.transpose(0, 1).to(q.dtype), s.transpose(0, 1)
        return out, lse
    shared = args[3] if case["op"] == "shared_decode" else None
    table = args[4 if shared is None else 5]
    pages = _bounds([-(-n // case["page"]) for n in keys])
    for b, m in enumerate(keys):
        ids = table[pages[b]:pages[b + 1]]
        if shared is not None:
            ids, m = torch.cat([shared, ids]), m + shared.numel() * case["page"]
        k, v = _rows_of(args[1], ids, m), _rows_of(args[2], ids, m)
        visible = None
        if case["op"] == "window_decode":
            at = torch.arange(m, device=q.device)
            visible = (at >= m - case["window"]) | (at < case["sinks"])
        o, s = _attend(q[b].float().unsqueeze(1), k, v, args[-1], visible)
        out[b], lse[b] = o[:, 0].to(q.dtype), s[:, 0]
    return out, lse


def run(state):
    return state["kernel"](*state["args"], **state["options"]) if own else _plain(state)


# ------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_row_block(q, k, v, scale, allowed):
    """One kv head: ``q`` (group, rows, d), ``k`` / ``v`` (keys, d), ``allowed`` (rows, keys) truth values."""
    logits = torch.matmul(q, k.t()) * scale
    logits = torch.where(allowed, logits, torch.full_like(logits, -math.inf))
    lse = torch.logsumexp(logits, dim=-1)
    return torch.matmul(torch.exp(logits - lse.unsqueeze(-1)), v), lse / math.log(2.0)


def exact(case, seed):
    args = _inputs(case, seed)
    if case["op"] == "linear":
        if 2 * case["M"] * case["N"] * case["K"] > 6e11:
            return None
        x, w, bias = (t.double() for t in args[:3])
        z = torch.matmul(x, w) + bias
        act = {"none": lambda t: t, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t),
               "gelu": lambda t: t * torch.special.ndtr(t),
               "gelu_tanh": lambda t: t * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3))}[case["act"]]
        z = act(z)
        return z + args[3].double() if case["residual"] else z
    new, keys = _lengths(case)
    q, page = args[0], case.get("page", 1)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    prefix = case["prefix"] // page * page if case["op"] == "shared_decode" else 0
    row = key = 0
    for n, m in zip(new, keys):
        if case["op"] == "window_prefill":
            where = torch.arange(key, key + m, device=q.device)
            if case["table"]:
                where = args[5].long()[where]
            key += m
        else:
            table = args[5 if case["op"] == "shared_decode" else 4].long()
            token = torch.arange(m, device=q.device)
            where = table[key + token // page] * page + token % page
            key += -(-m // page)
            if prefix:
                token = torch.arange(prefix, device=q.device)
                where = torch.cat([args[3].long()[token // page] * page + token % page, where])
        total = where.numel()
        position = torch.arange(total - n, total, device=q.device)
        for h in range(HKV):
            kh, vh = (t.reshape(-1, HKV, D)[:, h][where].double() for t in args[1:3])
            for lo in range(0, n, 512):
                at = position[lo:lo + 512]
                # (keys that no row of the block sees are left out before any product)
                first = max(0, int(total - n + lo) - case["window"] + 1) if "window" in case else 0
                head = min(case.get("sinks", 0), first)
                last = total - n + min(n, lo + 512)
                cols = torch.cat([torch.arange(head, device=q.device), torch.arange(first, last, device=q.device)])
                allowed = cols[None, :] <= at[:, None]
                if "window" in case:
                    allowed &= (at[:, None] - cols[None, :] < case["window"]) | (cols[None, :] < case["sinks"])
                block = q[row + lo:row + lo + at.numel(), h * G:(h + 1) * G].double().transpose(0, 1)
                o, s = _exact_row_block(block, kh[cols], vh[cols], args[-1], allowed)
                out[row + lo:row + lo + at.numel(), h * G:(h + 1) * G] = o.transpose(0, 1)
                lse[row + lo:row + lo + at.numel(), h * G:(h + 1) * G] = s.transpose(0, 1)
        row += n
    return out, lse


# ------------------------------------------------------------------------------- what a pass cannot do without
def _seen(case, first, last):
    """(query, key) pairs of the queries at positions ``first`` .. ``last`` - 1, and the keys that any of them sees."""
    w, s = case["window"], case["sinks"]
    pairs = 0
    for p in range(first, last):
        low = max(0, p - w + 1)
        pairs += p + 1 - low + min(s, low)
    low = max(0, first - w + 1)
    return pairs, last - low + min(s, low)


def work(case):
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * (M * K + K * N + N + M * N * (2 if case["residual"] else 1)), "flops": 2 * M * N * K}
    new, keys = _lengths(case)
    rows = sum(new)
    results = rows * HQ * (2 * 2 * D + 4)                     # queries in, values and log-sum-exp out
    token = 2 * 2 * HKV * D                                   # a key and its value, all heads
    if case["op"] == "shared_decode":
        prefix = case["prefix"] // case["page"] * case["page"]
        table = 4 * (prefix // case["page"] + sum(-(-n // case["page"]) for n in keys))
        return {"bytes": results + token * (prefix + sum(keys)) + table + 8 * len(keys),
                "flops": 4 * HQ * D * (prefix * len(keys) + sum(keys))}
    if case["op"] == "window_prefill":
        counts = [_seen(case, m - n, m) for n, m in zip(new, keys)]
        entries = 4 if case["table"] else 0
    else:
        counts = [_seen(case, m - 1, m) for m in keys]
        entries = 4 / case["page"]
    pairs, read = sum(p for p, _ in counts), sum(k for _, k in counts)
    return {"bytes": int(results + (token + entries) * read + 8 * len(keys)), "flops": 4 * HQ * D * pairs}
