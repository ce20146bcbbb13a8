"""The linear products with their epilogues, prompts and decode with a window, and decode over shared pages as two decoder layers use
them together: requests that begin with the same tokens, one layer that attends to all of them and one to a window with sinks.  Every
operator's result is checked against 64 bits from the very operands it was given; a decode step is also captured and replayed."""

import pytest
import torch

import cleave_amd
import cleave_amd.lang as cl
from cleave_amd import examples as C
from cleave_amd import pipeline as P
from cleave_amd.dynamic import reference as dref
from cleave_amd.pipeline.direct import kernel_for
from tests._attention64 import attend, same
from tests.test_gpu_linear_epilogue import check as check_linear

pytestmark = pytest.mark.gpu

HIDDEN, FFN, HQ, HKV, D, PAGE, WINDOW, SINKS = 256, 640, 8, 2, 64, 16, 40, 2
COMMON = 4                                     # pages that all requests begin with
OWN = [5, 33, 16, 1]                           # tokens of each request's own prompt
STEPS = 3
KEYS = [COMMON * PAGE + n for n in OWN]
POOL = COMMON + sum(-(-(n + STEPS) // PAGE) for n in OWN)
SCALE = D ** -0.5


class Linear:
    """``act(x @ w + b) + r`` with its weights; one kernel per row count, as the product's sizes are compiled in."""

    def __init__(self, K, N, gen, act=None, residual=False):
        self.act, self.residual, self.kernels = act, residual, {}
        self.w = (torch.randn(K, N, generator=gen, device="cuda") * K ** -0.5).bfloat16()
        self.b = (torch.randn(1, N, generator=gen, device="cuda") * 0.1).bfloat16()

    def __call__(self, x, *residual, log=None):
        M, K = x.shape
        if M not in self.kernels:
            prog = C.linear_op(self.act, residual=self.residual).trace(cl.bf16, M=M, N=self.w.shape[1], K=K)
            form = dict(template="skinny", tiling=dict(WAVES_N=1, WAVES_K=2)) if M <= 16 else \
                dict(template="gemm_dma", tiling=dict(BM=64, BN=64, BK=64, WM=2, WN=2))
            self.kernels[M] = kernel_for(prog, **form)
        args = [x, self.w, self.b, *residual]
        out = self.kernels[M](*args)
        if log is not None:
            log.append(("linear", out.clone(), args, (self.act, self.residual)))
        return out


class Layer:
    def __init__(self, gen, prompt, decode, windowed):
        self.qkv, self.out = Linear(HIDDEN, (HQ + 2 * HKV) * D, gen), Linear(HQ * D, HIDDEN, gen, residual=True)
        self.up, self.down = Linear(HIDDEN, FFN, gen, act="gelu_tanh"), Linear(FFN, HIDDEN, gen, residual=True)
        self.prompt, self.decode, self.windowed = prompt, decode, windowed
        self.k, self.v = (torch.zeros(POOL, PAGE, HKV, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def __call__(self, x, attend_rows, log=None):
        rows = self.qkv(x, log=log).view(-1, HQ + 2 * HKV, D)
        q, k, v = (t.contiguous() for t in rows.split((HQ, HKV, HKV), dim=1))
        h = self.out(attend_rows(self, q, k, v).view(-1, HQ * D), x, log=log)
        return self.down(self.up(h, log=log), h, log=log)


def seen_rows(new, keys, windowed):
    own = torch.arange(new, device="cuda")[:, None] + keys - new
    key = torch.arange(keys, device="cuda")[None]
    return (key <= own) & ((key > own - WINDOW) | (key < SINKS)) if windowed else key <= own


def check_log(log):
    for kind, out, args, form in log:
        if kind == "linear":
            check_linear(out, args, form[0], bias=True, residual=form[1])
            continue
        q, requests, windowed = args                                  # requests: (rows of q, their keys, their values)
        wants = [attend(q[rows], k, v, SCALE, seen_rows(len(rows), k.shape[0], windowed)) for rows, k, v in requests]
        want, _, tol, _ = [torch.cat(t) for t in zip(*wants)]
        same(out, want, tol, kind)


def gathered(cache, pages, n):
    page, slot = dref.paged_tokens(pages, 0, n, PAGE)
    return cache[page, slot].clone()


def test_prompts_then_decode_steps_eager_and_replayed():
    gen = torch.Generator(device="cuda").manual_seed(3)
    mix = cl.workloads.causal_prefill(batch=(1, 3), q_len=(3, 100), prefix=(0, 60), samples=2)
    lens = cl.workloads.paged_decode(batch=(1, 4), kv_len=(1, 200), samples=2, prefix=64)
    config = dict(schedule=P.ScheduleConfig(topk=1), max_workloads=2)
    print("decoder layers: compiling", flush=True)
    full = Layer(gen, cleave_amd.compile(C.prefill_op(HQ, HKV, D, ragged=True, dtype=cl.bf16), workloads=mix, **config),
                 cleave_amd.compile(C.shared_prefix_decode_op(HQ, HKV, D, PAGE, dtype=cl.bf16), workloads=lens, **config), False)
    windowed = Layer(gen, cleave_amd.compile(C.prefill_op(HQ, HKV, D, ragged=True, dtype=cl.bf16, window=WINDOW, sinks=SINKS), workloads=mix, **config),
                     cleave_amd.compile(C.paged_decode_op(HQ, HKV, D, PAGE, dtype=cl.bf16, window=WINDOW, sinks=SINKS), split=cl.Split("kv_len", (4,)),
                                        workloads=lens, **config), True)
    layers = [full, windowed]
    requests, order = len(OWN), torch.randperm(POOL, generator=gen, device="cuda").int()
    shared, rest, own_pages = order[:COMMON].contiguous(), order[COMMON:], []
    for n in OWN:
        count = -(-(n + STEPS) // PAGE)
        own_pages.append(rest[:count])
        rest = rest[count:]

    # ---- the prompts, packed one behind the other
    common = torch.randn(COMMON * PAGE, HIDDEN, generator=gen, device="cuda").bfloat16()
    x = torch.cat([t for n in OWN for t in (common, torch.randn(n, HIDDEN, generator=gen, device="cuda").bfloat16())])
    bounds = torch.tensor([0, *torch.tensor(KEYS).cumsum(0)], dtype=torch.int32, device="cuda")
    log = []

    def prompts(layer, q, k, v):
        out, _ = layer.prompt(q, k, v, bounds, bounds, SCALE)
        spans = [torch.arange(a, b, device="cuda") for a, b in zip(bounds.tolist(), bounds.tolist()[1:])]
        log.append(("prompts", out.clone(), (q, [(s, k[s], v[s]) for s in spans], layer.windowed), None))
        for r, s in enumerate(spans):
            for cache, new in ((layer.k, k), (layer.v, v)):
                if r == 0:
                    page, slot = dref.paged_tokens(shared, 0, COMMON * PAGE, PAGE)
                    cache[page, slot] = new[s[:COMMON * PAGE]]
                page, slot = dref.paged_tokens(own_pages[r], 0, OWN[r], PAGE)
                cache[page, slot] = new[s[COMMON * PAGE:]]
        return out

    for layer in layers:
        x = layer(x, prompts, log)
    torch.cuda.synchronize()
    check_log(log)

    # ---- decode steps: the tables stand in buffers that a captured step reads again
    own = dict(indptr=torch.zeros(requests + 1, dtype=torch.int32, device="cuda"), pages=torch.zeros(POOL, dtype=torch.int32, device="cuda"))
    both = dict(indptr=torch.zeros(requests + 1, dtype=torch.int32, device="cuda"),
                pages=torch.zeros(POOL + requests * COMMON, dtype=torch.int32, device="cuda"))
    last = torch.zeros(requests, dtype=torch.int32, device="cuda")
    at_page, at_slot = (torch.zeros(requests, dtype=torch.int64, device="cuda") for _ in range(2))
    x = x[(bounds[1:] - 1).long()].contiguous()

    def tables(step):
        lengths = [n + step + 1 for n in OWN]
        used = [-(-n // PAGE) for n in lengths]
        for table, head in ((own, 0), (both, COMMON)):
            entries = torch.cat([t for r, u in enumerate(used) for t in (shared[:head], own_pages[r][:u])])
            table["pages"][:entries.numel()] = entries
            table["indptr"].copy_(torch.tensor([0, *torch.tensor([u + head for u in used]).cumsum(0)]))
        last.copy_(torch.tensor([n - (u - 1) * PAGE for n, u in zip(lengths, used)]))
        at_page.copy_(torch.stack([own_pages[r][(n - 1) // PAGE] for r, n in enumerate(lengths)]))
        at_slot.copy_(torch.tensor([(n - 1) % PAGE for n in lengths]))
        return lengths

    def decode(lengths, log):
        def rows(layer, q, k, v):
            layer.k.index_put_((at_page, at_slot), k)
            layer.v.index_put_((at_page, at_slot), v)
            if layer.windowed:
                out, _ = layer.decode(q, layer.k, layer.v, both["indptr"], both["pages"], last, SCALE)
            else:
                out, _ = layer.decode(q, layer.k, layer.v, shared, own["indptr"], own["pages"], last, SCALE)
            if log is not None:
                kv = [tuple(torch.cat([gathered(c, shared, COMMON * PAGE), gathered(c, own_pages[r], n)]) for c in (layer.k, layer.v))
                      for r, n in enumerate(lengths)]
                log.append(("decode", out.clone(), (q, [(torch.tensor([r], device="cuda"), *t) for r, t in enumerate(kv)], layer.windowed), None))
            return out
        return rows

    def step(x, lengths=None, log=None):
        for layer in layers:
            x = layer(x, decode(lengths, log), log)
        return x

    start, ran = x.clone(), []
    for i in range(STEPS):
        log = []
        print(f"decoder layers: step {i}", flush=True)
        x = step(x, tables(i), log)
        torch.cuda.synchronize()
        check_log(log)
        ran.append(x.clone())

    held = start.clone()
    tables(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = step(held)
    for _ in range(2):                         # (the steps again, their keys and values written once more)
        held.copy_(start)
        for i in range(STEPS):
            tables(i)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(result, ran[i]), f"replayed step {i}"
            assert torch.equal(step(held.clone()), ran[i])           # an eager step in between
            held.copy_(result)
