"""GPU parity of attention with a window and sinks against the definition in 64 bits: decode over token tables and pages, single
and split; prompts over packed keys and token tables; windows and sinks around the 32-key step, requests around the window."""

import math

import pytest
import torch

import cleave_amd
import cleave_amd.lang as cl
from cleave_amd import examples as C
from cleave_amd import pipeline as P
from cleave_amd.codegen import HipCodeGen
from cleave_amd.dynamic import reference as dref
from cleave_amd.dynamic.paging import (PAGED_DECODE, PAGED_DECODE_SLAB, PAGED_PREFILL_CAUSAL, RAGGED_PREFILL_CAUSAL, CombineTiling,
                                       DenseAttention, PagingSpec, build_split_decode)
from cleave_amd.dynamic.paging.apply import _paged_outputs, _paged_params, _plan, _prefill_plan
from cleave_amd.runtime.compile import _compile, _load_main_kernel_from_code
from tests._attention64 import attend, same

pytestmark = pytest.mark.gpu


def compiled(source):
    loaded = _load_main_kernel_from_code(source)
    return _compile(loaded, loaded.manifest["out_idx"])


# ------------------------------------------------------------------------------------------------ decode
def decode_kernel(page, window, sinks, hq=8, hkv=2, d=128, dtype="float16", waves=4, split=None, prefetch=1, skew=0, ranges=0, lockstep=True):
    spec = PagingSpec(hq, hkv, kind=PAGED_DECODE_SLAB if page > 1 else PAGED_DECODE, page_size=page, window=window, sinks=sinks)
    spec.validate()
    dense = DenseAttention(-(-hq // hkv // 16) * 16, 32, d, waves * 64, dtype, dtype, waves=waves, prefetch=prefetch, skew=skew,
                           chunk_pages=ranges, lockstep=lockstep and ranges != 0)
    if split:
        return compiled(HipCodeGen().gen(build_split_decode(spec, dense, split, CombineTiling(split=split, cols=min(128, d)))))
    params, ops = _paged_params(spec, dense)
    outs, out_ops = _paged_outputs(spec, dense)
    return compiled(HipCodeGen().gen(_plan(spec, dense, "main", params + outs, {**ops, **out_ops})))


def decode_args(lens, page, hq=8, hkv=2, d=128, dtype=torch.float16, seed=0):
    pages = sum(-(-n // page) for n in lens)
    return dref.gqa_paged_decode_inputs((len(lens), hq, hkv, d, pages + 3, pages), lens, page_size=page, dtype=dtype, seed=seed)


def decode_want(args, lens, page, window, sinks):
    q, kc, vc, indptr, table = args[:5]
    results = []
    for b, n in enumerate(lens):
        page_of, slot = dref.paged_tokens(table, int(indptr[b]), n, page)
        at = torch.arange(n, device=q.device)
        seen = (at >= n - window) | (at < sinks)
        results.append(attend(q[b:b + 1], kc[page_of, slot], vc[page_of, slot], args[-1], seen[None]))
    return [torch.cat(t) for t in zip(*results)]


def check_decode(kernel, args, lens, page, window, sinks):
    out, lse = kernel(*args)
    torch.cuda.synchronize()
    want, want_lse, tol, lse_tol = decode_want(args, lens, page, window, sinks)
    same(out, want, tol, "out")
    same(lse, want_lse, lse_tol, "lse")


LENS = [1, 5, 31, 32, 33, 64, 65, 100, 0, 333, 129, 1000]


@pytest.mark.parametrize("page,split", [(1, None), (64, None), (1, 8), (16, 8)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 32), (64, 33), (100, 100), (97, 1), (2000, 4), (40, 400)])
def test_decode(page, split, window, sinks):
    print(f"window decode page={page} split={split} window={window} sinks={sinks}", flush=True)
    check_decode(decode_kernel(page, window, sinks, split=split), decode_args(LENS, page), LENS, page, window, sinks)


@pytest.mark.parametrize("page,ranges", [(1, -1), (64, -1), (16, 1), (64, 5)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 32), (64, 33), (100, 100), (97, 1), (2000, 4), (40, 400)])
def test_decode_by_items(page, ranges, window, sinks):
    """What is seen in equal parts by workgroups of one wave per kv head; more parts than steps leave some empty."""
    print(f"window decode by items page={page} ranges={ranges} window={window} sinks={sinks}", flush=True)
    check_decode(decode_kernel(page, window, sinks, split=2, ranges=ranges), decode_args(LENS, page), LENS, page, window, sinks)


@pytest.mark.parametrize("kw", [dict(hq=24, hkv=12), dict(hq=9, hkv=3), dict(hq=40, hkv=2), dict(d=64), dict(d=256, hq=6), dict(hq=32, hkv=8, dtype="bfloat16"),
                                dict(hq=32, hkv=8, lockstep=False), dict(prefetch=2)], ids=lambda kw: "_".join(f"{k}{v}" for k, v in kw.items()))
def test_decode_by_items_forms(kw):
    lens = [70, 3, 900, 129, 0]
    shape = {k: v for k, v in kw.items() if k in ("hq", "hkv", "d")}
    for page in (1, 64):
        print(f"window decode by items {kw} page={page}", flush=True)
        args = decode_args(lens, page, dtype=getattr(torch, kw.get("dtype", "float16")), **shape)
        check_decode(decode_kernel(page, 130, 5, split=2, ranges=-1, **kw), args, lens, page, 130, 5)


def test_decode_window_of_many_items():
    """A window of more rows than an item's LDS holds."""
    lens, window, sinks = [9000, 5000, 4], 4500, 700
    args = decode_args(lens, 16)
    print("window decode by items of a long window", flush=True)
    check_decode(decode_kernel(16, window, sinks, split=2, ranges=1), args, lens, 16, window, sinks)


@pytest.mark.parametrize("kw", [dict(waves=1), dict(waves=2, prefetch=2), dict(waves=8, split=2), dict(waves=1, split=4, hkv=8, hq=32, skew=30),
                                dict(d=64), dict(d=256, hq=6, waves=2), dict(dtype="bfloat16", hq=16, hkv=2, split=3), dict(hq=40, hkv=2)],
                         ids=lambda kw: "_".join(f"{k}{v}" for k, v in kw.items()))
def test_decode_forms(kw):
    lens = [70, 3, 900, 129]
    shape = {k: v for k, v in kw.items() if k in ("hq", "hkv", "d")}
    for page in (1, 64):
        print(f"window decode {kw} page={page}", flush=True)
        args = decode_args(lens, page, dtype=getattr(torch, kw.get("dtype", "float16")), **shape)
        check_decode(decode_kernel(page, 130, 5, **kw), args, lens, page, 130, 5)


@pytest.mark.parametrize("page", [1, 64])
@pytest.mark.parametrize("split,ranges", [(None, 0), (8, 0), (2, -1), (2, 3)])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_decode_never_reads_what_is_not_seen(page, split, ranges, value):
    """Keys and values outside window and sinks are undefined: pages that a server has handed on to other requests."""
    lens, window, sinks = [700, 90, 333], 100, 3
    args = decode_args(lens, page)
    want = decode_want(args, lens, page, window, sinks)
    for b, n in enumerate(lens):
        page_of, slot = dref.paged_tokens(args[4], int(args[3][b]), n, page)
        hidden = torch.arange(n, device="cuda")
        hidden = hidden[(hidden < n - window) & (hidden >= sinks)]
        for cache in args[1:3]:
            cache[page_of[hidden], slot[hidden]] = value
    print(f"window decode hidden={value} page={page} split={split} ranges={ranges}", flush=True)
    out, lse = decode_kernel(page, window, sinks, split=split, ranges=ranges)(*args)
    same(out, want[0], want[2], "out")
    same(lse, want[1], want[3], "lse")


@pytest.mark.parametrize("page", [1, 64])
@pytest.mark.parametrize("split,ranges", [(None, 0), (8, 0), (2, -1), (2, 3)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_decode_values_that_are_not_finite(page, split, ranges, value):
    """A seen value shows in its feature of its kv head's rows; a seen key that is undefined makes them undefined."""
    lens, window, sinks = [700, 90, 333], 100, 3
    args = decode_args(lens, page)
    for b, (position, head, feature) in enumerate(((650, 0, 5), (1, 1, 9), (333 - 100, 1, 127))):
        page_of, slot = dref.paged_tokens(args[4], int(args[3][b]), lens[b], page)
        args[2][page_of[position], slot[position], head, feature] = value
        if b == 2 and math.isnan(value):
            args[1][page_of[position + 1], slot[position + 1], 0, 3] = value
    print(f"window decode not finite {value} page={page} split={split} ranges={ranges}", flush=True)
    check_decode(decode_kernel(page, window, sinks, split=split, ranges=ranges), args, lens, page, window, sinks)


def test_decode_window_of_everything_is_plain_decode():
    lens = [200, 1, 0, 77]
    args = decode_args(lens, 64, hq=32, hkv=8)
    from tests.test_gpu_paged import paged_kernel

    for a, b in zip(decode_kernel(64, 4096, 0, hq=32, hkv=8)(*args), paged_kernel()(*args)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ prompts
def prefill_kernel(ragged, window, sinks, hq=8, hkv=2, d=128, dtype="bfloat16", ranges=-1):
    kind = RAGGED_PREFILL_CAUSAL if ragged else PAGED_PREFILL_CAUSAL
    spec = PagingSpec(hq, hkv, kind=kind, causal=True, window=window, sinks=sinks, **(dict(cache_inputs=("K", "V")) if ragged else {}))
    spec.validate()
    return compiled(HipCodeGen().gen(_prefill_plan(spec, DenseAttention(16, 32, d, hkv * 64, dtype, dtype, waves=hkv), ranges=ranges)))


def prefill_args(ragged, new, keys, hq=8, hkv=2, d=128, dtype=torch.bfloat16, seed=0):
    if ragged:
        return dref.gqa_ragged_prefill_inputs((hq, hkv, d, sum(new), sum(keys)), new, keys, dtype=dtype, seed=seed)
    return dref.gqa_paged_prefill_inputs((hq, hkv, d, sum(keys) + 7, sum(keys) + 2, sum(new)), new, keys, dtype=dtype, seed=seed)


def prefill_want(args, ragged, new, keys, window, sinks):
    results, at_q, at_k = [], 0, 0
    for n, m in zip(new, keys):
        rows = torch.arange(at_k, at_k + m, device="cuda")
        k, v = (args[1][rows], args[2][rows]) if ragged else (t[args[5][rows].long(), 0] for t in args[1:3])
        own = torch.arange(n, device="cuda")[:, None] + (m - n)
        key = torch.arange(m, device="cuda")[None, :]
        seen = (key <= own) & ((key > own - window) | (key < sinks))
        results.append(attend(args[0][at_q:at_q + n], k, v, args[-1], seen))
        at_q, at_k = at_q + n, at_k + m
    return [torch.cat(t) for t in zip(*results)]


def check_prefill(kernel, args, want):
    out, lse = kernel(*args)
    torch.cuda.synchronize()
    same(out, want[0], want[2], "out")
    same(lse, want[1], want[3], "lse")


NEW = [1, 4, 5, 33, 0, 64, 7, 130, 300]
KEYS = [1, 40, 5, 33, 9, 200, 3, 130, 1000]      # equal, cached keys, no queries, fewer keys than queries


@pytest.mark.parametrize("ragged,ranges", [(False, -1), (True, -1), (False, 1), (True, 1), (False, 7), (True, 2)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (31, 0), (32, 4), (33, 32), (64, 33), (100, 0), (97, 100), (5000, 4), (40, 500)])
def test_prefill(ragged, ranges, window, sinks):
    print(f"window prefill ragged={ragged} ranges={ranges} window={window} sinks={sinks}", flush=True)
    args = prefill_args(ragged, NEW, KEYS)
    check_prefill(prefill_kernel(ragged, window, sinks, ranges=ranges), args, prefill_want(args, ragged, NEW, KEYS, window, sinks))


@pytest.mark.parametrize("kw", [dict(hq=16, hkv=2), dict(hq=4, hkv=2), dict(d=64), dict(d=256), dict(dtype="float16", hq=32, hkv=8)],
                         ids=lambda kw: "_".join(f"{k}{v}" for k, v in kw.items()))
@pytest.mark.parametrize("ranges", [1, 3])
@pytest.mark.parametrize("ragged", [False, True], ids=["table", "packed"])
def test_prefill_forms(kw, ragged, ranges):
    new, keys = [150, 3, 70], [150, 900, 333]
    shape = {k: v for k, v in kw.items() if k != "dtype"}
    args = prefill_args(ragged, new, keys, dtype=getattr(torch, kw.get("dtype", "bfloat16")), **shape)
    print(f"window prefill {kw} ragged={ragged}", flush=True)
    check_prefill(prefill_kernel(ragged, 77, 3, ranges=ranges, **kw), args, prefill_want(args, ragged, new, keys, 77, 3))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("ranges", [1, 3])
@pytest.mark.parametrize("ragged", [False, True], ids=["table", "packed"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_prefill_values_that_are_not_finite(ragged, ranges, value, dtype):
    """Such a value shows in the rows that see its key and in no other, whichever of them share its tile; a key that is not finite
    makes the rows undefined that see it."""
    new, keys, window, sinks = [150, 3, 70], [150, 900, 333], 50, 3
    args = prefill_args(ragged, new, keys, dtype=dtype)
    at = torch.arange(sum(keys), device="cuda") if ragged else args[5].long()
    k, v = (t if ragged else t[:, 0] for t in args[1:3])
    for position, head, feature in ((1, 0, 5), (60, 1, 9), (149, 0, 127), (150 + 897, 1, 64), (150 + 500, 0, 3), (1050 + 280, 1, 1)):
        v[at[position], head, feature] = value
    if math.isnan(value):
        k[at[100], 0, 7] = value
    print(f"window prefill not finite {value} ragged={ragged} ranges={ranges}", flush=True)
    check_prefill(prefill_kernel(ragged, window, sinks, ranges=ranges, dtype=str(dtype)[6:]), args, prefill_want(args, ragged, new, keys, window, sinks))


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_prefill_never_reads_what_no_row_of_an_item_sees(value):
    """Through a table: entries of tokens ahead of the window lead to rows that are somebody else's by now."""
    new, keys, window, sinks = [40, 9], [700, 333], 100, 3
    args = prefill_args(False, new, keys)
    want = prefill_want(args, False, new, keys, window, sinks)
    base = 0
    for n, m in zip(new, keys):
        hidden = args[5][base + sinks:base + m - n - window + 1].long()
        args[1][hidden], args[2][hidden] = value, value
        base += m
    check_prefill(prefill_kernel(False, window, sinks), args, want)


def test_prefill_window_of_everything_is_plain_prefill():
    new, keys = [150, 3, 70], [150, 900, 333]
    args = prefill_args(True, new, keys, hq=32, hkv=8)
    from tests.test_gpu_prefill import prefill_kernel as plain

    for a, b in zip(prefill_kernel(True, 4096, 0, hq=32, hkv=8, ranges=1)(*args), plain(True, shared=True)(*args)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ through compile
def test_compiled_decode(cache_root):
    mix = cl.workloads.paged_decode(batch=(1, 4), kv_len=(30, 700), samples=2)
    fn = C.paged_decode_op(8, 2, 128, 16, window=100, sinks=4)
    kernel = cleave_amd.compile(fn, split=cl.Split("kv_len", (4,)), workloads=mix, schedule=P.ScheduleConfig(topk=1), max_workloads=2)
    assert not kernel.report.failures
    lens = [333, 1, 90]
    args = decode_args(lens, 16)
    for options in ({}, {"longest": 21}, {"longest": 1}):
        check_decode(lambda *a: kernel(*a, **options), args, lens, 16, 100, 4)
    again = cleave_amd.load(kernel.save(cache_root / "kernel"))
    assert again.attention.window == 100 and again.attention.sinks == 4
    for a, b in zip(again(*args), kernel(*args)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("ragged", [False, True], ids=["table", "packed"])
def test_compiled_prefill(ragged):
    mix = cl.workloads.causal_prefill(batch=(1, 3), q_len=(3, 200), prefix=(0, 300), samples=2)
    kernel = cleave_amd.compile(C.prefill_op(8, 2, 128, ragged=ragged, window=60, sinks=2), workloads=mix, schedule=P.ScheduleConfig(topk=1),
                                max_workloads=2)
    assert not kernel.report.failures
    args = prefill_args(ragged, NEW, KEYS)
    check_prefill(kernel, args, prefill_want(args, ragged, NEW, KEYS, 60, 2))


@pytest.mark.parametrize("ragged", [False, True], ids=["table", "packed"])
def test_a_request_has_the_same_bits_in_any_company(ragged):
    kernel = prefill_kernel(ragged, 60, 2, ranges=1)
    args = prefill_args(ragged, NEW, KEYS)
    out, lse = kernel(*args)
    at_q, at_k = 0, 0
    for n, m in zip(NEW, KEYS):
        bounds = [torch.tensor([0, x], dtype=torch.int32, device="cuda") for x in (n, m)]
        keys = [t[at_k:at_k + m] for t in args[1:3]] if ragged else args[1:3]
        alone = kernel(args[0][at_q:at_q + n], *keys, *bounds, *([] if ragged else [args[5][at_k:at_k + m]]), args[-1])
        assert torch.equal(alone[0], out[at_q:at_q + n]) and torch.equal(alone[1], lse[at_q:at_q + n])
        at_q, at_k = at_q + n, at_k + m
