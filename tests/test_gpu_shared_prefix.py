"""GPU parity of decode over pages that a batch shares, against the definition in 64 bits."""

import math

import pytest
import torch

import cleave_amd
import cleave_amd.lang as cl
from cleave_amd import examples as C
from cleave_amd import pipeline as P
from cleave_amd.codegen import HipCodeGen
from cleave_amd.dynamic import reference as dref
from cleave_amd.dynamic.paging import PAGED_DECODE, PAGED_DECODE_SLAB, DenseAttention, PagingSpec
from cleave_amd.dynamic.paging.apply import _shared_plan
from cleave_amd.runtime.compile import _compile, _load_main_kernel_from_code
from tests._attention64 import attend, same

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def poisoned(monkeypatch):
    """Fresh outputs and scratch begin as NaN: a partial that nobody writes is seen."""
    monkeypatch.setenv("CLEAVE_POISON_BUFFERS", "1")


def shared_kernel(page, hq=8, hkv=2, d=128, dtype="float16", lse=True):
    spec = PagingSpec(hq, hkv, kind=PAGED_DECODE_SLAB if page > 1 else PAGED_DECODE, page_size=page, emit_lse=lse, shared_input="SHARED",
                      shared_dim="n_shared")
    spec.validate()
    loaded = _load_main_kernel_from_code(HipCodeGen().gen(_shared_plan(spec, DenseAttention(-(-hq // hkv // 16) * 16, 32, d, 256, dtype, dtype))))
    return _compile(loaded, loaded.manifest["out_idx"])


def shared_args(shared, lens, page, hq=8, hkv=2, d=128, dtype=torch.float16, seed=0):
    pages = sum(-(-n // page) for n in lens)
    args = dref.gqa_paged_decode_inputs((len(lens), hq, hkv, d, shared + pages + 3, pages), lens, page_size=page, dtype=dtype, seed=seed, shared=shared)
    if not shared:
        args.insert(3, torch.empty(0, dtype=torch.int32, device="cuda"))
    return args


def shared_want(args, lens, page):
    q, kc, vc, first, indptr, table = args[:6]
    results = []
    for b, n in enumerate(lens):
        own = dref.paged_tokens(table, int(indptr[b]), n, page)
        both = [torch.cat(t) for t in zip(dref.paged_tokens(first, 0, first.numel() * page, page), own)]
        results.append(attend(q[b:b + 1], kc[both[0], both[1]], vc[both[0], both[1]], args[-1]))
    return [torch.cat(t) for t in zip(*results)]


def check(kernel, args, lens, page):
    out, lse = kernel(*args)
    torch.cuda.synchronize()
    want, want_lse, tol, lse_tol = shared_want(args, lens, page)
    same(out, want, tol, "out")
    same(lse, want_lse, lse_tol, "lse")


@pytest.mark.parametrize("page", [1, 16, 64])
@pytest.mark.parametrize("shared", [1, 2, 31, 33, 70])
@pytest.mark.parametrize("lens", [[1], [0], [5, 0, 33], [64, 1, 200, 0, 17] * 9], ids=lambda v: f"{len(v)}x{max(v)}")
def test_shared_pages(page, shared, lens):
    print(f"shared prefix page={page} shared={shared} lens={lens}", flush=True)
    check(shared_kernel(page), shared_args(shared, lens, page), lens, page)


@pytest.mark.parametrize("page", [1, 64])
def test_nothing_shared(page):
    """No shared page: plain paged decode; and neither shared nor own keys: zeros and -inf."""
    for lens in ([70, 1, 129], [0, 40, 0]):
        print(f"shared prefix page={page} nothing shared {lens}", flush=True)
        check(shared_kernel(page), shared_args(0, lens, page), lens, page)


@pytest.mark.parametrize("kw", [dict(hq=32, hkv=8), dict(hq=10, hkv=2), dict(hq=40, hkv=2), dict(hq=6, hkv=3, d=64), dict(hq=4, hkv=2, d=256),
                                dict(hq=32, hkv=4, dtype="bfloat16")], ids=lambda kw: "_".join(f"{k}{v}" for k, v in kw.items()))
@pytest.mark.parametrize("page", [1, 64])
def test_forms(kw, page):
    shape = {k: v for k, v in kw.items() if k != "dtype"}
    lens = [3, 150, 0, 40, 64, 9, 1] * 6
    print(f"shared prefix {kw} page={page}", flush=True)
    args = shared_args(700 // page, lens, page, dtype=getattr(torch, kw.get("dtype", "float16")), **shape)
    check(shared_kernel(page, **kw), args, lens, page)


@pytest.mark.parametrize("page,shared,lens", [(1, 5000, [700, 30]), (64, 129, [900, 1, 64] * 30), (64, 3, [65] * 300)])
def test_longer(page, shared, lens):
    print(f"shared prefix page={page} shared={shared} requests={len(lens)}", flush=True)
    check(shared_kernel(page, hq=32, hkv=8), shared_args(shared, lens, page, hq=32, hkv=8), lens, page)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
def test_scales(scale):
    lens = [40, 0, 100]
    args = shared_args(90, lens, 1)
    args[-1] = scale
    print(f"shared prefix scale={scale}", flush=True)
    check(shared_kernel(1), args, lens, 1)


def test_pages_that_are_named_twice_and_numbers_outside_the_cache():
    """A page may be shared and owned, or owned by two requests; page numbers past the cache read its last or first page."""
    lens, page = [130, 64, 20], 64
    args = shared_args(3, lens, page)
    args[5][1] = args[3][0]
    args[5][3] = args[5][0]
    print("shared prefix: pages named twice", flush=True)
    check(shared_kernel(page), args, lens, page)
    wild = [t.clone() if isinstance(t, torch.Tensor) else t for t in args]
    wild[3][1], wild[5][0] = 1 << 30, -7
    args[3][1], args[5][0] = args[1].shape[0] - 1, 0
    for a, b in zip(shared_kernel(page)(*wild), shared_kernel(page)(*args)):
        assert torch.equal(a, b)


def test_infinite_values_of_either_part():
    """An infinite value shows where its key has a weight: a shared one in every request, an own one in its request."""
    lens, page = [50, 7, 120], 1
    args = shared_args(200, lens, page)
    args[2][args[3][77], 0, 1, 5] = math.inf
    args[2][args[5][60], 0, 0, 9] = -math.inf                 # the third request's
    print("shared prefix: infinite values", flush=True)
    check(shared_kernel(page), args, lens, page)
    args[1][args[5][3], 0, 0, 0] = math.nan                   # a key of the first request's own
    check(shared_kernel(page), args, lens, page)
    args[1][args[3][1], 0, 1, 0] = math.nan                   # a shared one
    check(shared_kernel(page), args, lens, page)


def test_replayed_beside_eager_calls():
    kernel = shared_kernel(64, hq=32, hkv=8)
    lens = [100, 3, 64, 0]
    sets = [shared_args(20, lens, 64, hq=32, hkv=8, seed=s) for s in range(3)]
    args = [t.clone() if isinstance(t, torch.Tensor) else t for t in sets[0]]
    kernel(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernel(*args)
    for fresh in sets:
        for t, f in zip(args, fresh):
            if isinstance(t, torch.Tensor):
                t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, kernel(*args)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("page", [1, 64])
def test_compiled(cache_root, monkeypatch, page):
    monkeypatch.delenv("CLEAVE_POISON_BUFFERS")
    mix = cl.workloads.paged_decode(batch=(1, 5), kv_len=(1, 300), samples=2, prefix=500)
    kernel = cleave_amd.compile(C.shared_prefix_decode_op(8, 2, 128, page), split=cl.Split("kv_len", (4,)), workloads=mix,
                                schedule=P.ScheduleConfig(topk=1), max_workloads=2)
    assert not kernel.report.failures
    lens = [333, 1, 0, 90]
    args = shared_args(500 // page + 1, lens, page)
    check(kernel, args, lens, page)
    check(kernel, args, lens, page)                             # (the native call)
    again = cleave_amd.load(kernel.save(cache_root / "kernel"))
    for a, b in zip(again(*args), kernel(*args)):
        assert torch.equal(a, b)
