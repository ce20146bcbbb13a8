"""How attention with a window and decode over shared pages may be called: captured and replayed beside eager calls, on a stream that is
not the tensors' own, two calls at once, into outputs of the caller with partials in the library's array, empty batches, many
requests, rows behind the last request, and caches whose offsets pass 32 bits."""

import pytest
import torch

from cleave_amd.runtime.compile import _compile
from tests import test_gpu_shared_prefix as S
from tests import test_gpu_window as W
from tests._attention64 import attend, same

pytestmark = pytest.mark.gpu

DECODE_LENS = [333, 0, 64, 1, 900]


def decode_form(**form):
    """(kernel, argument sets by seed, check)"""
    kernel = W.decode_kernel(16, 100, 4, **form)
    return kernel, lambda seed: W.decode_args(DECODE_LENS, 16, seed=seed), lambda k, a: W.check_decode(k, a, DECODE_LENS, 16, 100, 4)


def prompt_form(ragged, ranges):
    kernel = W.prefill_kernel(ragged, 60, 2, ranges=ranges)
    return (kernel, lambda seed: W.prefill_args(ragged, W.NEW, W.KEYS, seed=seed),
            lambda k, a: W.check_prefill(k, a, W.prefill_want(a, ragged, W.NEW, W.KEYS, 60, 2)))


def shared_form(page):
    kernel = S.shared_kernel(page)
    return kernel, lambda seed: S.shared_args(40, DECODE_LENS, page, seed=seed), lambda k, a: S.check(k, a, DECODE_LENS, page)


FORMS = {"decode": lambda: decode_form(), "decode_split": lambda: decode_form(split=8), "decode_items": lambda: decode_form(split=2, ranges=3),
         "prompts_table": lambda: prompt_form(False, 1), "prompts_table_ranges": lambda: prompt_form(False, 3),
         "prompts_packed": lambda: prompt_form(True, 1), "prompts_packed_ranges": lambda: prompt_form(True, 3),
         "shared_pages": lambda: shared_form(16), "shared_tokens": lambda: shared_form(1)}


@pytest.fixture(params=FORMS)
def form(request):
    print(f"operator calls: {request.param}", flush=True)
    return FORMS[request.param]()


def equal(got, want):
    torch.cuda.synchronize()
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_replayed_beside_eager_calls(form):
    kernel, inputs, check = form
    args = [t.clone() if isinstance(t, torch.Tensor) else t for t in inputs(0)]
    other = inputs(9)
    check(kernel, args)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph, operands in zip(graphs, (args, other)):          # two captured graphs, each with scratch of its own
        with torch.cuda.graph(graph):
            outs.append(kernel(*operands))
    for seed in (1, 2, 0):
        for t, fresh in zip(args, inputs(seed)):
            if isinstance(t, torch.Tensor):
                t.copy_(fresh)
        graphs[0].replay()
        graphs[1].replay()
        assert equal(outs[0], kernel(*args)) and equal(outs[1], kernel(*other))
        check(lambda *a: outs[0], args)


def test_on_other_streams_two_at_once(form):
    kernel, inputs, _ = form
    sets = [inputs(seed) for seed in range(4)]
    want = [[t.clone() for t in kernel(*args)] for args in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(3):
        for stream, args in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(kernel(*args))
    torch.cuda.synchronize()
    assert all(equal(g, want[i % len(sets)]) for i, g in enumerate(got))


def test_outputs_of_the_caller_and_the_fixed_array(form):
    kernel, inputs, _ = form
    caller = _compile(kernel.loaded, None)
    for seed in (0, 1):
        args = inputs(seed)
        want = kernel(*args)
        outs = [torch.full_like(t, float("nan")) for t in want]
        caller.call_fixed_scratch(*args, *outs)
        assert equal(outs, want)
        outs = [torch.full_like(t, float("nan")) for t in want]
        caller(*args, *outs)
        assert equal(outs, want)


def test_empty_batches():
    for kernel, args in ((W.decode_kernel(16, 100, 4, split=2, ranges=3), W.decode_args([], 16)), (W.decode_kernel(16, 100, 4), W.decode_args([], 16)),
                         (W.prefill_kernel(True, 60, 2), W.prefill_args(True, [], [])), (W.prefill_kernel(False, 60, 2), W.prefill_args(False, [], [])),
                         (W.prefill_kernel(True, 60, 2, ranges=3), W.prefill_args(True, [0, 0], [0, 5])), (S.shared_kernel(16), S.shared_args(3, [], 16))):
        out, lse = kernel(*args)
        torch.cuda.synchronize()
        assert out.shape[0] == 0 and lse.shape[0] == 0


def test_caches_without_rows():
    """Whatever a table says, a cache of no pages holds no keys: zeros and -inf, and nothing is read."""
    for kernel, args in ((W.decode_kernel(16, 100, 4, split=2, ranges=3), W.decode_args(DECODE_LENS, 16)),
                         (W.decode_kernel(16, 100, 4, split=8), W.decode_args(DECODE_LENS, 16)), (W.decode_kernel(1, 100, 4), W.decode_args(DECODE_LENS, 1)),
                         (W.prefill_kernel(False, 60, 2, ranges=1), W.prefill_args(False, W.NEW, W.KEYS)),
                         (W.prefill_kernel(False, 60, 2, ranges=3), W.prefill_args(False, W.NEW, W.KEYS)),
                         (S.shared_kernel(16), S.shared_args(40, DECODE_LENS, 16)), (S.shared_kernel(1), S.shared_args(40, DECODE_LENS, 1))):
        args[1], args[2] = (t[:0].clone() for t in args[1:3])
        out, lse = kernel(*args)
        torch.cuda.synchronize()
        assert bool((out == 0).all()) and bool((lse == -torch.inf).all())


@pytest.mark.parametrize("ranges", [1, 2])
def test_prompts_of_many_requests(ranges):
    new = [(7 * i) % 5 * (i % 3) for i in range(300)]                        # more requests than a search reads at once, many without tokens
    keys = [n + (13 * i) % 90 for i, n in enumerate(new)]
    args = W.prefill_args(False, new, keys)
    W.check_prefill(W.prefill_kernel(False, 33, 1, ranges=ranges), args, W.prefill_want(args, False, new, keys, 33, 1))


@pytest.mark.parametrize("ranges", [1, 3])
def test_rows_behind_the_last_request_are_left(ranges):
    args = W.prefill_args(True, W.NEW, W.KEYS)
    kernel = W.prefill_kernel(True, 60, 2, ranges=ranges)
    want = W.prefill_want(args, True, W.NEW, W.KEYS, 60, 2)
    rows, more = args[0].shape[0], 150
    args[0] = torch.cat([args[0], torch.randn_like(args[0][:more])])
    out = torch.full_like(args[0], 7.0)
    lse = torch.full(out.shape[:2], 7.0, device="cuda")
    _compile(kernel.loaded, None)(*args, out, lse)
    torch.cuda.synchronize()
    assert bool((out[rows:] == 7).all()) and bool((lse[rows:] == 7).all())
    W.check_prefill(lambda *a: (out[:rows], lse[:rows]), args, want)


# Caches of 2^31 + elements of 16 bits: the requests' tokens lie at both ends.
FAR = (1 << 31) // (8 * 128) + 4096


def far_cache(page):
    pages = -(-FAR // page)
    caches = [torch.zeros(pages, page, 8, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    for cache in caches:
        for part in (cache[:2048 // page], cache[-2048 // page:]):
            part.copy_(torch.randn_like(part))
    return caches, pages


@pytest.mark.parametrize("page", [1, 64])
def test_caches_past_32_bits(page):
    """Decode with a window by splits and by items, and over shared pages: entries of the table from both ends of the cache."""
    (kc, vc), pages = far_cache(page)
    lens = [700, 90]
    count = sum(-(-n // page) for n in lens)
    ends = torch.cat([torch.arange(pages - count, pages, 2), torch.arange(0, count)])[torch.randperm(count + -(-count // 2), generator=torch.Generator().manual_seed(1))]
    table = ends[:count].int().cuda()
    args = W.decode_args(lens, page, hq=32, hkv=8)
    args[1], args[2], args[4] = kc, vc, table
    assert int(table.max()) * page * 8 * 128 > 1 << 31
    for split in (dict(), dict(split=2, ranges=3)):
        print(f"far cache page={page} {split}", flush=True)
        W.check_decode(W.decode_kernel(page, 500, 40, hq=32, hkv=8, **split), args, lens, page, 500, 40)
    args = S.shared_args(8, lens, page, hq=32, hkv=8)
    args[1], args[2], args[5] = kc, vc, table
    args[3] = (pages - 1 - torch.arange(8)).int().cuda()
    S.check(S.shared_kernel(page, hq=32, hkv=8), args, lens, page)


def test_prompts_past_32_bits():
    """Packed queries and keys of more than 2^31 elements: the last request's rows, and a table into the far end of a cache."""
    new, keys, window, sinks = [540000, 140], [FAR - 700, 700], 64, 40       # (32 query heads: 2^31 elements are 524288 rows)
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.zeros(n, h, 128, dtype=torch.bfloat16, device="cuda") for n, h in ((sum(new), 32), (sum(keys), 8), (sum(keys), 8)))
    for t, n in ((q, new[1]), (k, keys[1]), (v, keys[1])):
        t[-n:] = torch.randn(n, *t.shape[1:], generator=gen, device="cuda").bfloat16()
    bounds = [torch.tensor([0, n[0], sum(n)], dtype=torch.int32, device="cuda") for n in (new, keys)]
    scale = 128 ** -0.5
    rows, at = torch.arange(new[1], device="cuda")[:, None] + keys[1] - new[1], torch.arange(keys[1], device="cuda")[None]
    seen = (at <= rows) & ((at > rows - window) | (at < sinks))
    want, want_lse, tol, lse_tol = attend(q[-new[1]:], k[-keys[1]:], v[-keys[1]:], scale, seen)
    print("prompts past 32 bits: packed", flush=True)
    out, lse = W.prefill_kernel(True, window, sinks, hq=32, hkv=8)(q, k, v, *bounds, scale)
    torch.cuda.synchronize()
    same(out[-new[1]:], want, tol, "out")
    same(lse[-new[1]:], want_lse, lse_tol, "lse")
    assert bool((out[:100] == 0).all())                                      # (their values are zeros)
    del out, lse
    for ranges in (1, 3):
        print(f"prompts past 32 bits: table, {ranges} ranges", flush=True)
        table = torch.arange(FAR - 700, FAR, dtype=torch.int32, device="cuda")
        out, lse = W.prefill_kernel(False, window, sinks, hq=32, hkv=8, ranges=ranges)(
            q[-new[1]:].contiguous(), k.unsqueeze(1), v.unsqueeze(1), torch.tensor([0, new[1]], dtype=torch.int32, device="cuda"),
            torch.tensor([0, 700], dtype=torch.int32, device="cuda"), table, scale)
        torch.cuda.synchronize()
        same(out, want, tol, "out")
        same(lse, want_lse, lse_tol, "lse")


@pytest.mark.parametrize("hq,hkv", [(4, 2), (32, 2), (32, 16), (64, 4)])
def test_head_layouts(hq, hkv):
    """Groups of two and of 16, more kv heads than a workgroup has waves."""
    lens = [70, 0, 1, 333]
    args = W.decode_args(lens, 16, hq=hq, hkv=hkv)
    for form in (dict(), dict(split=4), dict(split=2, ranges=-1), dict(split=2, ranges=3, waves=min(hkv, 8))):
        print(f"head layouts {hq}/{hkv} decode {form}", flush=True)
        W.check_decode(W.decode_kernel(16, 50, 3, hq=hq, hkv=hkv, **{"waves": min(hkv, 8) if form.get("ranges") else 4, **form}), args, lens, 16, 50, 3)
    for ragged in (False, True):
        for ranges in (1, 3):
            print(f"head layouts {hq}/{hkv} prompts ragged={ragged} ranges={ranges}", flush=True)
            args = W.prefill_args(ragged, W.NEW, W.KEYS, hq=hq, hkv=hkv)
            W.check_prefill(W.prefill_kernel(ragged, 60, 2, hq=hq, hkv=hkv, ranges=ranges), args, W.prefill_want(args, ragged, W.NEW, W.KEYS, 60, 2))
    for page in (1, 16):
        print(f"head layouts {hq}/{hkv} shared page={page}", flush=True)
        S.check(S.shared_kernel(page, hq=hq, hkv=hkv), S.shared_args(20, lens, page, hq=hq, hkv=hkv), lens, page)
