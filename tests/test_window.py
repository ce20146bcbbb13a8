"""Windows and sinks of paged programs: what is traced, kept and refused, and that the kernels compile."""

import json

import pytest
import torch

import cleave_amd
import cleave_amd.lang as cl
from cleave_amd import examples as C
from cleave_amd.codegen import HipCodeGen
from cleave_amd.core.errors import CodegenError, SpecError
from cleave_amd.dynamic import OPERATORS, reference
from cleave_amd.dynamic.paging import (PAGED_DECODE, RAGGED_PREFILL_CAUSAL, CombineTiling, DenseAttention, PagingSpec, build_split_decode)
from cleave_amd.dynamic.paging.apply import _paged_outputs, _paged_params, _plan, _prefill_plan, window_ranges_expr
from cleave_amd.dynamic.paging.errors import InvalidSpec, UnsupportedTiling
from cleave_amd.frontend.paged import PagedProgram, trace_paged
from cleave_amd.pipeline.dynamic import PagedKernel
from cleave_amd.runtime import shim
from cleave_amd.runtime.compile import code_object_stats, eval_extent


@pytest.mark.parametrize("fn", [C.paged_decode_op(window=100, sinks=4), C.paged_decode_op(page=1, window=7), C.prefill_op(window=64, sinks=1),
                                C.prefill_op(ragged=True, window=64)], ids=lambda f: f.__name__)
def test_traced_and_kept(fn):
    attention = trace_paged(fn).attention()
    spec = attention.paging_spec()
    assert (spec.window, spec.sinks) == (attention.window, attention.sinks) and spec.window
    again = PagedProgram.from_doc(json.loads(json.dumps(attention.program.to_doc()))).attention()
    assert again.paging_spec() == spec


def test_programs_without_a_window_are_recorded_as_before():
    program = trace_paged(C.paged_decode_op())
    softmax = next(op for op in program.oplist if op.kind == "softmax")
    assert dict(softmax.attrs) == {"dim": 3, "causal": False}
    assert "shared" not in program.to_doc()["tables"][0]


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-3), dict(window=2.0), dict(window=True), dict(window=8, sinks=-1), dict(sinks=4),
                                dict(window=8, sinks=1.5)], ids=str)
def test_refused_numbers(kw):
    with pytest.raises(SpecError):
        cl.softmax(torch.zeros(2, 2), **kw)
    with pytest.raises(SpecError):
        trace_paged(C.paged_decode_op(**kw))


def test_refused_places():
    with pytest.raises(SpecError, match="paged program"):
        cl.softmax(torch.zeros(2, 2), window=4)

    @cleave_amd.jit
    def dense(q: cl.Tensor["H", "S", "D"], k: cl.Tensor["H", "T", "D"], v: cl.Tensor["H", "T", "D"]):
        return cl.softmax(q @ k.mT, window=4) @ v

    with pytest.raises(SpecError, match="paged program"):
        dense.trace(cl.f16, H=2, S=16, T=64, D=64)
    op = C.mla_paged_decode_op()
    body = op.fn

    def windowed(qn, qp, ckv_cache, kpe_cache, kv_indptr, kvi, sm_scale):
        pages = cl.PageTable(kv_indptr, kvi)
        c, r = cl.paged_gather(ckv_cache, pages), cl.paged_gather(kpe_cache, pages)
        return cl.softmax((qn @ c.mT + qp @ r.mT) * sm_scale, window=16) @ c

    windowed.__annotations__ = body.__annotations__
    with pytest.raises(SpecError, match="GQA"):
        trace_paged(windowed).attention().paging_spec()


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=1 << 30), dict(sinks=1), dict(window=4, sinks=-1), dict(window=True),
                                dict(window=4, shared_input="S", shared_dim="n"), dict(shared_input="S")], ids=str)
def test_refused_specs(kw):
    with pytest.raises(InvalidSpec):
        PagingSpec(8, 2, kind=PAGED_DECODE, **kw).validate()


def test_a_windowed_program_is_no_operator_of_the_table():
    for name, shipped in OPERATORS.items():
        if name.startswith("gqa_paged_decode_h32_kv8_d128_ps64"):
            assert shipped.matches(trace_paged(C.paged_decode_op(name=name)).attention())
            assert not shipped.matches(trace_paged(C.paged_decode_op(name=name, window=64)).attention())


def _decode_plan(window, sinks=0, d=128, **kw):
    spec = PagingSpec(8, 2, kind=PAGED_DECODE, window=window, sinks=sinks)
    dense = DenseAttention(16, 32, d, 256, "float16", "float16", **kw)
    params, ops = _paged_params(spec, dense)
    outs, out_ops = _paged_outputs(spec, dense)
    return spec, dense, _plan(spec, dense, "main", params + outs, {**ops, **out_ops})


def test_kernels_compile_without_spills():
    spec, dense, plan = _decode_plan(100, 4)
    sources = [HipCodeGen().gen(plan), HipCodeGen().gen(build_split_decode(spec, dense, 4, CombineTiling(split=4)))]
    items = DenseAttention(16, 32, 128, 128, "float16", "float16", waves=2, chunk_pages=-1, lockstep=True)
    sources.append(HipCodeGen().gen(build_split_decode(spec, items, 4, CombineTiling(split=4))))
    prefill = PagingSpec(8, 2, kind=RAGGED_PREFILL_CAUSAL, causal=True, window=100, sinks=4, cache_inputs=("K", "V"))
    for d in (64, 128, 256):
        sources.append(HipCodeGen().gen(_prefill_plan(prefill, DenseAttention(16, 32, d, 128, "bfloat16", "bfloat16", waves=2))))
    for source in sources:
        assert "#define CL_WINDOW 100" in source and "#define CL_SINKS 4" in source
        assert all(k["spilled_vgprs"] == 0 for k in code_object_stats(shim.compile_source(source)[0]))


def test_forms_that_have_no_window_are_refused():
    prefill = PagingSpec(8, 2, kind=RAGGED_PREFILL_CAUSAL, causal=True, window=100, cache_inputs=("K", "V"))
    with pytest.raises(UnsupportedTiling, match="window"):
        _prefill_plan(prefill, DenseAttention(16, 32, 128, 128, "bfloat16", "bfloat16"), shared=False)
    with pytest.raises(UnsupportedTiling, match="window"):
        _prefill_plan(prefill, DenseAttention(16, 32, 384, 128, "bfloat16", "bfloat16"))
    spec = PagingSpec(8, 2, kind=PAGED_DECODE, window=100)
    with pytest.raises(UnsupportedTiling, match="window"):
        build_split_decode(spec, DenseAttention(16, 32, 128, 128, "float16", "float16", waves=2, chunk_pages=-2), 4, CombineTiling(split=4))
    plan = _decode_plan(100)[2]
    plan.tiling["LOCKSTEP"] = 1
    with pytest.raises(CodegenError, match="chunked items"):
        HipCodeGen().gen(plan)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 33), (2048, 0), (5000, 700), (100000, 4)])
@pytest.mark.parametrize("ranges", [-1, 1, 7])
def test_ranges_of_a_window(window, sinks, ranges):
    """Whatever the request's length, a range's rows fit an item's LDS."""
    expr = window_ranges_expr(PagingSpec(8, 2, kind=PAGED_DECODE, window=window, sinks=sinks), ranges)
    for batch in (1, 3, 64, 5000):
        n = eval_extent(expr, {"batch": batch})
        assert n >= 1
        for length in (0, 1, window - 1, window, window + 1, window + sinks, window + 31, window + sinks + 65, 3 * window + 2 * sinks + 5):
            sink_steps = -(-sinks // 32)
            skip = max(0, max(0, length - window) // 32 - sink_steps)
            steps = -(-length // 32) - skip
            assert steps >= 0 and -(-steps // n) * 32 <= 2048
            seen = {t for s in range(steps) for t in range(32 * (s if s < sink_steps else s + skip), 32 * (s if s < sink_steps else s + skip) + 32)}
            assert all(t in seen for t in range(length) if t >= length - window or t < sinks)


def test_dispatch_counts_the_tokens_that_are_seen():
    kernel = PagedKernel.__new__(PagedKernel)
    kernel.name, kernel.dispatch_sources = "op", {"split": "", "single": ""}
    kernel.dispatch = {"min_tiles": 10, "lone_tiles": 10, "few_requests": 0, "kv_tile": 32, "page_size": 64, "seen_tokens": 200}
    assert kernel.dispatch_role(1000) == "single"
    kernel.dispatch["seen_tokens"] = 2000
    assert kernel.dispatch_role(1000) == "split"


def test_reference_of_a_window():
    """Against the mask written out, for requests shorter and longer than the window."""
    lens = [3, 40, 7]
    dims = (3, 4, 2, 64, 50, 50)
    args = reference.gqa_paged_decode_inputs(dims, lens, dtype=torch.float32, device="cpu")
    out, lse = reference.gqa_paged_decode_reference(dims, lens, dtype=torch.float32, window=6, sinks=2)(*args)
    for b, n in enumerate(lens):
        rows = args[4][int(args[3][b]):int(args[3][b + 1])].long()
        seen = [j for j in range(n) if j >= n - 6 or j < 2]
        for h in range(4):
            k, v = args[1][rows[seen], 0, h // 2], args[2][rows[seen], 0, h // 2]
            logits = k.double() @ args[0][b, h].double() * args[-1]
            torch.testing.assert_close(out[b, h].double(), torch.softmax(logits, 0) @ v.double(), rtol=1e-5, atol=1e-5)
            assert abs(float(lse[b, h]) - float(torch.logsumexp(logits, 0)) / 0.6931471805599453) < 1e-5


def test_prompt_workloads():
    mix = cl.workloads.causal_prefill(batch=(1, 3), q_len=(4, 100), prefix=(5, 9), samples=2)
    for batch, q_len in mix.axes():
        new, keys = mix.lengths(batch, q_len)
        assert len(new) == batch and max(new) == q_len and all(5 <= m - n <= 9 for n, m in zip(new, keys))
    with pytest.raises(SpecError):
        mix.factory(trace_paged(C.paged_decode_op()).attention())
