"""Products with an epilogue: what is recognised, what is refused, and that every form of the kernels compiles."""

import pytest
import torch

import cleave_amd
import cleave_amd.lang as cl
from cleave_amd import examples as C
from cleave_amd.core.errors import LoweringRejected, SpecError
from cleave_amd.lower.stages import split_stages
from cleave_amd.pipeline.direct import source_for, stage_graph
from cleave_amd.runtime import reference, shim

SIZES = dict(M=16, N=64, K=128)


def lowered(fn, dtype=cl.f16, **sizes):
    return stage_graph(fn.trace(dtype, **(sizes or SIZES))).lowered


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M", [1, 16])
def test_recognised(act, bias, residual, M):
    low = lowered(C.linear_op(act, residual=residual, bias=bias), M=M, N=64, K=128)
    assert low.family == "matmul"
    want = {"act": act or "none", "bias": bias, "res": residual}
    if M == 1 and act is None and bias != residual:            # (one row added to one row: either name is right)
        assert sum(low.problem["epilogue"][k] for k in ("bias", "res")) == 1
    elif act is None and not bias and not residual:
        assert "epilogue" not in low.problem
    else:
        assert low.problem["epilogue"] == want
        assert set(low.operands) == {"A", "B", *(["BIAS"] if bias else []), *(["RES"] if residual else [])}


def test_addends_in_any_order():
    @cleave_amd.jit
    def swapped(x: cl.Tensor["M", "K"], w: cl.Tensor["K", "N"], b: cl.Tensor[1, "N"], r: cl.Tensor["M", "N"]):
        return b + (r + x @ w)

    low = lowered(swapped)
    assert low.operands["BIAS"].name.endswith("_b") and low.operands["RES"].name.endswith("_r")


def refused(body, **notes):
    body.__annotations__ = notes
    used = {d.name for spec in notes.values() for d in spec.dims if hasattr(d, "name")}
    with pytest.raises(LoweringRejected):
        lowered(cleave_amd.jit(body), **{k: v for k, v in SIZES.items() if k in used})


MK, KN, ROW, MN = cl.Tensor["M", "K"], cl.Tensor["K", "N"], cl.Tensor[1, "N"], cl.Tensor["M", "N"]


def test_refused_forms():
    refused(lambda x, w, r: cl.relu(x @ w + r), x=MK, w=KN, r=MN)                     # a residual ahead of the activation
    refused(lambda x, w, b: cl.relu(x @ w) + b, x=MK, w=KN, b=ROW)                    # a row behind it
    refused(lambda x, w, r, s: x @ w + r + s, x=MK, w=KN, r=MN, s=MN)                 # two residuals
    refused(lambda x, w, b, c: cl.gelu(x @ w + b + c), x=MK, w=KN, b=ROW, c=ROW)      # two rows
    refused(lambda x, w, b: cl.gelu(cl.silu(x @ w + b)), x=MK, w=KN, b=ROW)           # two activations
    refused(lambda x, w, b: x @ w + b, x=MK, w=KN, b=cl.Tensor[1, "N", cl.f32])       # a bias of another type
    refused(lambda x, w, b: (x @ w + b) * 2.0, x=MK, w=KN, b=ROW)
    refused(lambda x, b: x @ x + b, x=cl.Tensor["M", "M"], b=cl.Tensor[1, "M"])


def test_gelu_takes_two_forms():
    with pytest.raises(SpecError):
        @cleave_amd.jit
        def op(x: MK, w: KN):
            return cl.gelu(x @ w, approximate="sigmoid")

        op.trace(cl.f16, **SIZES)
    x = torch.randn(8)
    assert torch.equal(cl.gelu(x, approximate="tanh"), torch.nn.functional.gelu(x, approximate="tanh"))
    assert torch.equal(cl.relu(x), x.clamp_min(0))


@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh", "silu", "relu"])
def test_split_reference_is_the_unsplit_one(act):
    """Partial sums and a combine that finishes them give what the whole product gives (f32 sums of 16-bit products of 128 terms of
    either order differ by less than the two rounded results' steps)."""
    g = stage_graph(C.linear_op(act, residual=True).trace(cl.f16, **SIZES))
    whole = reference.make_inputs(g, device="cpu", seed=1)
    partial, combine = split_stages(g, 2)
    parts = reference.execute(partial, whole)
    feed = [*parts, whole[2], whole[3]]
    assert [p.name for p in combine.placeholders][1:] == ["PlaceHolder_b", "PlaceHolder_r"]
    a, b = reference.execute(combine, feed)[0], reference.execute(g, whole)[0]
    torch.testing.assert_close(a, b, rtol=2.0 ** -10, atol=2.0 ** -14)


@pytest.mark.parametrize("template,tiling,split,sizes,form", [
    ("skinny", dict(WAVES_N=1, WAVES_K=2), None, dict(M=16, N=72, K=128), {}), ("skinny", dict(WAVES_N=1, WAVES_K=2), 2, dict(M=16, N=72, K=128), {}),
    ("gemm", dict(BM=64, BN=64, BK=64, WM=2, WN=2), None, dict(M=70, N=72, K=128), {}),
    ("gemm_dma", dict(BM=64, BN=64, BK=64, WM=2, WN=2), None, dict(M=70, N=70, K=128), dict(transposed=True)),
    ("gemm_dma", dict(BM=256, BN=256, BK=64, WM=2, WN=4), None, dict(M=300, N=264, K=192), {}),
    ("gemm_dma", dict(BM=32, BN=32, BK=64, WM=1, WN=1, KW=4), None, dict(M=32, N=64, K=1024), {}),
    ("gemm_dma", dict(BM=128, BN=256, BK=64, WM=2, WN=4, KS=2), None, dict(M=128, N=256, K=1024), {})])
def test_every_form_compiles(template, tiling, split, sizes, form):
    source = source_for(C.linear_op("gelu", residual=True, **form).trace(cl.bf16, **sizes), template=template, tiling=tiling, split=split)
    assert "#define CL_EPI_ACT 3" in source
    from cleave_amd.runtime.compile import code_object_stats

    code, log = shim.compile_source(source)
    assert all(entry["spilled_vgprs"] == 0 for entry in code_object_stats(code))
