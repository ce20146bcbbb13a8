"""GPU parity of products with an epilogue, ``act(x @ w + bias) + residual``, against the definition in 64 bits.

Tolerances: the f32 sum of K products of 16-bit values is off by at most K 2^-24 times the sum of their magnitudes; every activation
has a slope of at most 1.13 and is taken with a relative error below 2e-6 (reciprocal and exponential of a unit in the last place
each, the fitted tail 4e-7); the one rounding of the result is off by half a step."""

import pytest
import torch

import cleave_amd
import cleave_amd.lang as cl
from cleave_amd import examples as C
from cleave_amd import pipeline as P
from cleave_amd.pipeline.direct import kernel_for

pytestmark = pytest.mark.gpu

ACTS = (None, "relu", "silu", "gelu", "gelu_tanh")
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def act64(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    return z


def inputs(M, N, K, dtype, *, bias=True, residual=False, transposed=False, seed=0, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(scale, *shape):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    args = [normal(1.0, M, K), normal(spread * K ** -0.5, *((N, K) if transposed else (K, N)))]
    return args + ([normal(spread, 1, N)] if bias else []) + ([normal(1.0, M, N)] if residual else [])


def check(out, args, act, *, bias=True, residual=False, transposed=False):
    x, w = args[0].double(), args[1].double()
    w = w.t() if transposed else w
    z, size = x @ w, x.abs() @ w.abs()
    if bias:
        z = z + args[2].double()
        size = size + args[2].double().abs()
    y = act64(z, act)
    want = y + args[-1].double() if residual else y
    slack = 1.13 * (x.shape[1] + 2) * 2.0 ** -24 * size + 2e-6 * y.abs() + 2.0 ** -23 * want.abs()
    tol = slack + HALF_STEP[out.dtype] * (want.abs() + slack) + (2.0 ** -25 if out.dtype == torch.float16 else 0)
    off = (out.double() - want).abs()
    assert out.dtype == args[0].dtype and bool((off <= tol).all()), \
        f"off by up to {(off / tol).max().item():.2f} of the tolerance at {(off / tol).argmax().item()}"


def run(M, N, K, dtype=cl.f16, act="gelu", template=None, tiling=None, split=None, seed=0, **form):
    prog = C.linear_op(act, **form).trace(dtype, M=M, N=N, K=K)
    args = inputs(M, N, K, dtype.torch, seed=seed, **form)
    print(f"linear {prog.name} {dtype} {M}x{N}x{K} {template} {tiling} split={split}", flush=True)
    out = kernel_for(prog, template=template, tiling=tiling, split=split)(*args)
    torch.cuda.synchronize()
    check(out, args, act, **form)


FORMS = [dict(bias=True, residual=False), dict(bias=True, residual=True), dict(bias=False, residual=True), dict(bias=False, residual=False)]
PARTS = [(form, act) for form in FORMS for act in ACTS if act or any(form.values())]


@pytest.mark.parametrize("form,act", PARTS, ids=lambda v: str(v) if not isinstance(v, dict) else "_".join(k for k in v if v[k]) or "bare")
def test_activations_and_parts_few_rows(form, act):
    run(5, 264, 256, cl.f16, act, "skinny", dict(WAVES_N=1, WAVES_K=4), **form)


@pytest.mark.parametrize("form,act", PARTS, ids=lambda v: str(v) if not isinstance(v, dict) else "_".join(k for k in v if v[k]) or "bare")
def test_activations_and_parts_phased(form, act):
    run(300, 520, 192, cl.bf16, act, "gemm_dma", dict(BM=256, BN=256, BK=64, WM=2, WN=4), **form)


TILINGS = [
    ("skinny", dict(WAVES_N=2, WAVES_K=2), dict(M=16, N=1000, K=512)), ("skinny", dict(WAVES_N=1, WAVES_K=1), dict(M=64, N=136, K=64)),
    ("skinny", dict(WAVES_N=4, WAVES_K=2), dict(M=1, N=520, K=128)),
    ("gemm", dict(BM=64, BN=64, BK=64, WM=2, WN=2), dict(M=100, N=200, K=256)),
    ("gemm", dict(BM=16, BN=32, BK=64, WM=1, WN=1, GDEPTH=1), dict(M=37, N=88, K=72)),
    ("gemm_dma", dict(BM=64, BN=64, BK=64, WM=2, WN=2), dict(M=130, N=136, K=128)),
    ("gemm_dma", dict(BM=128, BN=128, BK=64, WM=2, WN=2, STAGES=3), dict(M=257, N=264, K=320)),
    ("gemm_dma", dict(BM=64, BN=128, BK=64, WM=2, WN=2, TAIL=2), dict(M=256, N=384, K=192)),
    ("gemm_dma", dict(BM=192, BN=256, BK=64, WM=2, WN=4), dict(M=389, N=264, K=192)),
    ("gemm_dma", dict(BM=128, BN=256, BK=64, WM=2, WN=4), dict(M=200, N=776, K=256)),
    ("gemm_dma", dict(BM=256, BN=128, BK=64, WM=4, WN=2), dict(M=257, N=136, K=128)),
    ("gemm_dma", dict(BM=32, BN=32, BK=64, WM=1, WN=1, KW=4), dict(M=70, N=72, K=1024)),
    ("gemm_dma", dict(BM=128, BN=256, BK=64, WM=2, WN=4, KS=3), dict(M=140, N=520, K=1536)),
    ("gemm", dict(BM=64, BN=64, BK=64, WM=2, WN=2, DMA=1), dict(M=65, N=72, K=136)),
]


@pytest.mark.parametrize("dtype", [cl.f16, cl.bf16], ids=["f16", "bf16"])
@pytest.mark.parametrize("template,tiling,sizes", TILINGS, ids=lambda v: v if isinstance(v, str) else "_".join(f"{k}{n}" for k, n in v.items()))
def test_tilings(template, tiling, sizes, dtype):
    run(*sizes.values(), dtype, "gelu_tanh", template, tiling, residual=True, seed=sizes["M"])


@pytest.mark.parametrize("template,tiling,split,sizes", [
    ("skinny", dict(WAVES_N=1, WAVES_K=2), 4, (16, 520, 512)), ("skinny", dict(WAVES_N=1, WAVES_K=1), 2, (1, 136, 128)),
    ("gemm_dma", dict(BM=64, BN=64, BK=64, WM=2, WN=2), 4, (100, 200, 512)), ("gemm", dict(BM=32, BN=32, BK=64, WM=1, WN=1), 2, (33, 40, 256))])
@pytest.mark.parametrize("act,residual", [("gelu", True), ("silu", False), (None, True)])
def test_split_k(template, tiling, split, sizes, act, residual):
    run(*sizes, cl.f16, act, template, tiling, split, residual=residual)


@pytest.mark.parametrize("N", [1, 2, 6, 129, 250])
@pytest.mark.parametrize("M", [1, 70])
def test_weight_given_nk_and_odd_widths(M, N):
    """Rows of C that are no whole pieces: the last columns of bias and residual are read one by one, and nothing is read past them."""
    run(M, N, 192, cl.f16, "silu", "gemm_dma", dict(BM=64, BN=64, BK=64, WM=2, WN=2), residual=True, transposed=True)
    run(M, N, 256, cl.bf16, "relu", "gemm", dict(BM=64, BN=64, BK=64, WM=2, WN=2), 2, residual=True, transposed=True)


def test_the_input_as_its_own_residual():
    @cleave_amd.jit
    def block(x: cl.Tensor["M", "K"], w: cl.Tensor["K", "K"], b: cl.Tensor[1, "K"]):
        return cl.silu(x @ w + b) + x

    for M, template, tiling in ((9, "skinny", dict(WAVES_N=1, WAVES_K=2)), (300, "gemm_dma", dict(BM=256, BN=256, BK=64, WM=2, WN=4))):
        prog = block.trace(cl.f16, M=M, K=256)
        x, w, b = inputs(M, 256, 256, torch.float16)
        out = kernel_for(prog, template=template, tiling=tiling)(x, w, b)
        check(out, [x, w, b, x], "silu", residual=True)
    split = kernel_for(block.trace(cl.f16, M=9, K=256), template="skinny", tiling=dict(WAVES_N=1, WAVES_K=2), split=2)(*inputs(9, 256, 256, torch.float16))
    x, w, b = inputs(9, 256, 256, torch.float16)
    check(split, [x, w, b, x], "silu", residual=True)


@pytest.mark.parametrize("act", ACTS[1:])
def test_far_arguments(act):
    """Pre-activations of up to +-6e4: the activations' exponentials overflow and underflow there, their limits do not; and small ones,
    where a tail of gelu is all there is."""
    K = 64
    x = torch.zeros(8, K, device="cuda", dtype=torch.float16)
    w = torch.zeros(K, 512, device="cuda", dtype=torch.float16)
    points = torch.cat([torch.linspace(-9, 9, 384), torch.tensor([-6e4, -300.0, -88.0, -40.0, 40.0, 88.0, 300.0, 6e4]), torch.linspace(-1e-3, 1e-3, 120)])
    bias = points.half().cuda().reshape(1, -1)
    prog = C.linear_op(act).trace(cl.f16, M=8, N=512, K=K)
    out = kernel_for(prog, template="skinny", tiling=dict(WAVES_N=1, WAVES_K=1))(x, w, bias)
    check(out, [x, w, bias], act)


@pytest.mark.parametrize("act", ACTS, ids=str)
def test_infinite_and_undefined_values(act):
    """A residual's or bias' infinity or NaN stays in its own element (or column)."""
    M, N, K = 20, 64, 64
    args = inputs(M, N, K, torch.float16, residual=True)
    args[3][3, 5], args[3][4, 6], args[2][0, 9], args[2][0, 33] = float("inf"), float("nan"), float("inf"), float("nan")
    prog = C.linear_op(act, residual=True).trace(cl.f16, M=M, N=N, K=K)
    out = kernel_for(prog, template="gemm_dma", tiling=dict(BM=64, BN=64, BK=64, WM=2, WN=2))(*args)
    assert out[3, 5] == float("inf") and out[4, 6].isnan() and bool((out[:, 9] == float("inf")).all()) and bool(out[:, 33].isnan().all())
    rest = torch.ones(M, N, dtype=torch.bool, device="cuda")
    rest[3, 5] = rest[4, 6] = False
    rest[:, 9] = rest[:, 33] = False
    assert bool(out[rest].isfinite().all())


def test_operands_that_start_anywhere():
    """Bias and residual from any element on (x and w are copied where they have to be)."""
    M, N, K = 70, 264, 192
    args = inputs(M, N, K, torch.float16, residual=True)
    moved = []
    for t in args:
        room = torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")
        at = room[3:3 + t.numel()].view(t.shape)
        at.copy_(t)
        moved.append(at)
    for template, tiling in (("gemm_dma", dict(BM=256, BN=256, BK=64, WM=2, WN=4)), ("gemm", dict(BM=64, BN=64, BK=64, WM=2, WN=2))):
        kernel = kernel_for(C.linear_op("gelu", residual=True).trace(cl.f16, M=M, N=N, K=K), template=template, tiling=tiling)
        assert torch.equal(kernel(*moved), kernel(*args))


def test_nothing_is_written_past_the_result():
    """Odd extents into a tensor inside a larger one: the neighbours stay."""
    M, N, K = 67, 130, 128
    args = inputs(M, N, K, torch.float16, residual=True, transposed=True)
    from cleave_amd.pipeline.direct import source_for
    from cleave_amd.runtime.compile import _compile, _load_main_kernel_from_code

    source = source_for(C.linear_op("relu", residual=True, transposed=True).trace(cl.f16, M=M, N=N, K=K), template="gemm_dma",
                        tiling=dict(BM=64, BN=64, BK=64, WM=2, WN=2))
    room = torch.full((M * N + 64,), 7.0, dtype=torch.float16, device="cuda")
    _compile(_load_main_kernel_from_code(source), None)(*args, room[32:32 + M * N].view(M, N))
    check(room[32:32 + M * N].view(M, N), args, "relu", residual=True, transposed=True)
    assert bool((room[:32] == 7).all()) and bool((room[32 + M * N:] == 7).all())


@pytest.mark.parametrize("sizes,split,act", [((16, 1032, 512), cl.Split("K", (2, 4)), "gelu_tanh"), ((333, 520, 384), False, "silu")])
def test_compiled_end_to_end(cache_root, sizes, split, act):
    M, N, K = sizes
    kernel = P.compile(C.linear_op(act, residual=True), shapes=dict(M=M, N=N, K=K), dtype=cl.f16, split=split,
                       schedule=P.ScheduleConfig(topk=4, split_k=getattr(split, "factors", ())),
                       eval=P.EvalConfig(warmup=2, iters=10, max_parallel=2))
    assert len(kernel.report.correct) == len(kernel.report) >= 1
    args = inputs(M, N, K, torch.float16, residual=True, seed=4)
    check(kernel(*args), args, act, residual=True)
    folder = kernel.save(cache_root / "kernel")
    assert torch.equal(cleave_amd.load(folder)(*args), kernel(*args))


def test_captured_and_replayed():
    M, N, K = 16, 520, 512
    kernel = kernel_for(C.linear_op("gelu", residual=True).trace(cl.f16, M=M, N=N, K=K), template="skinny", tiling=dict(WAVES_N=1, WAVES_K=2), split=4)
    args = inputs(M, N, K, torch.float16, residual=True)
    kernel(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernel(*args)
    for seed in (1, 2, 3):
        for t, fresh in zip(args, inputs(M, N, K, torch.float16, residual=True, seed=seed)):
            t.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kernel(*args))
        check(out, args, "gelu", residual=True)
