"""Pages that a decode's requests share: what is traced, kept and refused, and the launch-time cuts."""

import json

import pytest
import torch

import cleave_amd.lang as cl
from cleave_amd import examples as C
from cleave_amd.codegen import HipCodeGen
from cleave_amd.core.errors import SpecError
from cleave_amd.dynamic import reference
from cleave_amd.dynamic.paging import (PAGED_DECODE, PAGED_DECODE_SLAB, CombineTiling, DenseAttention, PagingSpec, build_split_decode)
from cleave_amd.dynamic.paging.apply import _check_tiling, _shared_plan, shared_ranges
from cleave_amd.dynamic.paging.errors import UnsupportedTiling
from cleave_amd.frontend.paged import PagedProgram, trace_paged
from cleave_amd.runtime import shim
from cleave_amd.runtime.compile import _load_main_kernel_from_code, code_object_stats, eval_extent
from cleave_amd.runtime.dispatch import postfix


def spec_of(page=64, hq=32, hkv=8):
    spec = PagingSpec(hq, hkv, kind=PAGED_DECODE_SLAB if page > 1 else PAGED_DECODE, page_size=page, shared_input="SHARED", shared_dim="n_shared")
    spec.validate()
    return spec


DENSE = DenseAttention(16, 32, 128, 256, "float16", "float16")


@pytest.mark.parametrize("page", [1, 64])
def test_traced_and_kept(page):
    attention = trace_paged(C.shared_prefix_decode_op(page=page)).attention()
    spec = attention.paging_spec()
    assert spec.shared_input == "PREFIX_INDICES" and spec.shared_dim == "n_shared"
    again = PagedProgram.from_doc(json.loads(json.dumps(attention.program.to_doc()))).attention()
    assert again.paging_spec() == spec and [p.name for p in again.inputs] == [p.name for p in attention.inputs]


def _traced(body, **changes):
    notes = dict(C.shared_prefix_decode_op(page=1).fn.__annotations__, **changes)
    body.__annotations__ = notes
    return trace_paged(body, name="op").attention().paging_spec()


def _decode(q, k_cache, v_cache, pages, sm_scale, **limits):
    k, v = cl.paged_gather(k_cache, pages), cl.paged_gather(v_cache, pages)
    return (cl.softmax((q.view(q.dims[0], 8, 4, 128) @ k.mT) * sm_scale, **limits) @ v).view(q.dims[0], 32, 128)


def test_refused_programs():
    def windowed(q, k_cache, v_cache, prefix_indices, kv_indptr, kv_indices, sm_scale):
        return _decode(q, k_cache, v_cache, cl.PageTable(kv_indptr, kv_indices, shared=prefix_indices), sm_scale, window=9)

    with pytest.raises(SpecError, match="without a window"):
        _traced(windowed)

    def matrix(q, k_cache, v_cache, prefix_indices, kv_indptr, kv_indices, sm_scale):
        return _decode(q, k_cache, v_cache, cl.PageTable(kv_indptr, kv_indices, shared=prefix_indices), sm_scale)

    assert _traced(matrix).shared_input == "PREFIX_INDICES"
    with pytest.raises(SpecError, match="vector"):
        _traced(matrix, prefix_indices=cl.Tensor[cl.Dim("a", dynamic=True), cl.Dim("b", dynamic=True), cl.i32])
    with pytest.raises(SpecError, match="named"):
        _traced(matrix, prefix_indices=cl.Tensor[32, cl.i32])
    with pytest.raises(SpecError, match="need indices"):
        cl.PageTable(None, shared=object())

    def other(q, k_cache, v_cache, prefix_indices, kv_indptr, kv_indices, sm_scale):
        return _decode(q, k_cache, v_cache, cl.PageTable(kv_indptr, kv_indices, shared=torch.zeros(3)), sm_scale)

    with pytest.raises(SpecError, match="PageTable"):
        _traced(other)


def test_refused_kernels():
    """The kernels that know nothing of shared pages refuse them, and the one that reads them needs some."""
    with pytest.raises(UnsupportedTiling, match="shared pages"):
        build_split_decode(spec_of(), DENSE, 4, CombineTiling(split=4))
    with pytest.raises(UnsupportedTiling, match="shared pages"):
        _check_tiling(PagingSpec(32, 8), DENSE, shared=True)
    with pytest.raises(UnsupportedTiling, match="256"):
        _check_tiling(spec_of(), DenseAttention(16, 32, 384, 256, "float16", "float16"), shared=True)


@pytest.mark.parametrize("page", [1, 16, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_kernels_compile_without_spills(page, d):
    for dtype in ("float16", "bfloat16"):
        source = HipCodeGen().gen(_shared_plan(spec_of(page), DenseAttention(16, 32, d, 256, dtype, dtype)))
        stats = code_object_stats(shim.compile_source(source)[0])
        assert len(stats) == 2 and all(k["spilled_vgprs"] == 0 and k["scratch_bytes"] == 0 for k in stats)


@pytest.mark.parametrize("hq,hkv", [(32, 8), (10, 2), (40, 2), (6, 3)])
@pytest.mark.parametrize("page", [1, 64])
def test_launch_time_cuts(hq, hkv, page):
    """For any batch: one range of either kind at least, every workgroup that the kernel counts on is launched, and the native
    plan's arithmetic is the manifest's."""
    spec = spec_of(page, hq, hkv)
    manifest = _load_main_kernel_from_code(HipCodeGen().gen(_shared_plan(spec, DenseAttention(-(-hq // hkv // 16) * 16, 32, 128, 256, "float16", "float16")))).manifest
    assert [list(r) for r in shared_ranges(spec, 128)] == manifest["derived_dims"]
    for batch in (1, 2, 7, 64, 300, 5000):
        for shared in (0, 1, 100, 40000):
            for own in (0, 1, 777, 300000):
                dims = {"batch": batch, "n_shared": shared, "n_idx": own, "num_pages": 10}
                for name, expr in manifest["derived_dims"]:
                    dims[name] = eval_extent(expr, dims)
                    postfix(expr, {n: i for i, n in enumerate(dims)})
                assert dims["prefix_ranges"] >= 1 and 1 <= dims["own_chunk"] * page <= 2048
                tiles, group = -(-batch * (hq // hkv) // 128), hq // hkv
                items = -(-own // dims["own_chunk"]) + batch
                blocks = -(-hkv * dims["prefix_ranges"] // 8) * 8 * tiles + items * -(-hkv // 4) * -(-group // 16)
                assert eval_extent(manifest["launches"][0]["grid"][0], dims) == blocks
                rows = next(p for p in manifest["params"] if p["name"] == "Partial_PM_split")["shape"][0]
                assert eval_extent(rows, dims) == batch * dims["prefix_ranges"] + items


def test_reference_of_shared_pages():
    """The shared tokens, then the request's own, as one list of keys."""
    lens, page, shared = [3, 0, 20], 4, 2
    dims = (3, 4, 2, 64, 20, 7)
    args = reference.gqa_paged_decode_inputs(dims, lens, page_size=page, dtype=torch.float32, device="cpu", shared=shared)
    assert args[3].numel() == 2 and len(args) == 8
    out, lse = reference.gqa_paged_decode_reference(dims, lens, page_size=page, dtype=torch.float32, shared=shared)(*args)
    start = args[4].tolist()
    for b, n in enumerate(lens):
        own = args[5][start[b]:start[b] + -(-n // page)].long()
        k, v = (torch.cat([c[args[3].long()].reshape(-1, 2, 64), c[own].reshape(-1, 2, 64)[:n]]) for c in args[1:3])
        for h in range(4):
            logits = k[:, h // 2].double() @ args[0][b, h].double() * args[-1]
            torch.testing.assert_close(out[b, h].double(), torch.softmax(logits, 0) @ v[:, h // 2].double(), rtol=1e-5, atol=1e-5)
