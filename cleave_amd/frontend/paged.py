"""Paged attention operators, written with ``cl.PageTable`` / ``cl.paged_gather`` / ``cl.Scalar`` /
``cl.softmax(return_lse=, causal=)``.

Tracing such a function gives a ``PagedProgram``; ``PagedProgram.attention()`` reads the operator
back off it: GQA or MLA, decode or causal prefill.  The public surface (class and property
names, what is refused) is that of ``python/cleave/frontend/paged.py``, so Cleave's dynamic demos
trace as they are.  Recognition works on an expression tree: the recorded ops are folded into
nested ``_Term`` nodes with the views taken out, and the operator is matched on that tree from
the output down.  A ``PagedProgram`` also has a plain-data form (``to_doc`` / ``from_doc``) so
that a compiled operator can be saved without pickling code.
"""

from __future__ import annotations

import inspect
import math
import random
import zlib
from typing import NamedTuple, Optional

from ..core.errors import SpecError
from . import composites
from .program import Program
from .recorder import Op, Recorder, dim_from_doc, dim_to_doc
from .tensor import (Dim, ScalarSpec, Split, Tensor, TensorSpec, as_dtype, as_splits, bf16, dim_name, f32,
                     is_number)

DEFAULT_KV_HINT = 4096   # kv length a dynamic kv dimension is planned at when it brings no hint
MIN_QUERY_ROWS = 16      # rows of one matrix-core tile
PREFILL_QUERY_ROWS = 64  # (token, head slot) rows of one GQA prefill block


# ================================================================================ declarations
class ScheduleHints:
    """Settings of a paged kernel that steer its schedule and leave its result alone."""

    KNOBS = ("grid_order", "rasterization", "warp_policy", "pass_configs", "index_window_tiles", "prefetch")

    def __init__(self, **knobs):
        unknown = sorted(k for k in knobs if k not in self.KNOBS)
        if unknown:
            raise SpecError(f"unknown schedule hints {unknown}; expected some of {self.KNOBS}")
        self.knobs = {k: tuple(v) if k == "grid_order" else v for k, v in knobs.items()}

    def __eq__(self, other):
        return isinstance(other, ScheduleHints) and self.knobs == other.knobs

    def __repr__(self):
        return "cl.ScheduleHints(" + ", ".join(f"{k}={v!r}" for k, v in self.knobs.items()) + ")"


class PageTable:
    """A CSR table over requests.  With ``indices``: request ``r`` owns the pages
    ``indices[indptr[r]:indptr[r+1]]`` (and ``last_page_len[r]`` tokens of the last one; needed
    exactly when pages hold more than one token).  Without: the table is *ragged*, request ``r``
    owns rows ``indptr[r]:indptr[r+1]`` of a packed tensor.

    ``shared``: pages that every request begins with, all of them full; a request's tokens are theirs, then those of its own
    pages (which may be none)."""

    def __init__(self, indptr, indices=None, last_page_len=None, length: Optional[Dim] = None, shared=None):
        if not (length is None or isinstance(length, Dim)):
            raise SpecError(f"PageTable(length=...) must be a cl.Dim, got {length!r}")
        if indices is None and last_page_len is not None:
            raise SpecError("PageTable: last_page_len needs indices (ragged rows have no pages)")
        if indices is None and shared is not None:
            raise SpecError("PageTable: shared pages need indices (ragged rows have no pages)")
        self.indptr, self.indices, self.last_page_len, self.shared = indptr, indices, last_page_len, shared
        self.length = length if length is not None else Dim("kv_len", dynamic=True, hint=DEFAULT_KV_HINT)

    ragged = property(lambda self: self.indices is None)

    @property
    def requests(self) -> Dim:
        """The request-count dimension: an ``indptr`` of length ``batch + 1`` names it ``batch``."""
        first = self.indptr.dims[0] if isinstance(self.indptr, Tensor) and self.indptr.dims else None
        name = dim_name(first) or ""
        return Dim(name[:-2] if name.endswith("+1") else "batch", dynamic=True)

    def columns(self):
        return (self.indptr, self.indices, self.last_page_len)


def paged_gather(cache, pages: PageTable):
    """``cache`` of shape (pages, page size[, heads], d) -- ragged: (rows[, heads], d) -- read
    per request through ``pages``: logically (requests[, heads], length, d)."""
    if not isinstance(pages, PageTable):
        raise SpecError(f"paged_gather(cache, pages): pages must be a cl.PageTable, got {pages!r}")
    if not isinstance(cache, Tensor):
        raise NotImplementedError("eager paged_gather: validate a paged operator over workloads")
    if not isinstance(cache.program, PagedProgram):
        raise SpecError("paged_gather needs a paged program (annotate the runtime scale as cl.Scalar)")
    return cache.program.apply("paged_gather", (cache,), pages=pages)


def _window_of(window, sinks):
    """``(window, sinks)`` as whole numbers, or a ``SpecError``."""
    for name, value, least in (("window", window, 1), ("sinks", sinks, 0)):
        if value is not None and (isinstance(value, bool) or not isinstance(value, int) or value < least):
            raise SpecError(f"softmax({name}=...) must be a whole number of at least {least}, got {value!r}")
    if window is None and sinks:
        raise SpecError("softmax(sinks=...) needs a window: without one every key before the query is visible")
    return window, int(sinks or 0)


def softmax(x, dim: int = -1, shift: Optional[float] = None, return_lse: bool = False, causal: bool = False,
            window: Optional[int] = None, sinks: int = 0):
    """Softmax over ``dim``.  ``return_lse``: also the base-2 log of the sum of exponentials.
    ``causal``: scores are masked bottom-right aligned (query ``i`` sees keys ``j <= i + kv_len -
    q_len``).  ``window``: a query sees the last ``window`` keys up to its own position only, and the first ``sinks`` keys of its
    request (the one query of a decode program stands at the request's last key).  All exist only in paged programs (and
    ``return_lse`` on torch tensors)."""
    traced = isinstance(x, Tensor)
    window, sinks = _window_of(window, sinks)
    if traced and isinstance(x.program, PagedProgram):
        return x.program.apply("softmax", (x,), dim=dim, return_lse=return_lse, causal=causal,
                               **({"window": window, "sinks": sinks} if window is not None else {}))
    if causal or window is not None or (traced and return_lse):
        which = "causal=True" if causal else "window=..." if window is not None else "return_lse=True"
        raise SpecError(f"softmax({which}) is only lowerable inside a paged program")
    if not return_lse:
        return composites.softmax(x, dim, shift)
    wide = x.float()
    return wide.softmax(dim).to(x.dtype), wide.logsumexp(dim) / math.log(2.0)


# ================================================================================ the program
class Param(NamedTuple):
    """One argument of the traced signature: its name, annotation, and value number."""

    name: str
    spec: object
    value: int

    @property
    def is_scalar(self) -> bool:
        return isinstance(self.spec, ScalarSpec)

    @property
    def kernel_name(self) -> str:
        """Its name in the kernel's signature: tensors in upper case (they become
        ``PlaceHolder_<NAME>``), scalars as written."""
        return self.name if self.is_scalar else self.name.upper()


class PagedProgram(Recorder):
    def __init__(self, name: str = "paged", dtype=bf16):
        super().__init__(name, dtype)
        self.params: list = []
        self.outputs: list = []      # (name, value number)
        self.tables: list = []
        self.hints = ScheduleHints()
        self.split = ()

    records = property(lambda self: self.oplist)

    def __repr__(self):
        text = self.listing(f"cleave.PagedProgram {self.name!r} dtype={self.dtype.name}")
        return "\n".join([text] + [f"  output {name} = %{number}" for name, number in self.outputs])

    def param(self, number: int) -> Optional[Param]:
        return next((p for p in self.params if p.value == number), None)

    def producer(self, number: int) -> Optional[Op]:
        return self._maker.get(number)

    def _mine(self, x, what: str) -> Tensor:
        if not self.owns(x):
            raise SpecError(f"{what}: expected a cl.Tensor of this program, got {x!r}")
        return x

    # ---------------------------------------------------------------- arguments and results
    def input(self, name: str, spec) -> Tensor:
        if isinstance(spec, ScalarSpec):
            handle = self.emit("scalar", (), [((), spec.dtype or f32)], name=name)
        else:
            handle = self.emit("input", (), [(spec.dims, spec.dtype)], name=name)
        self.params.append(Param(name, spec, handle.id))
        return handle

    def output(self, t: Tensor, name: Optional[str] = None) -> None:
        self._mine(t, "output")
        self.outputs.append((name or f"out{len(self.outputs)}", t.id))

    # ---------------------------------------------------------------- ops
    def apply(self, kind: str, operands, **attrs):
        handler = getattr(self, "_op_" + kind, None)
        if handler is not None:
            return handler(*operands, **attrs)
        if kind in ("add", "mul", "div"):
            return self._pointwise(kind, operands)
        if kind in ("exp", "sqrt", "silu"):
            (a,) = operands
            return self.emit(kind, [self._mine(a, kind).id], [(a.dims, a.dtype)])
        if kind == "sub":
            raise SpecError("tensor - tensor is only lowerable in a dense program")
        raise SpecError(f".{kind.replace('reduce_', '')} is only lowerable in a dense program")

    def _pointwise(self, kind, operands):
        """Shapes are not checked against each other: the widest operand gives the result's."""
        handles = [self._mine(x, kind) for x in operands if isinstance(x, Tensor)]
        for x in operands:
            if not isinstance(x, Tensor) and not is_number(x):
                raise SpecError(f"{kind}: unsupported operand {type(x).__name__}")
        lead = max(handles, key=lambda t: t.ndim)
        return self.emit(kind, [x.id if isinstance(x, Tensor) else float(x) for x in operands], [(lead.dims, lead.dtype)])

    def _op_paged_gather(self, cache, pages: PageTable):
        self._mine(cache, "paged_gather")
        for column in pages.columns():
            if column is not None:
                self._mine(column, "PageTable")
        if pages.shared is not None:
            self._mine(pages.shared, "PageTable")
        ranks = (2, 3) if pages.ragged else (3, 4)
        if cache.ndim not in ranks:
            layout = "(total[, heads], d)" if pages.ragged else "(num_pages, page_size[, heads], d)"
            raise SpecError(f"paged_gather: {'ragged rows' if pages.ragged else 'cache'} must be {layout}, got {cache!r}")
        if not any(known is pages for known in self.tables):
            self.tables.append(pages)
        number = [known is pages for known in self.tables].index(True)
        heads = cache.dims[(1 if pages.ragged else 2):-1]        # none for a headless (latent) cache
        return self.emit("paged_gather", [cache.id], [((pages.requests, *heads, pages.length, cache.dims[-1]), cache.dtype)],
                         pages=number)

    def _op_view(self, a, shape):
        self._mine(a, "view")
        return self.emit("view", [a.id], [(tuple(shape), a.dtype)], trans=a._trans)

    def _op_matmul(self, a, b):
        self._mine(a, "matmul"), self._mine(b, "matmul")
        if a.ndim != b.ndim or a.ndim < 2:
            raise SpecError(f"matmul rank mismatch: {a!r} @ {b!r}")
        return self.emit("matmul", [a.id, b.id], [((*a.dims[:-1], b.dims[-1]), a.dtype)],
                         trans_A=a._trans, trans_B=b._trans)

    def _op_reduce_sum(self, a, dim):
        self._mine(a, "sum")
        axis = dim % a.ndim
        return self.emit("reduce_sum", [a.id], [(a.dims[:axis] + (1,) + a.dims[axis + 1:], a.dtype)], dim=axis)

    def _op_softmax(self, x, dim, return_lse, causal, **limits):
        self._mine(x, "softmax")
        axis = dim % x.ndim
        results = [(x.dims, x.dtype)]
        if return_lse:
            results.append((x.dims[:axis] + x.dims[axis + 1:], f32))
        return self.emit("softmax", [x.id], results, dim=axis, causal=bool(causal), **limits)

    def attention(self) -> "PagedAttention":
        return PagedAttention.recognize(self)

    # ---------------------------------------------------------------- plain-data form
    def to_doc(self) -> dict:
        """Everything needed to rebuild the program, as JSON-safe data."""
        def spec_doc(spec):
            if isinstance(spec, ScalarSpec):
                return {"scalar": spec.dtype.name}
            return {"dims": [dim_to_doc(d) for d in spec.dims], "dtype": spec.dtype and spec.dtype.name,
                    "optional": spec.optional}

        def column(t):
            return None if t is None else t.id

        return {
            "format": 1, "name": self.name, "dtype": self.dtype.name,
            "split": [[s.dim, list(s.factors)] for s in self.split],
            "hints": {k: list(v) if isinstance(v, tuple) else v for k, v in self.hints.knobs.items()},
            "values": [{"dims": [dim_to_doc(d) for d in t.dims], "dtype": t.dtype.name} for t in self.values],
            "ops": [{"kind": op.kind, "args": list(op.args), "outs": list(op.outs), "attrs": dict(op.attrs)}
                    for op in self.oplist],
            "params": [{"name": p.name, "spec": spec_doc(p.spec), "value": p.value} for p in self.params],
            "tables": [{"indptr": column(t.indptr), "indices": column(t.indices),
                        "last_page_len": column(t.last_page_len), "length": dim_to_doc(t.length),
                        **({"shared": column(t.shared)} if t.shared is not None else {})} for t in self.tables],
            "outputs": [[name, number] for name, number in self.outputs],
        }

    @classmethod
    def from_doc(cls, doc: dict) -> "PagedProgram":
        if doc.get("format") != 1:
            raise SpecError(f"unknown paged-program format {doc.get('format')!r}")
        program = cls(doc["name"], doc["dtype"])
        program.split = tuple(Split(dim, factors) for dim, factors in doc["split"])
        program.hints = ScheduleHints(**doc["hints"])
        for number, value in enumerate(doc["values"]):
            program.values.append(Tensor(program, number, [dim_from_doc(d) for d in value["dims"]], as_dtype(value["dtype"])))
        for entry in doc["ops"]:
            op = Op(entry["kind"], entry["args"], entry["outs"], entry["attrs"])
            program.oplist.append(op)
            program._maker.update({number: op for number in op.outs})

        def spec_from(entry):
            if "scalar" in entry:
                return ScalarSpec(as_dtype(entry["scalar"]))
            return TensorSpec([dim_from_doc(d) for d in entry["dims"]], as_dtype(entry["dtype"]), entry["optional"])

        def column(number):
            return None if number is None else program.values[number]

        program.params = [Param(p["name"], spec_from(p["spec"]), p["value"]) for p in doc["params"]]
        program.tables = [PageTable(column(t["indptr"]), column(t["indices"]), column(t["last_page_len"]),
                                    dim_from_doc(t["length"]), column(t.get("shared"))) for t in doc["tables"]]
        program.outputs = [(name, number) for name, number in doc["outputs"]]
        return program


# ================================================================================ tracing
def _plain(fn):
    from .jit import JitFunction

    return fn.fn if isinstance(fn, JitFunction) else fn


def is_paged(obj) -> bool:
    """True for a ``PagedProgram`` and for a function one of whose parameters is annotated
    ``cl.Scalar[...]`` or ``cl.Tensor[...] | None``."""
    if isinstance(obj, (PagedProgram, Program)) or not callable(obj):
        return isinstance(obj, PagedProgram)
    try:
        parameters = inspect.signature(_plain(obj), eval_str=True).parameters.values()
    except (TypeError, ValueError, NameError):
        return False
    return any(isinstance(p.annotation, ScalarSpec) or getattr(p.annotation, "optional", False) is True
               for p in parameters)


def trace_paged(fn, dtype=None, *, name=None, hints: Optional[ScheduleHints] = None, split=None) -> PagedProgram:
    from .trace import annotated_parameters, named_results, unwrap

    if isinstance(fn, PagedProgram):
        fn.hints = fn.hints if hints is None else hints
        return fn
    hints = hints or getattr(fn, "options", {}).get("hints")
    body, dtype, split, name = unwrap(fn, dtype, split, name)
    program = PagedProgram(name, as_dtype(dtype) or bf16)
    program.split = as_splits(split)
    if hints is not None:
        program.hints = hints
    handles = []
    for parameter in annotated_parameters(body):
        if isinstance(parameter.annotation, (TensorSpec, ScalarSpec)):
            handles.append(program.input(parameter.name, parameter.annotation))
        elif parameter.default is not inspect.Parameter.empty:
            handles.append(parameter.default)
        else:
            raise SpecError(f"{body.__name__}: annotate {parameter.name!r} with cl.Tensor[...] / cl.Scalar[...]")
    for out_name, handle in named_results(body(*handles), body.__name__):
        program.output(handle, out_name)
    return program


# ================================================================================ recognition
class _Term:
    """A value as an expression: ``kind`` (an op kind, or ``argument`` / ``scalar argument`` /
    ``number``), the op or ``Param`` or literal behind it, and its operand terms.  Views are
    transparent: a view's term is its operand's."""

    __slots__ = ("kind", "what", "kids", "number")

    def __init__(self, kind, what, kids=(), number=None):
        self.kind, self.what, self.kids, self.number = kind, what, tuple(kids), number


def _term_of(program: PagedProgram, x) -> _Term:
    if not isinstance(x, int):
        return _Term("number", float(x))
    op = program.producer(x)
    if op.kind == "view":
        return _term_of(program, op.args[0])
    if op.kind in ("input", "scalar"):
        return _Term("scalar argument" if op.kind == "scalar" else "argument", program.param(x), number=x)
    return _Term(op.kind, op, [_term_of(program, a) for a in op.args], number=x)


class _Refusing:
    def __init__(self, program):
        self.program = program

    def __call__(self, why):
        raise SpecError(f"{self.program.name}: not a paged attention program: {why}")

    def expect(self, term: _Term, kind: str, what: str) -> _Term:
        if term.kind != kind:
            got = {"argument": "an input", "scalar argument": "a cl.Scalar", "number": "a constant"}.get(term.kind, term.kind)
            self(f"{what} should be a {kind}, got {got}")
        return term


class PagedAttention:
    """What a paged program computes, when it is one of
    GQA ``softmax((q @ gather(K).mT) * scale) @ gather(V)`` and
    MLA ``softmax((qn @ gather(CKV).mT + qp @ gather(KPE).mT) * scale) @ gather(CKV)``,
    each optionally with the lse as a second output.  A prefill gathers its queries through
    ragged rows and masks causally.  A softmax may carry a ``window`` (and ``sinks``); a decode's page table may have pages that
    all requests share."""

    def __init__(self, program, queries, caches, pages, scale, out, lse=None, rows=None, causal=False, window=None, sinks=0):
        self.program, self.queries, self.caches = program, tuple(queries), tuple(caches)
        self.pages, self.scale, self.out, self.lse, self.rows, self.causal = pages, scale, out, lse, rows, bool(causal)
        self.window, self.sinks = window, int(sinks or 0)

    @classmethod
    def recognize(cls, program: PagedProgram) -> "PagedAttention":
        refuse = _Refusing(program)
        if not 1 <= len(program.outputs) <= 2:
            refuse(f"expected (out[, lse]) outputs, got {len(program.outputs)}")
        out_number = program.outputs[0][1]

        # out = weights @ gather(V)
        product = refuse.expect(_term_of(program, out_number), "matmul", "the output")
        if product.what.attr("trans_A") or product.what.attr("trans_B"):
            refuse("the value matmul is transposed")
        weights = refuse.expect(product.kids[0], "softmax", "the value matmul's lhs")
        values = refuse.expect(product.kids[1], "paged_gather", "the value matmul's rhs")
        if weights.what.attr("dim") != program.value(weights.what.args[0]).ndim - 1:
            refuse("softmax must reduce the last (KV) axis")

        # weights = softmax(scores * scale)
        scaled = refuse.expect(weights.kids[0], "mul", "the softmax input (scores * cl.Scalar)")
        factors = [k for k in scaled.kids if k.kind == "scalar argument"]
        others = [k for k in scaled.kids if k.kind != "scalar argument"]
        if len(factors) != 1 or len(others) != 1 or others[0].kind == "number":
            refuse("the scores must be scaled by a cl.Scalar argument")

        # scores = q @ gather(K).mT  [+ q' @ gather(K').mT]
        def score(term):
            term = refuse.expect(term, "matmul", "a score")
            if term.what.attr("trans_A") or not term.what.attr("trans_B"):
                refuse("a score matmul must be q @ k.mT")
            query, keys = term.kids[0], refuse.expect(term.kids[1], "paged_gather", "a key")
            rows = None
            if query.kind == "paged_gather":                   # a prefill's queries
                rows = query.what.attr("pages")
                if not program.tables[rows].ragged:
                    refuse("queries are gathered through ragged rows (a cl.PageTable without indices)")
                query = query.kids[0]
            if query.kind != "argument":
                refuse("the query should be a cl.Tensor argument")
            return query.what, rows, keys

        parts = [score(k) for k in others[0].kids] if others[0].kind == "add" else [score(others[0])]
        gathers = [keys for _, _, keys in parts] + [values]
        tables = {g.what.attr("pages") for g in gathers}
        if len(tables) != 1:
            refuse("every cache must be gathered through the same cl.PageTable")
        row_tables = {rows for _, rows, _ in parts}
        if len(row_tables) != 1:
            refuse("every query must be gathered through the same ragged rows")
        (table,), (rows,) = tables, row_tables
        if rows == table:
            refuse("the queries and the caches need their own tables")
        for g in gathers:
            if g.kids[0].kind != "argument":
                refuse("a cache should be a cl.Tensor argument")
        caches = [g.kids[0].what for g in gathers]
        if len(parts) == 2 and caches[2] != caches[0]:
            refuse("the latent (MLA) form reads the compressed cache as its values")

        lse_number = None
        if len(program.outputs) == 2:
            lse_number = program.outputs[1][1]
            through = lse_number
            while program.producer(through).kind == "view":
                through = program.producer(through).args[0]
            if len(weights.what.outs) != 2 or through != weights.what.outs[1]:
                refuse("the second output must be the softmax's lse")
        return cls(program, [q for q, _, _ in parts], caches[:2], program.tables[table], factors[0].what, out_number,
                   lse_number, None if rows is None else program.tables[rows], weights.what.attr("causal"),
                   weights.what.attr("window"), weights.what.attr("sinks", 0))

    # ---------------------------------------------------------------- facts about the operator
    is_mla = property(lambda self: len(self.queries) == 2)
    is_prefill = property(lambda self: self.rows is not None)
    query = property(lambda self: self.queries[0])
    kv_len = property(lambda self: self.pages.length)
    num_qo_heads = property(lambda self: int(self.query.spec.dims[1]))
    head_dim = property(lambda self: int(self.query.spec.dims[-1]))
    pe_dim = property(lambda self: int(self.queries[1].spec.dims[-1]) if self.is_mla else None)
    page_size = property(lambda self: 1 if self.pages.ragged else int(self.caches[0].spec.dims[1]))

    @property
    def num_kv_heads(self) -> int:
        return 1 if self.is_mla else int(self.caches[0].spec.dims[1 if self.pages.ragged else 2])

    @property
    def kind(self) -> str:
        """The access layer (``cleave_amd.dynamic.paging.kinds``) this operator needs."""
        from ..dynamic.paging import kinds

        name = self.program.name
        if self.is_prefill != self.causal:
            raise SpecError(f"{name}: only causal prefill is built: ragged query rows go with cl.softmax(..., causal=True)")
        if self.pages.ragged and not self.is_prefill:
            raise SpecError(f"{name}: ragged (unpaged) KV is only built for prefill")
        if self.is_mla and self.pages.ragged:
            raise SpecError(f"{name}: MLA reads a paged cache; ragged MLA is not built")
        if self.is_mla and (self.window is not None or self.pages.shared is not None):
            raise SpecError(f"{name}: a window and shared pages are built for GQA, not for MLA")
        if self.pages.shared is not None and (self.is_prefill or self.window is not None):
            raise SpecError(f"{name}: shared pages are built for decode, without a window")
        layer = {
            (True, True): kinds.MLA_PAGED_PREFILL_CAUSAL, (True, False): kinds.MLA_PAGED_DECODE,
            (False, True): kinds.RAGGED_PREFILL_CAUSAL if self.pages.ragged else kinds.PAGED_PREFILL_CAUSAL,
            (False, False): kinds.PAGED_DECODE_SLAB if self.page_size > 1 else kinds.PAGED_DECODE,
        }
        return layer[self.is_mla, self.is_prefill]

    def _param_of(self, column) -> Optional[Param]:
        return None if column is None else self.program.param(column.id)

    @property
    def inputs(self) -> list:
        """The kernel's arguments in the traced signature's order.  A ``last_page_len`` that an
        operator with one token per page never reads is left out."""
        last = self._param_of(self.pages.last_page_len)
        skip = last if self.page_size == 1 else None
        return [p for p in self.program.params if skip is None or p is not skip]

    @property
    def query_rows(self) -> int:
        """Rows of the dense body one block computes: a head group rounded up to whole
        matrix-core tiles; a GQA prefill block has at least 64 (token, head slot) rows."""
        group = self.num_qo_heads // self.num_kv_heads
        rows = max(1, math.ceil(group / MIN_QUERY_ROWS)) * MIN_QUERY_ROWS
        return max(rows, PREFILL_QUERY_ROWS) if self.is_prefill and not self.is_mla else rows

    def output_dims(self) -> list:
        return [self.program.value(number).dims for number in (self.out, self.lse) if number is not None]

    def output_dtypes(self) -> list:
        return [self.program.dtype, f32][: len(self.output_dims())]

    # ---------------------------------------------------------------- hand-over to the back end
    def paging_spec(self, hints: Optional[ScheduleHints] = None):
        """The ``PagingSpec`` / ``MLASpec`` of this operator: every tensor and dimension named as
        the traced signature names it."""
        from ..dynamic.paging import PAGED_KINDS, MLASpec, PagingSpec

        kind, name = self.kind, self.program.name
        hints = hints or self.program.hints
        indptr, indices, last = (self._param_of(c) for c in self.pages.columns())
        caches, query = self.caches, self.query
        if not self.is_mla and caches[0].spec.dims != caches[1].spec.dims:
            raise SpecError(f"K and V caches differ: {caches[0].spec.dims} vs {caches[1].spec.dims}")
        for q, c in zip(self.queries, caches):
            if q.spec.dims[-1] != c.spec.dims[-1]:
                raise SpecError(f"{q.name} width {q.spec.dims[-1]} != {c.name} width {c.spec.dims[-1]}")

        def axis(param, i=0):
            return dim_name(param.spec.dims[i])

        said = {"kind": kind, "num_qo_heads": self.num_qo_heads, "page_size": self.page_size,
                "emit_lse": self.lse is not None, "scale_input": self.scale.kernel_name,
                "indptr_input": indptr.kernel_name, "cache_inputs": tuple(c.kernel_name for c in caches),
                ("tokens_dim" if self.is_prefill else "batch_dim"): axis(query)}
        if self.is_mla:
            said["query_inputs"] = tuple(q.kernel_name for q in self.queries)
        else:
            said.update(num_kv_heads=self.num_kv_heads, query_input=query.kernel_name)
        if self.is_mla or kind in PAGED_KINDS:
            said.update(index_input=indices.kernel_name, index_dim=axis(indices), pages_dim=axis(caches[0]))
        else:
            said["kv_tokens_dim"] = axis(caches[0])
        if self.is_prefill:
            row_ptr = self._param_of(self.rows.indptr)
            if axis(row_ptr) != axis(indptr):
                raise SpecError(f"{row_ptr.name} and {indptr.name} must share one length")
            said.update(query_indptr_input=row_ptr.kernel_name, causal=True)
        if (axis(indptr) or "").isidentifier():
            said["indptr_dim"] = axis(indptr)
        if self.page_size > 1 and not self.is_mla:
            if last is None:
                raise SpecError(f"page_size={self.page_size}: the PageTable needs last_page_len")
            said["last_page_len_input"] = last.kernel_name
        elif last is not None and (self.is_mla or not last.spec.optional):
            raise SpecError(f"{name} reads no last_page_len; drop it or make it optional")
        if self.window is not None:
            said.update(window=self.window, sinks=self.sinks)
        if self.pages.shared is not None:
            shared = self._param_of(self.pages.shared)
            if shared is None or len(shared.spec.dims) != 1:
                raise SpecError(f"{name}: the shared pages are a vector argument of page numbers")
            said.update(shared_input=shared.kernel_name, shared_dim=axis(shared))
        nameless = [field for field, value in said.items() if value is None]
        if nameless:
            raise SpecError(f"{name}: {nameless} must be named cl.Dims")
        spec_type = MLASpec if self.is_mla else PagingSpec
        try:
            spec = spec_type(**said, **hints.knobs)
        except TypeError as e:
            raise SpecError(f"{spec_type.__name__} has no such schedule knob: {e}") from None
        spec.validate()
        return spec

    def dense_body(self) -> "DenseBody":
        """The dense attention one block computes, as an ordinary program: ``query_rows`` rows
        against a kv axis planned at its hint, the scale written as ``1 / sqrt(head_dim)``."""
        rows, d = self.query_rows, self.head_dim
        kv = Dim(self.kv_len.name, self.kv_len.hint or DEFAULT_KV_HINT, dynamic=True)
        body = DenseBody(f"{self.program.name}.dense", self.program.dtype)
        if self.is_mla:
            shapes = {"QN": (rows, d), "CKV": (kv, d), "QP": (rows, self.pe_dim), "KPE": (kv, self.pe_dim)}
            qn, ckv, qp, kpe = (body.input(name, shape) for name, shape in shapes.items())
            scores, values = (qn @ ckv.mT) + (qp @ kpe.mT), ckv
        else:
            q, k, values = (body.input(name, shape) for name, shape in (("Q", (rows, d)), ("K", (kv, d)), ("V", (kv, d))))
            scores = q @ k.mT
        weights = (scores / math.sqrt(d)).exp()
        body.output((weights / weights.sum(-1, keepdim=True)) @ values)
        return body


class DenseBody(Program):
    """The per-block dense attention of a paged operator."""


# ================================================================================ workloads
class PagedDecodeWorkloads:
    """Synthetic decode workloads: every ``batch`` size times ``samples`` kv lengths spread
    geometrically over ``kv_len``.  In a workload the first request has the full length and the
    others are uniform in [length / 2, length], drawn from a generator seeded by the CRC-32 of
    ``repr((seed, batch, length))`` (``python/cleave/frontend/paged.py:575-618``).  ``prefix``: tokens
    of the pages that the requests of an operator with shared pages begin with (rounded up to whole pages; other
    operators have none); ``kv_len`` counts the tokens behind them."""

    def __init__(self, batch=(1, 7, 64), kv_len=(1, 8192), samples: int = 3, seed: int = 0, prefix: int = 2048):
        self.batch, self.kv_len, self.samples, self.seed = tuple(batch), tuple(kv_len), int(samples), int(seed)
        self.prefix = int(prefix)

    def __repr__(self):
        return f"cl.workloads.paged_decode(batch={self.batch}, kv_len={self.kv_len}, samples={self.samples}, seed={self.seed})"

    def axes(self) -> list:
        shortest, longest = self.kv_len
        steps = max(1, self.samples)
        ratio = longest / shortest
        lengths = sorted({round(shortest * ratio ** (i / max(1, steps - 1))) for i in range(steps)})
        return [(int(b), int(n)) for b in self.batch for n in lengths]

    def lengths(self, batch: int, kv_len: int) -> list:
        draw = random.Random(zlib.crc32(repr((self.seed, batch, kv_len)).encode()))
        floor = max(self.kv_len[0], kv_len // 2)
        return [kv_len] + [draw.randint(floor, kv_len) for _ in range(batch - 1)]

    def factory(self, attention: PagedAttention, keep: int = 0):
        """A generator function of ``(key, inputs, expected outputs)`` over ``keep`` of the axes
        (all of them for 0)."""
        from ..dynamic import reference
        from ..runtime.autotune import sampled, workload_key

        page, dtype = attention.page_size, attention.program.dtype.torch
        heads = (attention.num_qo_heads, attention.num_kv_heads, attention.head_dim)
        axes = sampled(self.axes(), keep)
        shared = math.ceil(self.prefix / page) if attention.pages.shared is not None else 0
        limits = {"window": attention.window, "sinks": attention.sinks, "shared": shared}

        def generate():
            for batch, length in axes:
                lens = self.lengths(batch, length)
                pages = sum(math.ceil(n / page) for n in lens)
                dims = (batch, *heads, pages + shared, pages)
                inputs = reference.gqa_paged_decode_inputs(dims, lens, page_size=page, dtype=dtype, shared=shared)
                expected = reference.gqa_paged_decode_reference(dims, lens, page_size=page, dtype=dtype, **limits)(*inputs)
                yield workload_key((batch, length)), inputs, expected

        return generate


class CausalPrefillWorkloads:
    """Synthetic prompts for a GQA causal prefill: every ``batch`` size times ``samples`` numbers of new tokens spread
    geometrically over ``q_len``, the first request with all of them and the others uniform in [length / 2, length]; ``prefix``: the
    range of keys a request already has in its cache, uniform too.  Drawn as ``PagedDecodeWorkloads`` draws."""

    def __init__(self, batch=(1, 8), q_len=(1, 2048), prefix=(0, 1024), samples: int = 3, seed: int = 0):
        self.batch, self.q_len, self.prefix = tuple(batch), tuple(q_len), tuple(prefix)
        self.samples, self.seed = int(samples), int(seed)

    def __repr__(self):
        return (f"cl.workloads.causal_prefill(batch={self.batch}, q_len={self.q_len}, prefix={self.prefix}, samples={self.samples}, "
                f"seed={self.seed})")

    def axes(self) -> list:
        return PagedDecodeWorkloads(self.batch, self.q_len, self.samples).axes()

    def lengths(self, batch: int, q_len: int):
        """``(new tokens, keys)`` of every request."""
        draw = random.Random(zlib.crc32(repr((self.seed, batch, q_len)).encode()))
        floor = max(self.q_len[0], q_len // 2)
        new = [q_len] + [draw.randint(floor, q_len) for _ in range(batch - 1)]
        return new, [n + draw.randint(*self.prefix) for n in new]

    def factory(self, attention: PagedAttention, keep: int = 0):
        from ..dynamic import reference
        from ..runtime.autotune import sampled, workload_key

        if attention.is_mla or not attention.is_prefill:
            raise SpecError(f"{attention.program.name}: cl.workloads.causal_prefill makes prompts of a GQA causal prefill")
        dtype = attention.program.dtype.torch
        heads = (attention.num_qo_heads, attention.num_kv_heads, attention.head_dim)
        axes = sampled(self.axes(), keep)
        limits = {"window": attention.window, "sinks": attention.sinks}

        def generate():
            for batch, q_len in axes:
                new, keys = self.lengths(batch, q_len)
                if attention.pages.ragged:
                    dims = (*heads, sum(new), sum(keys))
                    make, refer = reference.gqa_ragged_prefill_inputs, reference.gqa_ragged_prefill_reference
                else:
                    dims = (*heads, sum(keys), sum(keys), sum(new))
                    make, refer = reference.gqa_paged_prefill_inputs, reference.gqa_paged_prefill_reference
                inputs = make(dims, new, keys, dtype=dtype)
                yield workload_key((batch, q_len)), inputs, refer(dims, new, keys, dtype=dtype, **limits)(*inputs)

        return generate


class workloads:  # noqa: N801  (spelled ``cl.workloads.paged_decode(...)``)
    paged_decode = PagedDecodeWorkloads
    causal_prefill = CausalPrefillWorkloads
