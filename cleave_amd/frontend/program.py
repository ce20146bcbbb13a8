"""``Program``: a dense tensor program, recorded op by op, that a kernel is compiled from.

Same builder surface as ``python/cleave/frontend/program.py:48-363`` (``dim`` / ``dims`` / ``input`` /
``output``, ``ops``, ``fingerprint()``, ``can_split()``, ``to_graph_structure()`` in the
superoptimizer's op-dict schema, ``random_inputs()``, ``reference()``).  Built differently: the op
vocabulary is one table (``VOCABULARY``) whose rows say, per kind, how result shapes follow from
operand shapes, how torch evaluates it, and what it adds to its op dict; ``apply``,
``reference`` and ``to_graph_structure`` are loops over that table.

``reference`` is the user-facing eager evaluator (fp32 throughout, outputs cast at the end);
compiled kernels never route through it.
"""

from __future__ import annotations

import hashlib
import json
from typing import Callable, NamedTuple, Optional

from ..core.errors import SpecError, SuperoptError
from .recorder import Op, Recorder, dim_to_doc  # noqa: F401  (Op is part of the public surface)
from .tensor import Dim, DType, Tensor, as_dtype, extent, f16, is_number, split_names


class InputSpec(NamedTuple):
    name: str
    dims: tuple
    dtype: DType

    @property
    def shape(self) -> tuple:
        return tuple(extent(d) for d in self.dims)


class OutputSpec(NamedTuple):
    name: str
    tensor: Tensor

    @property
    def shape(self) -> tuple:
        return self.tensor.shape


# ================================================================================ shape rules
def _same_shape(operands, attrs):
    return operands[0].dims


def _broadcast(operands, attrs):
    """Equal ranks; per axis equal extents, or one of them 1 (the other's axis is kept)."""
    tensors = [x for x in operands if isinstance(x, Tensor)]
    if len(tensors) == 1:
        return tensors[0].dims
    a, b = tensors
    if a.ndim != b.ndim:
        raise SpecError(f"rank mismatch {a.shape} vs {b.shape}")
    merged = []
    for da, db in zip(a.dims, b.dims):
        ea, eb = extent(da), extent(db)
        if ea != eb and ea != 1 and eb != 1:
            raise SpecError(f"shapes not broadcastable {a.shape} vs {b.shape}")
        merged.append(db if ea == 1 and eb != 1 else da)
    return tuple(merged)


def _reduced(operands, attrs):
    (a,), axis = operands, attrs["dim"]
    return a.dims[:axis] + (1,) + a.dims[axis + 1:]


def _product(operands, attrs):
    """(..., m, k) @ (..., k, n); a leading extent may be a whole multiple of the other's (heads
    sharing kv heads), and the larger one is the result's."""
    a, b = operands
    if a.ndim != b.ndim or a.ndim < 2:
        raise SpecError(f"matmul rank mismatch: {a.shape} @ {b.shape}")
    if extent(a.dims[-1]) != extent(b.dims[-2]):
        raise SpecError(f"matmul inner dims differ: {a.shape} @ {b.shape}")
    lead = []
    for da, db in zip(a.dims[:-2], b.dims[:-2]):
        big, small = sorted((extent(da), extent(db)), reverse=True)
        if big % small:
            raise SpecError(f"matmul batch dims not grouped-broadcastable: {a.shape} @ {b.shape}")
        lead.append(da if extent(da) >= extent(db) else db)
    return (*lead, a.dims[-2], b.dims[-1])


# ================================================================================ the vocabulary
class OpRule(NamedTuple):
    arity: int
    shape: Callable                       # (operand handles / floats, attrs) -> result dims
    torch: Callable                       # (torch module, evaluated operands, attrs) -> tensor
    scalars: str = "none"                 # a literal operand: none | commutes (goes second) | keeps (its place)
    label: Optional[Callable] = None      # attrs -> the <kind> in "kn_<kind>_op" (default: the kind)
    extras: Optional[Callable] = None     # Op -> more keys of its op dict


def _scalar_keys(op):
    literal = op.scalar_args()
    return {"scalar": float(literal[0]), "scalar_on_left": not isinstance(op.args[0], int)} if literal else {}


def _elementwise(fn, scalars):
    keys = _scalar_keys if scalars != "none" else None
    return OpRule(2, _broadcast, lambda torch, xs, attrs: fn(*xs), scalars, extras=keys)


def _unary(name):
    return OpRule(1, _same_shape, lambda torch, xs, attrs: name(torch)(xs[0]))


def _reduction(method):
    return OpRule(1, _reduced, lambda torch, xs, attrs: getattr(xs[0], method)(attrs["dim"], keepdim=True),
                  label=lambda attrs, kind: f"{kind}_{attrs['dim']}")


VOCABULARY = {
    "add": _elementwise(lambda x, y: x + y, "commutes"),
    "mul": _elementwise(lambda x, y: x * y, "commutes"),
    "div": _elementwise(lambda x, y: x / y, "keeps"),
    "sub": _elementwise(lambda x, y: x - y, "none"),
    "exp": _unary(lambda torch: torch.exp),
    "sqrt": _unary(lambda torch: torch.sqrt),
    "silu": _unary(lambda torch: torch.nn.functional.silu),
    "relu": _unary(lambda torch: torch.relu),
    "gelu": _unary(lambda torch: torch.nn.functional.gelu),
    "gelu_tanh": _unary(lambda torch: lambda x: torch.nn.functional.gelu(x, approximate="tanh")),
    "reduce_sum": _reduction("sum"),
    "reduce_max": _reduction("amax"),
    "matmul": OpRule(2, _product,
                     lambda torch, xs, attrs: grouped_matmul(xs[0], xs[1], attrs["trans_A"], attrs["trans_B"]),
                     extras=lambda op: {"trans_A": bool(op.attr("trans_A")), "trans_B": bool(op.attr("trans_B"))}),
}
UNARY_KINDS = ("exp", "sqrt", "silu", "relu", "gelu", "gelu_tanh")
BINARY_KINDS = ("add", "sub", "mul", "div")
REDUCE_KINDS = ("reduce_sum", "reduce_max")


class Program(Recorder):
    def __init__(self, name: str = "program", dtype=f16):
        super().__init__(name, dtype)
        self.split = ()
        self.inputs: list = []
        self.outputs: list = []
        self._known_dims: dict = {}

    # ---------------------------------------------------------------- dimensions and arguments
    def dim(self, name: str, size=None, dynamic: bool = False, hint=None) -> Dim:
        return self._admit(Dim(name, size, dynamic, hint))

    def dims(self, **sizes) -> tuple:
        return tuple(self.dim(name, size) for name, size in sizes.items())

    def _admit(self, d: Dim) -> Dim:
        """Register a dimension under its name.  Mentioning a known name bare (no size, no hint,
        not dynamic) means the known one; any other disagreement is an error."""
        known = self._known_dims.get(d.name)
        if known is not None and known != d:
            if d.sized or d.dynamic:
                raise SpecError(f"dim {d.name!r} redeclared: {known} vs {d}")
            return known
        d.extent                       # an unsized dimension is refused here
        self._known_dims[d.name] = d
        return d

    def _resolve_axis(self, owner: str, d):
        if isinstance(d, Dim):
            return self._admit(d)
        if isinstance(d, str):
            if d not in self._known_dims:
                raise SpecError(f"input {owner!r}: unknown dim {d!r}; declare it with .dim()/.dims()")
            return self._known_dims[d]
        if isinstance(d, int) and not isinstance(d, bool) and d > 0:
            return d
        raise SpecError(f"input {owner!r}: bad dim {d!r}")

    def input(self, name: str, dims, dtype=None) -> Tensor:
        if name in (spec.name for spec in self.inputs):
            raise SpecError(f"duplicate input name {name!r}")
        spec = InputSpec(name, tuple(self._resolve_axis(name, d) for d in dims), as_dtype(dtype) or self.dtype)
        self.inputs.append(spec)
        return self.emit("input", (), [(spec.dims, spec.dtype)], name=name)

    def output(self, t: Tensor, name: Optional[str] = None) -> None:
        self.need(t, "output")
        name = name or f"out{len(self.outputs)}"
        if name in (spec.name for spec in self.outputs):
            raise SpecError(f"duplicate output name {name!r}")
        self.outputs.append(OutputSpec(name, t))
        self.emit("output", (t.id,), (), name=name)

    # ---------------------------------------------------------------- recording
    def apply(self, kind: str, operands, **attrs) -> Tensor:
        """What every ``Tensor`` operator calls."""
        rule = VOCABULARY.get(kind)
        if rule is None:
            raise SpecError(f".{kind} is only lowerable inside a paged (dynamic) program")
        operands = list(operands)
        if kind == "matmul":
            for x in operands:
                if not self.owns(x):
                    raise SpecError("matmul operands must be cl.Tensors of the same Program")
            attrs = {"trans_A": operands[0]._trans, "trans_B": operands[1]._trans}
        else:
            literal = [i for i, x in enumerate(operands) if not isinstance(x, Tensor)]
            for i in literal:
                if not is_number(operands[i]):
                    raise SpecError(f"{kind}: unsupported operand {type(operands[i]).__name__}")
                operands[i] = float(operands[i])
            if literal == [0] and rule.scalars == "commutes":
                operands.reverse()
            elif literal and (rule.scalars == "none" or len(literal) > 1):
                raise SpecError(f"{kind}: unsupported operand {type(operands[literal[0]]).__name__}")
            for x in operands:
                if isinstance(x, Tensor):
                    self.need(x, kind[len("reduce_"):] if kind in REDUCE_KINDS else kind)
        if "dim" in attrs:
            rank, axis = operands[0].ndim, attrs["dim"]
            if not -rank <= axis < rank:
                raise SpecError(f"{kind[len('reduce_'):]}: dim {axis} out of range for rank {rank}")
            attrs["dim"] = axis % rank
        try:
            shape = rule.shape(operands, attrs)
        except SpecError as e:
            raise SpecError(f"{kind}: {e}") if not str(e).startswith("matmul") else e
        first = next(x for x in operands if isinstance(x, Tensor))
        return self.emit(kind, [x.id if isinstance(x, Tensor) else x for x in operands], [(shape, first.dtype)], **attrs)

    # ---------------------------------------------------------------- reading
    @property
    def ops(self) -> list:
        """Argument and compute records in call order (outputs are in ``.outputs``)."""
        return [op for op in self.oplist if op.kind != "output"]

    @property
    def op_count(self) -> int:
        return len(self.ops)

    @property
    def sizes(self) -> dict:
        return {name: d.extent for name, d in self._known_dims.items()}

    @property
    def dynamic_dims(self) -> tuple:
        return tuple(d for d in self._known_dims.values() if d.dynamic)

    def __repr__(self):
        return self.listing(f"cleave.Program {self.name!r} dtype={self.dtype.name} dims={self.sizes} "
                            f"fingerprint={self.fingerprint()[:12]}")

    def fingerprint(self) -> str:
        """A sha256 over what the program computes: element types, argument shapes (dimension
        names, extents, dynamic flags), and the ops with operands, literals and attributes.
        Argument and output names, and the program's own name, do not enter."""
        canon = [self.dtype.name]
        canon += [[spec.dtype.name, [dim_to_doc(d) if not isinstance(d, Dim) else [d.name, d.extent, d.dynamic]
                                     for d in spec.dims]] for spec in self.inputs]
        for op in self.oplist:
            operands = [a if isinstance(a, int) else float(a).hex() for a in op.args]
            canon.append([op.kind, operands, [[k, v] for k, v in op.attrs if k != "name"]])
        return hashlib.sha256(json.dumps(canon, separators=(",", ":")).encode()).hexdigest()

    def can_split(self, split=()) -> list:
        """For each argument, one flag per axis: is that axis a dimension named in ``split``?"""
        wanted = split_names(split)
        present = {d.name for spec in self.inputs for d in spec.dims if isinstance(d, Dim)}
        absent = [name for name in wanted if name not in present]
        if absent:
            raise SpecError(f"split dims {absent} are not dims of any input (have {sorted(present)})")
        return [tuple(isinstance(d, Dim) and d.name in wanted for d in spec.dims) for spec in self.inputs]

    # ---------------------------------------------------------------- hand-over to the lowering
    def to_graph_structure(self) -> list:
        """The program as op dicts in the superoptimizer's ``get_graph_structure()`` schema
        (``python/cleave/core/schema.py``): ``op_type`` ``kn_<kind>_op``; ``input_tensors`` /
        ``output_tensors`` entries with ``num_dims``, ``dim`` and a ``guid`` (value number + 1;
        argument tensors also carry ``dtype``); matmuls add ``trans_A`` / ``trans_B``; binaries
        with a literal add ``scalar`` / ``scalar_on_left``."""
        arguments = {op.out for op in self.oplist if op.kind == "input"}

        def describe(number):
            handle = self.values[number]
            entry = {"num_dims": handle.ndim, "dim": list(handle.shape), "guid": number + 1}
            if number in arguments:
                entry["dtype"] = handle.dtype.name
            return entry

        structure = []
        for op in self.oplist:
            rule = VOCABULARY.get(op.kind)
            label = rule.label(dict(op.attrs), op.kind) if rule and rule.label else op.kind
            entry = {"op_type": f"kn_{label}_op",
                     "input_tensors": [describe(a) for a in op.value_args()],
                     "output_tensors": [describe(o) for o in op.outs]}
            if rule and rule.extras:
                entry.update(rule.extras(op))
            structure.append(entry)
        return structure

    def to_tile_graph(self, split=()):
        """In Cleave this replays the program onto the C++ superoptimizer's graph.  That engine is
        not part of this back end; ``cleave_amd.pipeline.superoptimize`` proposes graphs."""
        raise SuperoptError("the C++ superoptimizer is not bundled with this back end; "
                            "use cleave_amd.pipeline.superoptimize(program, config)")

    # ---------------------------------------------------------------- eager evaluation
    def _arguments(self, positional, named) -> list:
        if positional and named:
            raise TypeError("pass inputs either positionally or by name, not both")
        order = [spec.name for spec in self.inputs]
        if named:
            missing, extra = [n for n in order if n not in named], sorted(set(named) - set(order))
            if missing or extra:
                raise TypeError(f"inputs: missing {missing}, unexpected {extra}")
            positional = [named[n] for n in order]
        if len(positional) != len(order):
            raise TypeError(f"{self.name}: expected {len(order)} inputs, got {len(positional)}")
        for spec, x in zip(self.inputs, positional):
            if tuple(x.shape) != spec.shape:
                raise SpecError(f"input {spec.name!r}: shape {tuple(x.shape)} != {spec.shape}")
        return list(positional)

    def reference(self, *inputs, **named) -> list:
        """Evaluate with torch, on whatever device the inputs are on: arguments raised to fp32,
        every op in fp32, each output cast to its own element type."""
        import torch

        feed = iter(self._arguments(inputs, named))
        held = {}
        for op in self.ops:
            if op.kind == "input":
                held[op.out] = next(feed).float()
            else:
                operands = [held[a] if isinstance(a, int) else a for a in op.args]
                held[op.out] = VOCABULARY[op.kind].torch(torch, operands, dict(op.attrs))
        return [held[spec.tensor.id].to(spec.tensor.dtype.torch) for spec in self.outputs]

    def random_inputs(self, seed: int = 0, device: str = "cuda") -> list:
        """Seeded arguments drawn on the CPU (so a CPU run and a GPU run see the same bits), then
        moved: standard normal; uniform in [0.5, 1.5) for what feeds a square root or divides;
        integers in [0, 16) for int32 arguments."""
        import torch

        source = torch.Generator(device="cpu").manual_seed(seed)
        keep_positive = self._positive_inputs()
        drawn = []
        for spec in self.inputs:
            if spec.dtype.name == "int32":
                x = torch.randint(0, 16, spec.shape, generator=source, dtype=torch.int32)
            elif spec.name in keep_positive:
                x = torch.rand(spec.shape, generator=source) + 0.5
            else:
                x = torch.randn(spec.shape, generator=source)
            drawn.append(x.to(dtype=spec.dtype.torch, device=device))
        return drawn

    def _positive_inputs(self) -> set:
        """Names of the arguments that are taken the square root of, or divided by, directly."""
        argument_name = {op.out: op.attr("name") for op in self.oplist if op.kind == "input"}
        sensitive = [op.args[0] for op in self.oplist if op.kind == "sqrt"]
        sensitive += [op.args[1] for op in self.oplist if op.kind == "div"]
        return {argument_name[v] for v in sensitive if v in argument_name}


def grouped_matmul(a, b, trans_a=False, trans_b=False):
    """``a @ b`` on torch tensors where, on a leading axis, the shorter operand's entries are
    each used for a run of the longer one's (``repeat_interleave``): 32 query heads over 8 kv
    heads pair head ``h`` with kv head ``h // 4``."""
    a = a.mT if trans_a else a
    b = b.mT if trans_b else b
    for axis, (na, nb) in enumerate(zip(a.shape[:-2], b.shape[:-2])):
        if na < nb:
            a = a.repeat_interleave(nb // na, dim=axis)
        elif nb < na:
            b = b.repeat_interleave(na // nb, dim=axis)
    return a @ b
