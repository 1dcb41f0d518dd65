# SPDX-License-Identifier: BSD-3-Clause
"""Graph -> kernel-launch plan of the HIP backend.

Every operator node of an XTC graph becomes one launch of a hand-written
gfx950 kernel, except where the producer/consumer pattern lets a kernel
absorb its neighbour (the MI355X design choice: keep intermediates out of
HBM):
  * pad2d/pad on H and W feeding conv2d input 0 -> folded into the
    implicit-GEMM loader (out-of-window taps read `constant_value`);
  * bias_add on a matmul/conv2d result -> GEMM epilogue;
  * relu on a matmul/conv2d(/bias_add) result -> GEMM epilogue.
Such a fusion happens only when the intermediate is used once and is not a graph
output.  mx4_scales, the mx4_codes of the same tensor for these scales and a
mx4_dequantize of the pair are one launch that writes all of them; codes and scales
made for the rows of one 4-bit product alone go into its call.  The fp8_scales and
fp8_codes of a tensor are one launch too, with the values of the pair or with the scales
and codes of the transposed tensor; the gradients of one layer_norm are one call where x's
comes first, or the sums alone are asked for.  A matmul operand with
layout [1, 0] (stored transposed) becomes the launch's trans_a / trans_b flag, a
grouped_matmul's matrices with [0, 2, 1] its trans_w; other operators require natural
layouts.  reshape is a view; unpad is a crop kernel (16-byte row copies when the innermost dim is kept).  The reference lowers each node to its own
linalg op (src/xtc/backends/mlir/MlirOps.py:166-887) and fuses only through
transform-dialect producer fusion (MlirCompilerPasses.py:378-412).

The plan uses only the graph interfaces (nodes, operation, inputs/outputs,
types), so it accepts any Graph that follows xtc.itf.graph.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from math import prod
from typing import Any

from ...utils.bf16 import is_bf16, itemsize

__all__ = ["Buffer", "Launch", "Plan", "lower_graph", "UnsupportedGraph"]

F32 = "float32"
BF16 = "bfloat16"
F64 = "float64"


class UnsupportedGraph(ValueError):
    """The graph uses an operator or dtype the HIP backend does not run."""


@dataclass
class Buffer:
    """A tensor of the plan: a payload argument or a workspace slice."""

    uid: str
    shape: tuple[int, ...]
    dtype: str
    kind: str  # "input" | "output" | "temp" | "alias"
    arg_index: int = -1  # payload argument position for inputs/outputs
    offset: int = 0  # byte offset in the workspace for temps
    alias_of: str | None = None

    @property
    def nbytes(self) -> int:
        return prod(self.shape) * itemsize(self.dtype)


@dataclass
class Launch:
    """One kernel launch.  `node` is the scheduled node the launch serves
    (the matmul/conv2d for fused GEMMs); `absorbed` lists fused nodes."""

    # "matmul" | "conv2d" | "relu" | "pad" | "unpad" | "copy" | "cast" |
    # "grouped_matmul" | "grouped_matmul_grad_w" |
    # "mx4_quantize" | "mx4_encode" | "mx4_dequantize" | "mx4_matmul" |
    # "mx4_quantize_matmul" (inputs x, the scratch codes and scales, then mx4_matmul's) |
    # "layer_norm" | "layer_norm_grad" | "fp8_quantize" | "fp8_encode" | "fp8_dequantize" |
    # "fp8_matmul" | "expert_layer"
    kind: str
    node: str
    inputs: list[str]
    output: str
    attrs: dict[str, Any] = field(default_factory=dict)
    absorbed: list[str] = field(default_factory=list)


@dataclass
class Plan:
    name: str
    buffers: dict[str, Buffer]
    launches: list[Launch]
    args: list[str]  # payload argument uids: graph inputs then outputs
    workspace_bytes: int
    scheduled: dict[str, Any]  # node name -> graph node, for scheduled launches

    def buffer(self, uid: str) -> Buffer:
        b = self.buffers[uid]
        while b.alias_of is not None:
            b = self.buffers[b.alias_of]
        return b


def _shape(t: Any) -> tuple[int, ...]:
    return tuple(int(d) for d in t.constant_shape) if hasattr(t, "constant_shape") else tuple(int(d) for d in t.shape)


def _dtype(t: Any) -> str:
    return str(t.dtype)


def _pad_hw(node: Any, rank: int) -> tuple[int, int, int, int] | None:
    """(top, bottom, left, right) if the pad only touches axes H, W of NHWC."""
    padding = node.operation.attrs.get("padding")
    if isinstance(padding, dict):
        per = {a % rank: tuple(v) for a, v in padding.items()}
    else:
        per = {a: tuple(padding) for a in range(rank)}
    per = {a: v for a, v in per.items() if tuple(v) != (0, 0)}
    if any(a not in (rank - 3, rank - 2) for a in per):
        return None
    top, bottom = per.get(rank - 3, (0, 0))
    left, right = per.get(rank - 2, (0, 0))
    return int(top), int(bottom), int(left), int(right)


_NORM_GRADS = ("layer_norm_grad_x", "layer_norm_grad_weight", "layer_norm_grad_bias")
NORM_PARTS = 512  # XTC_HIP_LAYER_NORM_PARTS


def fp8_key(op: Any) -> tuple[int, bool]:
    return int(op.attrs.get("rows", 1)), bool(op.attrs.get("transpose", False))


def expert_layer_attrs(op: Any, shapes: list[tuple[int, ...]], dtype: str) -> dict[str, Any]:
    (t, k), e = shapes[0], shapes[1][0]
    dense = len(shapes) == 4
    up = shapes[2][1]
    activation = str(op.attrs.get("activation", "swiglu"))
    weights = "dense" if dense else "mx4" if shapes[2][2] == 16 * shapes[3][2] and shapes[3][1] == up else "fp8"
    return {"dtype": dtype, "weights": weights, "T": t, "E": e, "K": k, "H": up // 2 if activation == "swiglu" else up,
            "top_k": int(op.attrs.get("top_k", 2)), "activation": activation, "normalize": bool(op.attrs.get("normalize", True)),
            "hidden": str(op.attrs.get("hidden_dtype", "float32"))}


def expert_layer_workspace(a: dict[str, Any]) -> int:
    """What xtc_hip_expert_layer asks for, in bytes."""
    slots, hidden = a["T"] * a["top_k"], -(-a["H"] // 32) * 32
    parts = ((4 if a["dtype"] == F32 else 6) * slots * hidden, 4 * slots * a["K"], 32 * a["T"] * a["E"], 4 * slots, 4 * -(-a["K"] // 16))
    return sum(-(-p // 256) * 256 for p in parts)


def lower_graph(graph: Any) -> Plan:
    nodes = graph.nodes  # uid -> node, any itf Graph
    inputs = list(graph.inputs)
    outputs = list(graph.outputs)
    if graph.outputs_types is None:
        raise UnsupportedGraph("graph types are not known: call graph.forward_types() first")

    op_nodes = [n for uid, n in nodes.items() if uid not in inputs]
    users: dict[str, list[Any]] = {}
    for n in op_nodes:
        for u in n.inputs:
            users.setdefault(u, []).append(n)

    def out_type(uid: str) -> Any:
        if uid in inputs:
            return graph.inputs_types[inputs.index(uid)]
        return nodes[uid].outputs_types[0]

    def drop_temp(uid: str) -> None:
        b = buffers.get(uid)
        if b is not None and b.kind == "temp":
            del buffers[uid]

    def single_internal_use(uid: str) -> Any | None:
        us = users.get(uid, [])
        if len(us) == 1 and uid not in outputs:
            return us[0]
        return None

    buffers: dict[str, Buffer] = {}
    for idx, uid in enumerate(inputs):
        t = out_type(uid)
        buffers[uid] = Buffer(uid, _shape(t), _dtype(t), "input", arg_index=idx)
    for idx, uid in enumerate(outputs):
        if uid in buffers:
            raise UnsupportedGraph(f"graph input {uid} is also an output")
        t = out_type(uid)
        buffers[uid] = Buffer(uid, _shape(t), _dtype(t), "output", arg_index=len(inputs) + idx)

    absorbed: set[str] = set()
    launches: list[Launch] = []
    scheduled: dict[str, Any] = {}

    # Nodes in a topological order: graph.nodes may hold them in build order.
    order: list[Any] = []
    seen: set[str] = set(inputs)

    def visit(n: Any) -> None:
        stack = [(n, False)]
        while stack:
            cur, done = stack.pop()
            if done:
                order.append(cur)
                continue
            if cur.uid in seen:
                continue
            seen.add(cur.uid)
            stack.append((cur, True))
            for u in reversed(cur.inputs):
                if u not in seen and u in nodes:
                    stack.append((nodes[u], False))

    for n in op_nodes:
        visit(n)

    # pad producers folded into the conv2d loader, decided before any launch
    pad_fusion: dict[str, tuple[Any, tuple[int, int, int, int]]] = {}
    for n in order:
        if n.operation.name != "conv2d" or n.inputs[0] in inputs:
            continue
        pad_node = nodes[n.inputs[0]]
        if pad_node.operation.name not in ("pad2d", "pad") or single_internal_use(pad_node.uid) is not n:
            continue
        rank = len(_shape(out_type(pad_node.inputs[0])))
        hw = _pad_hw(pad_node, rank) if rank >= 3 else None
        if hw is not None:
            pad_fusion[n.uid] = (pad_node, hw)
            absorbed.add(pad_node.uid)

    def transposed_inputs(n: Any) -> tuple[bool, ...]:
        """Per input: stored transposed (layout [1, 0]).  Only the two 2-D
        operands of a matmul may be (MlirOps.py:171-178); other operators
        need natural layouts, as in the reference (MlirOps.py:45-52)."""
        flags = []
        for idx, u in enumerate(n.inputs):
            t = out_type(u)
            lay = getattr(t, "layout", None)
            shp = _shape(t)
            if lay is None or list(lay) == list(range(len(shp))):
                flags.append(False)
            elif n.operation.name == "matmul" and idx < 2 and len(shp) == 2 and list(lay) == [1, 0]:
                flags.append(True)
            elif n.operation.name == "grouped_matmul" and idx == 1 and list(lay) == [0, 2, 1]:
                flags.append(True)
            else:
                raise UnsupportedGraph(
                    f"{n.operation.name} {n.name}: tensor layout {list(lay)} of input {idx} is not supported "
                    "(only [1, 0] on a 2-D matmul operand and [0, 2, 1] on the matrices of grouped_matmul)"
                )
        return tuple(flags)

    def fp8_attrs(x: str, op: Any) -> dict[str, Any]:
        xs = _shape(out_type(x))
        block_rows, transpose = fp8_key(op)
        return {"dtype": _dtype(out_type(x)), "matrices": prod(xs[:-2]), "rows": xs[-2], "K": xs[-1], "block_rows": block_rows,
                "transpose": transpose, "codes": None, "values": None, "other": None}

    for n in order:
        trans = transposed_inputs(n)  # also checks the nodes a kernel absorbs
        if n.uid in absorbed:
            continue
        op = n.operation
        name = op.name
        t_out = n.outputs_types[0]
        if n.uid not in buffers:
            buffers[n.uid] = Buffer(n.uid, _shape(t_out), _dtype(t_out), "temp")
        if name in ("matmul", "conv2d"):
            in_dt = {_dtype(out_type(u)) for u in n.inputs}
            if len(in_dt) != 1 or not in_dt <= {F32, BF16, F64}:
                raise UnsupportedGraph(
                    f"{name} {n.name}: inputs must both be float32, float64 or bfloat16, got {in_dt}")
            attrs: dict[str, Any] = {"dtype": in_dt.pop(), "relu": False, "threshold": 0.0, "bias": None}
            fused: list[str] = []
            src_inputs = list(n.inputs)
            if name == "matmul":
                i, j, k = (int(op.dims[d]) for d in ("i", "j", "k"))
                attrs.update(M=i, N=j, K=k, trans_a=trans[0], trans_b=trans[1])
            else:
                pads = (0, 0, 0, 0)
                pad_value = 0.0
                if n.uid in pad_fusion:
                    pad_node, pads = pad_fusion[n.uid]
                    pad_value = float(pad_node.operation.attrs.get("constant_value", 0))
                    src_inputs[0] = pad_node.inputs[0]
                    fused.append(pad_node.name)
                ishape = _shape(out_type(src_inputs[0]))
                r, s, c, f = _shape(out_type(n.inputs[1]))
                stride = op.attrs.get("stride", 1)
                sh, sw = (stride, stride) if isinstance(stride, int) else (tuple(stride) * 2)[:2]
                attrs.update(
                    NB=prod(ishape[:-3]),
                    H=ishape[-3],
                    W=ishape[-2],
                    C=c,
                    F=f,
                    R=r,
                    S=s,
                    stride=(int(sh), int(sw)),
                    pads=pads,
                    pad_value=pad_value,
                    M=int(op.dims["b"]) * int(op.dims["h"]) * int(op.dims["w"]),
                    N=f,
                    K=r * s * c,
                )
            # epilogue fusions: bias_add then relu
            out_uid = n.uid
            nxt = single_internal_use(out_uid)
            if nxt is not None and nxt.operation.name == "bias_add" and nxt.inputs[0] == out_uid:
                attrs["bias"] = nxt.inputs[1]
                src_inputs.append(nxt.inputs[1])
                fused.append(nxt.name)
                absorbed.add(nxt.uid)
                drop_temp(out_uid)
                out_uid = nxt.uid
                nxt = single_internal_use(out_uid)
            if nxt is not None and nxt.operation.name == "relu":
                attrs["relu"] = True
                attrs["threshold"] = float(nxt.operation.attrs.get("threshold", 0))
                fused.append(nxt.name)
                absorbed.add(nxt.uid)
                drop_temp(out_uid)
                out_uid = nxt.uid
            out_dt = _dtype(nodes[out_uid].outputs_types[0])
            if out_uid not in buffers:
                buffers[out_uid] = Buffer(out_uid, _shape(nodes[out_uid].outputs_types[0]), out_dt, "temp")
            target = out_uid
            if attrs["dtype"] == F64:
                # fp64 kernels accumulate and store fp64 (the reference's
                # output dtype is the input's, operators.py:176-188)
                if out_dt != F64:
                    raise UnsupportedGraph(f"{name} {n.name}: float64 inputs need a float64 output, not {out_dt}")
            elif is_bf16(out_dt):
                # kernels accumulate and store fp32; a cast kernel narrows it
                target = out_uid + ".f32"
                buffers[target] = Buffer(target, buffers[out_uid].shape, F32, "temp")
            elif out_dt != F32:
                raise UnsupportedGraph(f"{name} {n.name}: output dtype {out_dt} is not supported")
            launches.append(Launch(name, n.name, src_inputs, target, attrs, fused))
            scheduled[n.name] = n
            if target != out_uid:
                launches.append(Launch("cast", n.name, [target], out_uid, {"n": prod(buffers[out_uid].shape)}))
        elif name == "relu":
            dt = _dtype(t_out)
            if dt not in (F32, F64):
                raise UnsupportedGraph(f"relu {n.name}: only float32 and float64 run standalone")
            attrs = {"threshold": float(op.attrs.get("threshold", 0)), "n": prod(_shape(t_out)), "dtype": dt}
            launches.append(Launch("relu", n.name, [n.inputs[0]], n.uid, attrs))
            scheduled[n.name] = n
        elif name in ("pad", "pad2d"):
            dt = _dtype(t_out)
            if dt not in (F32, F64):
                raise UnsupportedGraph(f"{name} {n.name}: only float32 and float64 run standalone")
            ishape = _shape(out_type(n.inputs[0]))
            padding = op.attrs.get("padding")
            rank = len(ishape)
            if isinstance(padding, dict):
                per = [(0, 0)] * rank
                for a, v in padding.items():
                    per[a % rank] = (int(v[0]), int(v[1]))
            else:
                per = [(int(padding[0]), int(padding[1]))] * rank
            attrs = {"shape": ishape, "pads": per, "value": float(op.attrs.get("constant_value", 0)), "dtype": dt}
            launches.append(Launch("pad", n.name, [n.inputs[0]], n.uid, attrs))
            scheduled[n.name] = n
        elif name == "unpad":
            # a crop: out[o] = in[o + before] per dim (operators.py:683-702)
            dt = _dtype(t_out)
            if dt not in (F32, F64, BF16):
                raise UnsupportedGraph(f"unpad {n.name}: dtype {dt} is not supported")
            ishape = _shape(out_type(n.inputs[0]))
            padding = op.attrs.get("padding")
            rank = len(ishape)
            if isinstance(padding, dict):
                per = [(0, 0)] * rank
                for a, v in padding.items():
                    per[a % rank] = (int(v[0]), int(v[1]))
            else:
                per = [(int(padding[0]), int(padding[1]))] * rank
            attrs = {"shape": ishape, "pads": per, "elem": 2 if dt == BF16 else 8 if dt == F64 else 4}
            launches.append(Launch("unpad", n.name, [n.inputs[0]], n.uid, attrs))
            scheduled[n.name] = n
        elif name in ("grouped_matmul", "grouped_matmul_grad_w"):
            xs, ws = _shape(out_type(n.inputs[0])), _shape(out_type(n.inputs[1]))
            attrs = {"dtype": _dtype(out_type(n.inputs[0])), "out": _dtype(t_out), "trans_w": trans[1],
                     "E": _shape(out_type(n.inputs[2]))[0], "T": xs[0], "K": xs[1], "N": ws[-1]}
            launches.append(Launch(name, n.name, list(n.inputs), n.uid, attrs))
            scheduled[n.name] = n
        elif name == "mx4_scales":
            # the codes for these scales and the values of the pair come from the
            # same pass over x
            xs = _shape(out_type(n.inputs[0]))
            attrs = {"dtype": _dtype(out_type(n.inputs[0])), "rows": prod(xs[:-1]), "K": xs[-1], "codes": None,
                     "values": None}
            fused = []
            own = [u for u in users.get(n.uid, [])
                   if u.operation.name == "mx4_codes" and list(u.inputs) == [n.inputs[0], n.uid]]
            if own:
                attrs["codes"] = own[0].uid
                fused.append(own[0])
                pair = [u for u in users.get(own[0].uid, [])
                        if u.operation.name == "mx4_dequantize" and list(u.inputs) == [own[0].uid, n.uid]
                        and _shape(u.outputs_types[0]) == xs and _dtype(u.outputs_types[0]) == attrs["dtype"]]
                if pair:
                    attrs["values"] = pair[0].uid
                    fused.append(pair[0])
            for u in fused:
                transposed_inputs(u)
                absorbed.add(u.uid)
                if u.uid not in buffers:
                    buffers[u.uid] = Buffer(u.uid, _shape(u.outputs_types[0]), _dtype(u.outputs_types[0]), "temp")
            launches.append(Launch("mx4_quantize", n.name, [n.inputs[0]], n.uid, attrs, [u.name for u in fused]))
            scheduled[n.name] = n
        elif name == "mx4_codes":
            xs = _shape(out_type(n.inputs[0]))
            attrs = {"dtype": _dtype(out_type(n.inputs[0])), "rows": prod(xs[:-1]), "K": xs[-1]}
            launches.append(Launch("mx4_encode", n.name, list(n.inputs), n.uid, attrs))
            scheduled[n.name] = n
        elif name == "mx4_dequantize":
            shape = _shape(t_out)
            attrs = {"dtype": _dtype(t_out), "rows": prod(shape[:-1]), "K": shape[-1]}
            launches.append(Launch("mx4_dequantize", n.name, list(n.inputs), n.uid, attrs))
            scheduled[n.name] = n
        elif name in ("mx4_matmul", "grouped_mx4_matmul"):
            bs = _shape(out_type(n.inputs[3]))
            attrs = {"out": _dtype(t_out), "E": bs[0] if name == "grouped_mx4_matmul" else 0,
                     "M": _shape(t_out)[0], "N": bs[-2], "blocks": bs[-1]}
            ln = Launch("mx4_matmul", n.name, list(n.inputs), n.uid, attrs)
            # rows quantised for this product alone
            q = next((q for q in launches if q.kind == "mx4_quantize"
                      and [q.attrs["codes"], q.output] == ln.inputs[:2] and not q.attrs["values"]), None)
            if (q and [u.uid for u in users[q.attrs["codes"]]] == [n.uid]
                    and {u.uid for u in users[q.output]} == {q.attrs["codes"], n.uid}
                    and not {q.attrs["codes"], q.output} & set(outputs)):
                launches.remove(q)
                ln = Launch("mx4_quantize_matmul", n.name, [*q.inputs, *ln.inputs], n.uid, {**attrs, **q.attrs},
                            [q.node, *q.absorbed])
            launches.append(ln)
            scheduled[n.name] = n
        elif name == "layer_norm":
            xs = _shape(t_out)
            attrs = {"dtype": _dtype(t_out), "params": _dtype(out_type(n.inputs[1])), "rows": prod(xs[:-1]), "K": xs[-1],
                     "eps": float(op.attrs.get("eps", 1e-5))}
            launches.append(Launch("layer_norm", n.name, list(n.inputs), n.uid, attrs))
            scheduled[n.name] = n
        elif name in _NORM_GRADS:
            # the gradients that the graph asks for of one norm and dy: one call
            x, dy = n.inputs[0], n.inputs[-1]  # the bias's alone has dy only
            weight = n.inputs[1] if name == "layer_norm_grad_x" else None
            xs = _shape(out_type(x))
            eps = float(op.attrs.get("eps", 1e-5))
            results: dict[str, str | None] = {g: None for g in _NORM_GRADS}
            results[name] = n.uid
            fused = []
            for u in users.get(dy, []):
                kind = u.operation.name
                if u.uid in absorbed or u.name in scheduled or u is n or kind not in _NORM_GRADS[1:] or results[kind]:
                    continue
                if kind == "layer_norm_grad_weight" and (list(u.inputs) != [x, dy] or float(u.operation.attrs.get("eps", 1e-5)) != eps):
                    continue
                if name == "layer_norm_grad_bias":
                    continue
                results[kind] = u.uid
                fused.append(u)
            for u in fused:
                transposed_inputs(u)
                absorbed.add(u.uid)
                if u.uid not in buffers:
                    buffers[u.uid] = Buffer(u.uid, _shape(u.outputs_types[0]), _dtype(u.outputs_types[0]), "temp")
            rows = prod(xs[:-1])
            ws = None
            if results["layer_norm_grad_weight"] or results["layer_norm_grad_bias"]:
                ws = n.uid + ".sums"
                buffers[ws] = Buffer(ws, (2 * min(rows, NORM_PARTS) * xs[-1] + 2 * rows,), F32, "temp")
            attrs = {"dtype": _dtype(out_type(x)), "params": _dtype(out_type(weight)) if weight else F32, "rows": rows, "K": xs[-1],
                     "eps": eps, "weight": weight, "results": list(results.values()), "workspace": ws}
            launches.append(Launch("layer_norm_grad", n.name, [x, dy], n.uid, attrs, [u.name for u in fused]))
            scheduled[n.name] = n
        elif name == "fp8_scales":
            attrs = fp8_attrs(n.inputs[0], op)
            key = (attrs["block_rows"], attrs["transpose"])

            def codes_of(scales: Any, like: tuple[int, bool]) -> Any | None:
                return next((u for u in users.get(scales.uid, []) if u.operation.name == "fp8_codes"
                             and list(u.inputs) == [scales.inputs[0], scales.uid] and fp8_key(u.operation) == like), None)

            fused = []
            codes = codes_of(n, key)
            if codes is not None:
                attrs["codes"] = codes.uid
                fused.append(codes)
                # those of the transposed tensor from the same pass, or the values
                turned = (key[0], not key[1])
                other = next(((u, c) for u in users.get(n.inputs[0], []) if u.operation.name == "fp8_scales" and u.uid not in absorbed
                              and u.name not in scheduled and fp8_key(u.operation) == turned and (c := codes_of(u, turned)) is not None), None)
                if other is not None:
                    attrs["other"] = [u.uid for u in other]
                    fused += other
                elif not key[1]:
                    xs = _shape(out_type(n.inputs[0]))
                    pair = [u for u in users.get(codes.uid, [])
                            if u.operation.name == "fp8_dequantize" and list(u.inputs) == [codes.uid, n.uid]
                            and _shape(u.outputs_types[0]) == xs and _dtype(u.outputs_types[0]) == attrs["dtype"]]
                    if pair:
                        attrs["values"] = pair[0].uid
                        fused.append(pair[0])
            for u in fused:
                transposed_inputs(u)
                absorbed.add(u.uid)
                if u.uid not in buffers:
                    buffers[u.uid] = Buffer(u.uid, _shape(u.outputs_types[0]), _dtype(u.outputs_types[0]), "temp")
            launches.append(Launch("fp8_quantize", n.name, [n.inputs[0]], n.uid, attrs, [u.name for u in fused]))
            scheduled[n.name] = n
        elif name == "fp8_codes":
            launches.append(Launch("fp8_encode", n.name, list(n.inputs), n.uid, fp8_attrs(n.inputs[0], op)))
            scheduled[n.name] = n
        elif name == "fp8_dequantize":
            shape, ss = _shape(t_out), _shape(out_type(n.inputs[1]))
            attrs = {"dtype": _dtype(t_out), "matrices": prod(shape[:-2]), "rows": shape[-2], "K": shape[-1], "transpose": False,
                     "block_rows": 1 if ss[-2] == shape[-2] else 128}
            launches.append(Launch("fp8_dequantize", n.name, list(n.inputs), n.uid, attrs))
            scheduled[n.name] = n
        elif name == "fp8_matmul":
            bs, bss = _shape(out_type(n.inputs[2])), _shape(out_type(n.inputs[3]))
            attrs = {"out": _dtype(t_out), "M": _shape(t_out)[0], "N": bs[0], "blocks": bss[1], "b_block_rows": 1 if bss[0] == bs[0] else 128,
                     "sums": str(op.attrs.get("sums", "fp32"))}
            launches.append(Launch("fp8_matmul", n.name, list(n.inputs), n.uid, attrs))
            scheduled[n.name] = n
        elif name == "expert_layer":
            attrs = expert_layer_attrs(op, [_shape(out_type(u)) for u in n.inputs], _dtype(t_out))
            ws = n.uid + ".layer"
            buffers[ws] = Buffer(ws, (expert_layer_workspace(attrs),), "uint8", "temp")
            attrs["workspace"] = ws
            launches.append(Launch("expert_layer", n.name, list(n.inputs), n.uid, attrs))
            scheduled[n.name] = n
        elif name == "reshape":
            if n.uid in outputs:
                launches.append(Launch("copy", n.name, [n.inputs[0]], n.uid, {}))
            else:
                buffers[n.uid].kind = "alias"
                buffers[n.uid].alias_of = n.inputs[0]
        else:
            raise UnsupportedGraph(
                f"operator {name} ({n.name}) is not supported by the HIP backend "
                "(supported: matmul, conv2d, relu, pad, pad2d, unpad, bias_add after matmul/conv2d, reshape, "
                "grouped_matmul, grouped_matmul_grad_w, mx4_scales, mx4_codes, mx4_dequantize, mx4_matmul, "
                "grouped_mx4_matmul, layer_norm and its gradients, fp8_scales, fp8_codes, fp8_dequantize, fp8_matmul, "
                "expert_layer)"
            )

    # workspace layout: temps packed at 256-byte alignment
    offset = 0
    for b in buffers.values():
        if b.kind == "temp":
            b.offset = offset
            offset += (b.nbytes + 255) // 256 * 256
    return Plan(
        name=graph.name or "payload",
        buffers=buffers,
        launches=launches,
        args=inputs + outputs,
        workspace_bytes=offset,
        scheduled=scheduled,
    )
