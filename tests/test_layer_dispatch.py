# SPDX-License-Identifier: BSD-3-Clause
"""What the layer norm, 8-bit and expert layer entry points refuse, and what they
launch, on the CPU: libxtc_hip.so runs against the stand-in for the HIP runtime."""

from __future__ import annotations

import pytest

from test_dispatch import pytestmark, run  # noqa: F401

CALLS = """
P = ctypes.c_void_p
L.xtc_hip_expert_layer_workspace.restype = ctypes.c_uint64

def call(fn, *args):
    fake.fake_launches()
    rc = getattr(L, fn)(*[ctypes.byref(a) if isinstance(a, ctypes.Structure) else P(a) if type(a) is int else a for a in args])
    got = fake.fake_launches().decode().splitlines()
    assert not (rc and got), got
    rows = [g.replace("void ", "").replace("xtc_hip::", "").replace("(anonymous namespace)::", "").split("|") for g in got]
    return capi.last_error() if rc else [[name.split("(")[0], grid] for name, grid, _ in rows]

def norm(fn="xtc_hip_layer_norm", args=None, **kw):
    n = 4 if fn == "xtc_hip_layer_norm" else 7
    return call(fn, capi.LayerNormDesc(**{**dict(dtype=1, param_dtype=0, rows=4, K=8, eps=1e-5), **kw}), *(args or (256,) * n))

def fp8(fn, args, **kw):
    return call(fn, capi.Fp8Desc(**{**dict(dtype=1, matrices=1, rows=4, K=128, block_rows=1), **kw}), *args)

def product(args=(256,) * 5, **kw):
    return call("xtc_hip_fp8_matmul", capi.Fp8MatmulDesc(**{**dict(out_dtype=0, M=4, N=8, blocks=1, b_block_rows=1), **kw}), *args)

def layer(args=None, room=None, **kw):
    d = capi.ExpertLayerDesc(**{**dict(dtype=1, weights=0, activation=1, T=4, E=8, K=64, H=32, top_k=2, normalize=1), **kw})
    need = L.xtc_hip_expert_layer_workspace(ctypes.byref(d)) if room is None else room
    ops = (256,) * 8 if d.weights else (256, 256, 256, None, 256, None, 256, 256)
    ops = list(args or ops)
    return call("xtc_hip_expert_layer", d, *ops[:7], ctypes.c_uint64(need), ops[7])
"""


def agree(got, want):
    for message, why in zip(got, want, strict=True):
        assert isinstance(message, str) and why in message, (why, message)


def test_layer_norm_refusals(run):  # noqa: F811
    most = 2**31 - 1
    wrong = [("unsupported dtype", dict(dtype=2)), ("unsupported dtype", dict(param_dtype=2)), ("of the parameters", dict(dtype=0, param_dtype=1)),
             ("invalid sizes", dict(rows=-1)), ("invalid sizes", dict(K=0)), ("eps", dict(eps=-1.0)), ("eps", dict(eps=float("inf"))),
             ("eps", dict(eps=float("nan"))), ("row strides", dict(ldx=7)), ("row strides", dict(ldy=7)), ("too many", dict(K=most)),
             ("too many", dict(rows=2**31)), ("too many", dict(rows=2**31 - 1, K=2**30, ldx=most))]
    got = run(CALLS + f"""
inf, nan = float("inf"), float("nan")
for fn in ("xtc_hip_layer_norm", "xtc_hip_layer_norm_grad"):
    for kw in {[kw for _, kw in wrong]!r}:
        out.append(norm(fn, **kw))
    out.append(call(fn, None, *(256,) * (4 if fn == "xtc_hip_layer_norm" else 7)))
out.append(norm(args=(None, 256, 256, 256)))
out.append(norm(args=(256, 256, 256, None)))
G = "xtc_hip_layer_norm_grad"
out.append(norm(G, (256, 256, 256, None, None, None, 256)))
out.append(norm(G, (256, 256, 256, 256, 256, 256, None)))
out.append(norm(G, (None, 256, 256, 256, 256, 256, 256)))
out.append(norm(G, (256, 256, None, 256, 256, 256, 256)))
""")
    each = [w for w, _ in wrong] + ["null descriptor"]
    agree(got, each * 2 + ["null operand"] * 2 + ["no result", "workspace"] + ["null operand"] * 2)


def test_layer_norm_launches(run):  # noqa: F811
    """Threads and runs a row by its length alone; gradients in at most 512 parts."""
    got = run(CALLS + """
G = "xtc_hip_layer_norm_grad"
for K in (1, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385):
    out.append(norm(K=K, rows=100000) + norm(G, K=K, rows=100000))
out.append(norm(rows=0) + norm(G, rows=0))
out.append(norm(args=(256, None, None, 256)))
out.append(norm(G, (256, None, 256, 256, None, None, None)))
out.append(norm(G, (256, 256, 256, None, 256, None, 256)))
for rows in (1, 5):
    out.append(norm(G, rows=rows) + norm(G, rows=rows, K=5000))
""")
    forms = [[g[0].rsplit("_", 0)[0].split("<")[0] + " " + ",".join(g[0].rstrip(">").split(", ")[-2:]) for g in row[:2]] for row in got[:12]]
    want = ["64,1", "64,1", "64,2", "64,2", "256,1", "256,1", "256,2", "256,2", "1024,1", "1024,1", "1024,2", "1024,2"]
    assert [f[0] for f in forms] == ["layer_norm " + w for w in want]
    want[6:8] = ["512,1"] * 2
    assert [f[1] for f in forms] == ["layer_norm_grad " + w for w in want]
    for row in got[:12]:
        assert row[1][1] == "512 1 1" and row[2][0] == "layer_norm_grad_sum" and int(row[0][1].split()[0]) <= 1024
    assert [g[0].split("<")[0] for g in got[12]] == ["layer_norm_long", "layer_norm_long", "layer_norm_grad_columns", "layer_norm_grad_sum"]
    assert [g[0] for g in got[13]] == ["layer_norm_grad_sum"]  # zeros
    assert [len(g) for g in got[14:17]] == [1, 1, 2]
    assert [[g[1] for g in row if "sum" not in g[0]] for row in got[17:]] == [["1 1 1", "1 1 1"], ["2 1 1", "5 1 1"]]


def test_fp8_refusals(run):  # noqa: F811
    most = 2**31 - 1
    fns = [("xtc_hip_fp8_quantize", 4), ("xtc_hip_fp8_quantize_both", 5), ("xtc_hip_fp8_encode", 3), ("xtc_hip_fp8_dequantize", 3)]
    wrong = [("unsupported dtype", dict(dtype=2)), ("invalid sizes", dict(rows=-1)), ("invalid sizes", dict(K=0)),
             ("invalid sizes", dict(matrices=-1)), ("blocks of 2 rows", dict(block_rows=2)), ("row stride", dict(ld=127)),
             ("too many", dict(K=most)), ("too many", dict(matrices=most, rows=2**36, K=2**20))]
    got = run(CALLS + f"""
for fn, n in {fns!r}:
    for kw in {[kw for _, kw in wrong]!r}:
        out.append(fp8(fn, (256,) * n, **kw))
    out.append(fp8(fn, (None,) + (256,) * (n - 1)))
    out.append(call(fn, None, *(256,) * n))
Q = "xtc_hip_fp8_quantize"
out.append(fp8(Q, (256, None, None, None)))
out.append(fp8(Q, (256, 256, 256, 256), transpose=1))
out.append(fp8(Q, (256, 264, 256, 256)))
out.append(fp8(Q, (256, 264, 256, None), transpose=1))
out.append(fp8("xtc_hip_fp8_quantize_both", (256,) * 5, transpose=1))
out.append(fp8("xtc_hip_fp8_quantize_both", (256, 256, 256, 264, 256)))
for i in range(1, 5):
    out.append(fp8("xtc_hip_fp8_quantize_both", [None if i == j else 256 for j in range(5)]))
out.append(fp8("xtc_hip_fp8_encode", (256, 256, 264)))
out.append(fp8("xtc_hip_fp8_dequantize", (256,) * 3, transpose=1))
out.append(fp8("xtc_hip_fp8_dequantize", (264, 256, 256)))
""")
    each = [w for w, _ in wrong] + ["null operand", "null descriptor"]
    agree(got, each * 4 + ["null operand", "dequantize", "16-byte aligned", "16-byte aligned", "transpose must be 0", "16-byte aligned"]
          + ["null operand"] * 4 + ["16-byte aligned", "transpose must be 0", "16-byte aligned"])


def test_fp8_matmul_refusals(run):  # noqa: F811
    most = 2**31 - 1
    wrong = [("unsupported result dtype", dict(out_dtype=2)), ("invalid sizes", dict(M=-1)), ("invalid sizes", dict(N=0)),
             ("invalid sizes", dict(blocks=0)), ("blocks of 2 rows", dict(b_block_rows=2)), ("row stride", dict(ldc=7)),
             ("too many", dict(M=most)), ("too many", dict(N=most)), ("too many", dict(blocks=2**16)),
             ("too many", dict(M=2**31 - 2048, N=2**31 - 2048))]
    got = run(CALLS + f"""
for kw in {[kw for _, kw in wrong]!r}:
    out.append(product(**kw))
for i in range(5):
    out.append(product([None if i == j else 256 for j in range(5)]))
for i in (0, 2):
    out.append(product([264 if i == j else 256 for j in range(5)]))
out.append(call("xtc_hip_fp8_matmul", None, *(256,) * 5))
""")
    agree(got, [w for w, _ in wrong] + ["null operand"] * 5 + ["16-byte aligned"] * 2 + ["null descriptor"])


def test_fp8_launches(run):  # noqa: F811
    """Every kernel is reached, by sizes alone: scales off every boundary change nothing."""
    got = run(CALLS + """
out.append([fp8("xtc_hip_fp8_" + fn, (256,) * n, dtype=dtype, **kw) for dtype in (0, 1) for fn, n, kw in (
    ("quantize", 4, {}), ("quantize", 4, dict(block_rows=128)), ("quantize_both", 5, {}), ("quantize_both", 5, dict(block_rows=128)),
    ("encode", 3, {}), ("encode", 3, dict(transpose=1)), ("encode", 3, dict(block_rows=128)), ("dequantize", 3, {}))])
out.append([fp8("xtc_hip_fp8_quantize", (256, 256, 256, None), transpose=1, block_rows=r) for r in (1, 128)])
out.append([fp8("xtc_hip_fp8_quantize", (256, 256, 256, 256), **{n: 0}) for n in ("rows", "matrices")] + [product(M=0)])
for o in (0, 1):
    out.append([product(out_dtype=o, M=M, N=N, blocks=b) for M, N, b in
                ((1, 1, 1), (16, 8192, 64), (17, 8192, 64), (32, 8192, 64), (64, 4096, 32), (512, 4096, 32), (1024, 1024, 64), (4096, 2048, 32),
                 (2048, 2048, 16), (8192, 8192, 32), (8192, 8192, 64), (100000, 300, 3))])
out.append(product((256, 257, 256, 259, 260), M=4096, N=2048, blocks=32))
""")
    kernels = [[g[0] for g in one] for one in got[0]]
    assert [len(k) for k in kernels] == [1] * 16
    assert {k[0].split("<")[0] for k in kernels} == {"fp8_quantize_rows", "fp8_quantize_tiles", "fp8_dequantize"}
    for dtype in (0, 8):
        assert [k[0].split("<")[0].rsplit("_", 1)[1] for k in kernels[dtype : dtype + 8]] == ["rows", "tiles", "tiles", "tiles", "rows", "tiles", "tiles", "dequantize"]
        assert [k[0].endswith(("true>", "1>")) for k in kernels[dtype : dtype + 7]] == [False] * 4 + [True] * 3
    assert [g[0][0].split("<")[0] for g in got[1]] == ["fp8_quantize_tiles"] * 2
    assert got[2] == [[], [], []]
    tile = {"fp8_rows": "rows", "2, 4, 4, 2": "256", "2, 2, 4, 4": "256", "2, 2, 2, 2": "128", "2, 2, 1, 1": "64"}
    for fast, row in ((False, got[3]), (True, got[4])):
        names = [one[0][0] for one in row]
        kinds = [next(v for k, v in tile.items() if k in n) for n in names]
        # the fastest tile measured; to fp32 the two smaller ones are within 4 % at 2048 x 2048 x 2048
        assert kinds[:5] == ["rows"] * 5 and kinds[5:7] == ["64"] * 2 and kinds[7] == "128" and kinds[9:11] == ["256"] * 2, kinds
        assert kinds[8] == "128" if fast else kinds[8] in ("128", "64"), kinds
        assert all(("<true" in n or "<1" in n) == fast for n in names if "fp8_dma" in n), names
        assert ["1, 2>" in n for n in names[:5]] == [True, True, False, False, False], names
    assert got[5] == got[3][7]


def test_expert_layer_refusals(run):  # noqa: F811
    most = 2**31 - 1
    wrong = [("unsupported dtype", dict(dtype=2)), ("unsupported kind", dict(weights=3)), ("take bf16 rows", dict(dtype=0, weights=1)),
             ("take bf16 rows", dict(dtype=0, weights=2)), ("unsupported activation", dict(activation=2)),
             *[("invalid sizes", {n: -1}) for n in ("T", "E", "K", "H", "top_k")], *[("invalid sizes", {n: 0}) for n in ("E", "K", "H", "top_k")],
             ("too many", dict(T=65)), ("too many", dict(E=257)), ("too many", dict(E=64, top_k=17)), ("too many", dict(top_k=9)),
             ("too many", dict(K=most)), ("too many", dict(H=most)), ("too many", dict(T=64, E=256, K=2**31 - 1024, ldx=2**31 - 1024)),
             ("row strides", dict(ldx=63)), ("row strides", dict(ldy=63))]
    got = run(CALLS + f"""
for kw in {[kw for _, kw in wrong]!r}:
    out.append(layer(room=2**62, **kw))
    out.append(L.xtc_hip_expert_layer_workspace(ctypes.byref(capi.ExpertLayerDesc(**{{**dict(dtype=1, T=4, E=8, K=64, H=32, top_k=2), **kw}}))))
out.append(L.xtc_hip_expert_layer_workspace(None))
dense, packed = (256, 256, 256, None, 256, None, 256, 256), (256,) * 8
for i in (0, 1, 2, 4, 6, 7):
    out.append(layer([None if i == j else v for j, v in enumerate(dense)]))
for i in (3, 5):
    out.append(layer([None if i == j else v for j, v in enumerate(packed)], weights=1))
    out.append(layer([256 if i == j else v for j, v in enumerate(dense)]))
for i in (2, 4):
    out.append(layer([264 if i == j else v for j, v in enumerate(packed)], weights=2))
out.append(layer([264 if j == 6 else v for j, v in enumerate(dense)]))
out.append(layer(room=100))
out.append(call("xtc_hip_expert_layer", None, 256, 256, 256, None, 256, None, 256, ctypes.c_uint64(2**40), 256))
""")
    n = 2 * len(wrong)
    agree(got[:n:2], [w for w, _ in wrong])
    # strides and pieces of work need no workspace of their own
    assert [w for w, (why, _) in zip(got[1:n:2], wrong) if why != "row strides"][:-1] == [0] * (len(wrong) - 3) and got[n] == 0
    agree(got[n + 1:], ["null operand"] * 6 + ["null operand", "that have none"] * 2 + ["16-byte aligned"] * 2
          + ["16-byte aligned", "a workspace of 100 bytes", "null descriptor"])


def test_expert_layer_launches(run):  # noqa: F811
    """Logits by a launch of their own where router and tokens are long; waves that share
    out k by fours, and by twos where there are many rows of packed matrices."""
    got = run(CALLS + """
for kw in (dict(T=0), dict(T=1), dict(T=33), dict(T=32, E=144, top_k=1), dict(T=17, E=33), dict(T=4, E=8, K=8192), dict(T=64, E=256, top_k=16, K=4096, H=2048)):
    out.append(layer(**kw))
for weights in (0, 1, 2):
    for act in (0, 1):
        out.append(layer(weights=weights, activation=act) + layer(weights=weights, activation=act, H=8192))
out.append(layer(dtype=0) + layer(dtype=0, H=8192, activation=0))
""")
    kinds = [[g[0].split("<")[0] for g in one] for one in got]
    two, three = ["layer_up", "layer_down"], ["layer_logits", "layer_up", "layer_down"]
    assert kinds[:7] == [[], two, three, three, three, three, three], kinds[:7]
    assert all(k == two * 2 for k in kinds[7:])
    groups = [int(g[1].split()[0]) for one in got for g in one if "logits" not in g[0]]
    assert max(groups) <= 768 and min(groups) >= 1
    names = {g[0] for one in got[7:] for g in one}
    # pieces of down have 32 rows where there are enough of them for the CUs
    assert got[5][2][0].startswith("layer_down<1, 2, 4") and got[1][1][0].startswith("layer_down<1, 1, 4")
    # up by activation and depth, down by depth; dense ones have one depth
    assert len(names) == 2 * (2 * 2 + 2) + 2 * (2 + 1), sorted(names)


def test_payloads_of_sixteen_arguments(run):  # noqa: F811
    """A norm, a router and matrices with scales are eight operands and a result."""
    got = run("""
seen = []
P = ctypes.CFUNCTYPE(None, *[ctypes.c_void_p] * 16)
fn = P(lambda *a: seen.append(a))
res = (ctypes.c_double * 4)()
for n in (9, 16, 17):
    del seen[:]
    args = (ctypes.c_void_p * 17)(*range(1, 18))
    L.xtc_hip_evaluate_perf(res, 0, None, 1, 1, 0, ctypes.cast(fn, ctypes.c_void_p), args, n)
    out.append([list(a) for a in seen[:1]] + [L.xtc_hip_evaluate_status()])
""")
    assert got[0] == [[*range(1, 10), *[None] * 7], 0] and got[1] == [list(range(1, 17)), 0] and got[2] == [1]
