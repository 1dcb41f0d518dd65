# SPDX-License-Identifier: BSD-3-Clause
"""What the expert and 4-bit entry points refuse, and what they launch, on the
CPU: libxtc_hip.so runs against the stand-in for the HIP runtime."""

from __future__ import annotations

import pytest

from test_dispatch import pytestmark, run  # noqa: F401

CALLS = """
def call(fn, *args):
    fake.fake_launches()
    rc = getattr(L, fn)(*[ctypes.byref(a) if isinstance(a, ctypes.Structure) else a for a in args])
    got = fake.fake_launches().decode().splitlines()
    assert not (rc and got), got
    return capi.last_error() if rc else [[g.split("|")[0].replace("void ", "").replace("xtc_hip::", "").split("(")[0], g.split("|")[1]] for g in got]

def grouped(fn="xtc_hip_grouped_matmul", args=(256, 256, 256, 256), **kw):
    return call(fn, capi.GroupedMatmulDesc(**{**dict(dtype=1, out_dtype=0, E=2, T=4, N=8, K=8), **kw}), *args)

def mx4(fn, args, **kw):
    return call(fn, capi.Mx4Desc(**{**dict(dtype=0, rows=2, K=32), **kw}), *args)

def mx4_matmul(args=(256, 256, 256, 256, None, 256), **kw):
    return call("xtc_hip_mx4_matmul", capi.Mx4MatmulDesc(**{**dict(out_dtype=0, M=2, N=8, blocks=1), **kw}), *args)
"""


@pytest.mark.parametrize("fn", ["xtc_hip_grouped_matmul", "xtc_hip_grouped_matmul_grad_w"])
def test_grouped_refusals(run, fn):  # noqa: F811
    most = 2**31 - 1
    wrong = [("unsupported dtype", dict(dtype=2)), ("unsupported dtype", dict(dtype=9)),
             ("unsupported result dtype", dict(dtype=0, out_dtype=1)), ("unsupported result dtype", dict(out_dtype=2)),
             *[("invalid sizes", {n: -1}) for n in ("E", "T", "N", "K")], *[("invalid sizes", {n: 0}) for n in ("E", "N", "K")],
             *[("row stride", {n: 7}) for n in ("ldx", "ldw", "ldy")], ("stride", dict(stride_w=-1)),
             ("too many", dict(T=most, N=most, ldy=most)), ("too many", dict(N=most)), ("too many", dict(K=most)),
             ("too many", dict(T=2**31 - 1024, N=2**31 - 1024, K=2**31 - 1024, E=2**31 - 1024))]
    if fn.endswith("grad_w"):
        wrong += [("transposed gradient", dict(trans_w=1)), ("overlap", dict(stride_w=63))]
    got = run(CALLS + f"""
for kw in {[kw for _, kw in wrong]!r}:
    out.append(grouped({fn!r}, **kw))
for i in range(4):
    out.append(grouped({fn!r}, tuple(None if i == j else 256 for j in range(4))))
out.append(call({fn!r}, None, 256, 256, 256, 256))
""")
    for message, (why, kw) in zip(got, wrong):
        assert isinstance(message, str) and why in message, (kw, message)
    assert all("null operand" in m for m in got[len(wrong) : -1]) and "null descriptor" in got[-1]


def test_mx4_refusals(run):  # noqa: F811
    most = 2**31 - 1
    fns = [("xtc_hip_mx4_quantize", 4), ("xtc_hip_mx4_encode", 3), ("xtc_hip_mx4_dequantize", 3)]
    wrong = [("unsupported dtype", dict(dtype=2)), ("invalid sizes", dict(rows=-1)), ("invalid sizes", dict(K=0)),
             ("invalid sizes", dict(K=most)), ("row stride", dict(ld=31))]
    got = run(CALLS + f"""
for fn, n in {fns!r}:
    for kw in {[kw for _, kw in wrong]!r}:
        out.append(mx4(fn, (256,) * n, **kw))
    out.append(mx4(fn, (None,) + (256,) * (n - 1)))
    out.append(call(fn, None, *(256,) * n))
out.append(mx4("xtc_hip_mx4_quantize", (256, None, None, None)))
out.append(mx4("xtc_hip_mx4_quantize", (256, 260, 256, 256)))
out.append(mx4("xtc_hip_mx4_encode", (256, 256, 260)))
out.append(mx4("xtc_hip_mx4_dequantize", (260, 256, 256)))
""")
    want = [w for w, _ in wrong] + ["null operand", "null descriptor"]
    for message, why in zip(got, want * 3 + ["null operand"] + ["16-byte aligned"] * 3, strict=True):
        assert isinstance(message, str) and why in message, (why, message)


def test_mx4_matmul_refusals(run):  # noqa: F811
    most = 2**31 - 1
    wrong = [("unsupported result dtype", dict(out_dtype=2)), *[("invalid sizes", {n: -1}) for n in ("E", "M", "N", "blocks")],
             ("without sizes", dict(E=2)), ("row stride", dict(ldc=7)), ("too many", dict(M=most, N=most, ldc=most)),
             ("too many", dict(blocks=2**27)), ("too many", dict(M=2**31 - 1024, N=2**31 - 1024))]
    got = run(CALLS + f"""
for kw in {[kw for _, kw in wrong]!r}:
    out.append(mx4_matmul(**kw))
out.append(mx4_matmul((256,) * 6))
for i in (0, 2):
    out.append(mx4_matmul([260 if i == j else None if j == 4 else 256 for j in range(6)]))
for i in (0, 1, 2, 3, 5):
    out.append(mx4_matmul([None if j in (i, 4) else 256 for j in range(6)]))
""")
    want = [w for w, _ in wrong] + ["with sizes"] + ["16-byte aligned"] * 2 + ["null operand"] * 5
    for message, why in zip(got, want, strict=True):
        assert isinstance(message, str) and why in message, (why, message)


def test_mx4_quantize_matmul_refusals(run):  # noqa: F811
    wrong = [("unsupported dtype", dict(dtype=2), {}), ("row stride", dict(ld=31), {}), ("invalid sizes", {}, dict(N=0)),
             ("without sizes", {}, dict(E=2)), ("to multiply", dict(rows=3), {}), ("to multiply", dict(K=33), {}),
             ("to multiply", {}, dict(blocks=2)), ("two streams", dict(stream=512), {})]
    got = run(CALLS + f"""
def quantize_matmul(rows, desc, args=(256, 256, 256, 256, 256, None, 256)):
    rows = capi.Mx4Desc(**{{**dict(dtype=1, rows=2, K=32), **rows}})
    desc = capi.Mx4MatmulDesc(**{{**dict(out_dtype=0, M=2, N=8, blocks=1), **desc}})
    return call("xtc_hip_mx4_quantize_matmul", rows, desc, *args)
for rows, desc in {[w[1:] for w in wrong]!r}:
    out.append(quantize_matmul(rows, desc))
for i in (0, 1, 2, 3, 4, 6):
    out.append(quantize_matmul({{}}, {{}}, [None if j in (i, 5) else 256 for j in range(7)]))
for i in (1, 3):
    out.append(quantize_matmul({{}}, {{}}, [260 if i == j else None if j == 5 else 256 for j in range(7)]))
out.append(call("xtc_hip_mx4_quantize_matmul", None, capi.Mx4MatmulDesc(), *(256,) * 7))
out.append(call("xtc_hip_mx4_quantize_matmul", capi.Mx4Desc(dtype=1, rows=2, K=32), *(None,) * 8))
# few rows in one launch, others and fp32 ones in two
out.append(quantize_matmul({{}}, {{}}))
out.append(quantize_matmul(dict(dtype=0), {{}}))
out.append(quantize_matmul(dict(rows=4096), dict(M=4096, N=4096)))
out.append(quantize_matmul(dict(rows=0), dict(M=0)))
""")
    want = [w[0] for w in wrong] + ["null operand"] * 6 + ["16-byte aligned"] * 2 + ["null descriptor"] * 2
    for message, why in zip(got, want):
        assert isinstance(message, str) and why in message, (why, message)
    assert [len(g) for g in got[len(want):]] == [1, 2, 2, 0], got[len(want):]


def test_calls_without_rows_launch_nothing(run):  # noqa: F811
    got = run(CALLS + """
out.append(grouped(T=0, args=(None,) * 4))
out.append(mx4_matmul((None,) * 6, M=0))
out.append(mx4("xtc_hip_mx4_quantize", (None,) * 4, rows=0))
""")
    assert got == [[]] * 3


def test_gradients_are_split_where_scratch_can_be_had(run):  # noqa: F811
    """Few tiles over many rows: in parts with scratch of the stream; one part on a
    stream that is being captured and where there is no memory."""
    got = run(CALLS + """
def grad():
    return grouped("xtc_hip_grouped_matmul_grad_w", E=1, T=32768, K=256, N=256)
fake.fake_memory(1 << 10)
out.append(grad())
fake.fake_memory((1 << 32) - 1)
fake.fake_capturing(1)
out.append(grad())
fake.fake_capturing(0)
out.append(grad())
""")
    (none,), (captured,), (split, total) = got  # a second kernel adds the parts up
    assert none == captured and none[0] == split[0] and total[0] == "grouped_grad_sum"
    # 16 tiles in 16 parts; grids are filled up to whole runs (128 workgroups)
    assert (int(none[1].split()[0]), int(split[1].split()[0])) == (128, 256)


def test_mx4_tiles_by_size(run):  # noqa: F811
    """Few tiles go to waves that share their depth, more to the DMA tiles that cost
    least, blocks of no whole slabs to the kernel of any."""
    got = run(CALLS + """
for M, N, blocks in ((16, 8192, 256), (32, 8192, 256), (700, 1000, 12), (2100, 2056, 68), (4100, 3336, 36), (2100, 2056, 69)):
    out.append(mx4_matmul(M=M, N=N, blocks=blocks))
""")
    want = ["mx4_rows<float, 1,", "mx4_rows<float, 2,", "2, 2, 2, 2, 4, false>", "2, 2, 4, 4, 2, false>", "2, 4, 8, 4, 2, true>", "mx4_any"]
    for ((name, _),), part in zip(got, want, strict=True):
        assert part in name, (name, part)
