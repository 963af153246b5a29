"""The paged cache held in 8 bits, without a device: the format's definition, and what its operators refuse."""
import numpy as np
import pytest
import torch

from oracle import quant_cache
from tests.test_host_calls import fake  # noqa: F401  (the fixture)


def test_the_table_is_e4m3():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(codes, quant_cache.VALUES) and codes[-1] == quant_cache.LARGEST


@pytest.mark.parametrize("width", [4, 64, 130])
def test_rows_are_rounded_once_to_the_nearest_code(width):
    """Against torch's own cast of the exactly scaled row; sizes from the smallest f32 to the largest."""
    rng = np.random.default_rng(width)
    size = 2.0 ** rng.integers(-149, 128, (400, 1))
    rows = (rng.standard_normal((400, width)) * size).clip(-3.4e38, 3.4e38).astype(np.float32)
    rows[0], rows[1, 1:], rows[2, 0] = 0.0, 0.0, 448.0 * 2.0 ** 3
    codes, scales = quant_cache.encode_rows(rows)
    assert scales.min() >= 1 and scales.max() <= 247
    factor = 2.0 ** (scales.astype(np.float64) - 127)[:, None]
    most = np.abs(rows.astype(np.float64)).max(-1)
    assert (most <= 448.0 * factor[:, 0]).all() and ((most > 224.0 * factor[:, 0]) | (scales == 1)).all()
    cast = torch.from_numpy(rows.astype(np.float64) / factor).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    exact = (rows / factor).astype(np.float32) == rows / factor      # (the cast's own input is rounded elsewhere: subnormals)
    assert np.array_equal(codes[exact], cast[exact]) and exact.mean() > 0.9
    error = np.abs(quant_cache.decode_rows(codes, scales) - rows)
    assert (error <= np.maximum(np.abs(rows) * 2.0 ** -4, 2.0 ** -10 * factor)).all()


def test_rows_with_no_number():
    rows = np.array([[np.inf, 1.0, -3.0, np.nan], [np.nan] * 4, [-np.inf, 0.0, 0.0, -0.0]], np.float32)
    values = quant_cache.decode_rows(*quant_cache.encode_rows(rows))
    finite = np.isfinite(rows)
    assert np.array_equal(np.isnan(values), ~finite)
    assert np.array_equal(values[finite], rows[finite])


CACHE = """
P, pt, H, D, lanes, T = 6, 16, 2, 128, 3, 3
codes = lambda p=P, t=pt, h=H, w=D // 4, dtype=DType.U32: hip.alloc(dtype, (p, t, h, w))
scales = lambda p=P, h=H, w=pt // 4: hip.alloc(DType.U32, (p, 2, h, w))
table, tables = hip.alloc(DType.U32, (4, 2)), hip.alloc(DType.U32, (lanes, 4, 2))
gens, cu, starts = hip.alloc(DType.U32, (P,)), hip.alloc(DType.U32, (lanes + 1,)), hip.alloc(DType.U32, (lanes,))
active, one = hip.alloc(DType.U32, (lanes,)), hip.alloc(DType.U32, (1,))
rows = lambda t=T, h=H, d=D, dtype=DType.BF16: hip.alloc(dtype, (t, h, d))

def submit(op, inputs, outputs):
    commands = CommandList()
    commands.dispatch_many(op, inputs, outputs)
    hip.submit(commands).wait()

def refused(op, inputs, outputs):
    launched()
    try:
        submit(op, inputs, outputs)
    except BackendError as e:
        assert e.status.name == "INVALID_INPUT", e
        assert launched() == [], "a refused dispatch launches nothing"
        return
    raise SystemExit(f"accepted: {op} {[t.shape for t in inputs]} {[t.shape for t in outputs]}")
"""


def test_copies_that_are_refused(fake):  # noqa: F811
    fake(CACHE + """
from dataclasses import replace
into, out = (lambda start=0, page=pt: Op.paged_quant_copy(0, start, page)), (lambda start=0, page=pt: Op.paged_quant_copy(1, start, page))
plane = lambda t=None, index=0: (scales() if t is None else t).narrow(1, index, 1)
flat = hip.alloc(DType.U32, (P, H, pt // 4))
# what is taken: both directions, planes of a cache's scales, activity, any float, no rows, the last position
held = scales()
from forja_amd.core import Layout
def as_plane(t, index):
    p, _, h, w = t.shape
    return t.with_layout(Layout(DType.U32, index * h * w, (p, h, w), (2 * h * w, w, 1), t.layout.buffer_len))
for s in (flat, as_plane(held, 0), as_plane(held, 1)):
    for dtype in (DType.BF16, DType.F16, DType.F32):
        submit(into(), [rows(dtype=dtype), table, gens], [codes(), s])
        submit(out(), [codes(), s, table, gens, one], [rows(dtype=dtype)])
submit(into(64), [rows(0), table, gens], [codes(), flat])
submit(into(61), [rows(), table, gens, one], [codes(), flat])
submit(out(61), [codes(), flat, table, gens], [rows()])
assert len(launched()) > 0
good = [rows(), table, gens]
refused(into(62), good, [codes(), flat])                                         # past the table
refused(out(62), [codes(), flat, table, gens], [rows()])
refused(into(0, 0), good, [codes(), flat])                                       # page sizes
refused(into(0, 8), good, [codes(), flat])
refused(replace(into(), bits=4), good, [codes(), flat])
refused(replace(into(), direction=2), good, [codes(), flat])
refused(into(), [rows(d=64), table, gens], [codes(), flat])                      # widths, heads, types
refused(into(), [rows(h=1), table, gens], [codes(), flat])
refused(into(), [rows(dtype=DType.U32), table, gens], [codes(), flat])
refused(into(), [rows(d=516), table, gens], [codes(w=129), flat])
refused(into(), good, [codes(dtype=DType.F32), flat])
refused(into(), good, [codes(), hip.alloc(DType.F32, (P, H, pt // 4))])
refused(into(), good, [codes(), hip.alloc(DType.U32, (P, H, pt // 4 + 1))])
refused(into(), good, [codes(), flat.with_layout(Layout(DType.U32, 0, (P, H, 4), (4, 4, 1), flat.layout.buffer_len))])  # pages overlap
refused(into(), good, [codes(), hip.alloc(DType.U32, (P, pt // 4, H)).permute([0, 2, 1])])
refused(into(), [rows(), table, hip.alloc(DType.U32, (P + 1,))], [codes(), flat])
refused(into(), [rows(), hip.alloc(DType.U32, (4, 3)), gens], [codes(), flat])
refused(into(), [rows(), table, gens, active], [codes(), flat])
refused(into(), [rows(), table], [codes(), flat])
refused(into(), good, [codes()])
refused(out(), [codes(), flat, table], [rows()])
same = hip.alloc(DType.U32, (P, pt, H, D // 4))                                  # codes and scales in one place
refused(into(), good, [same, same.with_layout(Layout(DType.U32, 0, (P, H, 4), (8, 4, 1), same.layout.buffer_len))])
""")


def test_attention_that_is_refused(fake):  # noqa: F811
    fake(CACHE + """
from dataclasses import replace
Hq = 4
op = Op.paged_quant_attention_ragged(0.1, pt)
q = lambda t=T, h=Hq, d=D, dtype=DType.BF16: hip.alloc(dtype, (t, h, d))
ins = lambda **kw: [kw.get("q", q()), kw.get("k", rows()), kw.get("v", rows()), kw.get("tables", tables), kw.get("gens", gens),
                    kw.get("cu", cu), kw.get("starts", starts)]
outs = lambda **kw: [kw.get("out", q()), kw.get("kc", codes()), kw.get("vc", codes()), kw.get("scales", scales())]
for dtype in (DType.BF16, DType.F16, DType.F32):
    submit(op, ins(q=q(dtype=dtype), k=rows(dtype=dtype), v=rows(dtype=dtype)), outs())
    submit(Op.paged_quant_attention_ragged(0.1, pt, True), ins() + [active], outs(out=q(dtype=dtype)))
submit(op, ins(q=q(0), k=rows(0), v=rows(0)), outs(out=q(0)))
submit(op, ins(v=rows(d=64)), outs(out=q(d=64), vc=codes(w=16)))
assert len(launched()) > 0
for page in (0, 8, 32):
    refused(Op.paged_quant_attention_ragged(0.1, page), ins(), outs())
refused(Op.paged_quant_attention_ragged(float("inf"), pt), ins(), outs())
refused(replace(op, bits=4), ins(), outs())
refused(replace(op, k=2), ins(), outs())
refused(op, ins(q=q(h=3)), outs(out=q(h=3)))
refused(op, ins(q=q(dtype=DType.F32)), outs())                       # new rows of another type than the queries
refused(op, ins(q=q(d=64)), outs(out=q(d=64)))
refused(op, ins(v=rows(d=260)), outs(out=q(d=260), vc=codes(w=65)))   # wider values than there are kernels for
refused(op, ins(k=rows(h=1)), outs())
refused(op, ins(k=rows(t=2)), outs())
refused(op, ins(), outs(out=q(dtype=DType.U32)))
refused(op, ins(), outs(vc=codes(p=P + 1)))
refused(op, ins(), outs(scales=hip.alloc(DType.U32, (P, 1, H, pt // 4))))
refused(op, ins(), outs(scales=hip.alloc(DType.U32, (P, 2, H, pt // 2))))
refused(op, ins(), outs(scales=hip.alloc(DType.U32, (P, H, 2, pt // 4)).permute([0, 2, 1, 3])))
refused(op, ins(cu=hip.alloc(DType.U32, (lanes,))), outs())
refused(op, ins(starts=hip.alloc(DType.U32, (lanes + 1,))), outs())
refused(op, ins(gens=hip.alloc(DType.U32, (P + 1,))), outs())
refused(op, ins(tables=hip.alloc(DType.U32, (lanes, 4, 3))), outs())
refused(op, ins() + [one], outs())
refused(op, ins()[:6], outs())
refused(op, ins(), outs()[:3])
pool = codes()
refused(op, ins(), outs(kc=pool, vc=pool))
""")


def test_workspace_is_asked_for_the_splits_there_are(fake):  # noqa: F811
    """Rows that are attended in one piece have no partial results: static submissions take any number of them, and ordinary ones
    keep no memory for them."""
    fake("""
def batch(tokens, lanes, heads, promise=False):
    pools = [hip.alloc(DType.U32, (4, 16, 4, 32)) for _ in range(2)] + [hip.alloc(DType.U32, (4, 2, 4, 4))]
    rows = [hip.alloc(DType.BF16, (tokens, h, 128)) for h in (heads, 4, 4)]
    words = [hip.alloc(DType.U32, s) for s in ((lanes, 4, 2), (4,), (lanes + 1,), (lanes,))]
    commands = CommandList()
    commands.dispatch_many(Op.paged_quant_attention_ragged(0.1, 16, promise), rows + words, [hip.alloc(DType.BF16, (tokens, heads, 128)), *pools])
    return commands
for tokens, lanes, heads in ((2600, 1, 32), (9000, 3, 32), (2600, 2600, 32), (700, 2, 128)):
    for promise in {False, tokens == lanes}:
        launched()
        hip.submit_static(batch(tokens, lanes, heads, promise))
        assert any("prompt_kernel" in name or "decode_kernel" in name for name in launched())
big = batch(8256, 70, 40)
held = hip.memory_usage()
hip.submit(big).wait()
# 117 splits of 70 lanes' single rows; 20 KiB and 8 bytes a head for each
assert hip.memory_usage() - held < (70 * 117 * 40 * 520 + (4 << 20)), hip.memory_usage() - held
""")


@pytest.mark.parametrize("promise", [False, True])
def test_a_plan_ends_with_the_lanes_that_it_is_of(fake, promise):  # noqa: F811
    """Layers of a submission share a plan until one of its inputs is written; static submissions too."""
    fake(CACHE + f"""
tokens, promise = {3 if promise else 9}, {promise}
op = Op.paged_quant_attention_ragged(0.1, pt, promise)
rows = [hip.alloc(DType.BF16, (tokens, h, D)) for h in (4, H, H)]
words = [tables, gens, cu, starts, active]
out, pools = hip.alloc(DType.BF16, (tokens, 4, D)), [codes(), codes(), scales()]
for written in words + [pools[2]]:
    source = hip.alloc(DType.U32, written.shape)
    commands = CommandList()
    for layer in range(2):
        commands.dispatch_many(op, rows + words, [out, *pools])
    commands.dispatch(Op.copy(), [source], written)
    for layer in range(2):
        commands.dispatch_many(op, rows + words, [out, *pools])
    for submit_list in (lambda: hip.submit(commands).wait(), lambda: hip.submit_static(commands)):
        launched()
        submit_list()
        names = ["plan" if "prepare_kernel" in n else "attend" for n in launched() if "prepare_kernel" in n or "prompt_kernel" in n or "decode_kernel" in n]
        want = ["plan", "attend", "attend"] * 2 if written is not pools[2] else ["plan"] + ["attend"] * 4
        assert names == want, (written.shape, names)
""")
