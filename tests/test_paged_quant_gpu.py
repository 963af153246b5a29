"""The paged cache held in 8 bits on the device, against its definition in 64 bits (oracle/quant_cache.py).

What is stored, and what is read back, has no freedom: bits are compared.  An attended row o = sum w v may be off by
  * the rounding of the output: half a step, eps / 2 of |o|;
  * the rounding of the weights, each by at most `weight` of itself: weight * A, A = sum w |v|.  2^-8 where weights are
    bf16, 2^-16 where they are two bf16 pieces;
  * the scores: 2 delta A (a weight and the sum it is divided by), delta the largest error of a score.  Products are
    exact; 2^-24 of S = |scale| sum |q k| for each of up to 512 f32 additions and for each of four factors is below
    2^-14 S at worst (the scaled products of 8-bit codes keep about 2^-13 of the largest of the products they add:
    within that, as no product here is half of S); and a query element is held to 2^-18 of its row's largest at least: 2^-18 Z, Z = |scale| max|q|
    sum |k|.  exp adds a few f32 steps: 2^-21;
  * the f32 sums over n keys, n / 4 + 64 additions in a chain at most: (n / 4 + 64) 2^-23 A."""
import math

import numpy as np
import pytest

from forja_amd.core import BackendError, CommandList, DType, INTO_PAGES, Layout, OUT_OF_PAGES, Op, Status
from oracle import cpu_backend as orc
from oracle import quant_cache
from tests.helpers import from_f32, to_f32, upload

pytestmark = pytest.mark.gpu

HALF_STEP = {DType.F32: 2.0 ** -24, DType.F16: 2.0 ** -11, DType.BF16: 2.0 ** -8}


def rounded(values, dtype):
    return to_f32(from_f32(np.asarray(values), dtype), dtype).reshape(np.shape(values))


def run(backend, op, inputs, outputs, static=False):
    commands = CommandList()
    commands.dispatch_many(op, inputs, outputs)
    if static:
        backend.submit_static(commands)
    else:
        backend.submit(commands).wait()


def within(got, want, bound):
    beyond = np.where(np.isnan(got) | np.isnan(want), np.inf, np.abs(got - want) - bound)
    worst = np.unravel_index(np.argmax(beyond), beyond.shape)
    assert beyond[worst] <= 0, f"{worst}: {got[worst]} for {want[worst]}, {bound[worst]} allowed"


def padded(page_tokens):
    return -(-page_tokens // 4) * 4


def plane_of(scales, index):
    """One plane [P, H, w] of a cache's scales [P, 2, H, w]."""
    p, _, h, w = scales.shape
    return scales.with_layout(Layout(DType.U32, index * h * w, (p, h, w), (2 * h * w, w, 1), scales.layout.buffer_len))


def read_bytes(backend, tensor):
    return np.frombuffer(backend.read_buffer_range(tensor.buffer, 0, tensor.layout.buffer_len), np.uint8)


def hard_rows(rng, shape, dtype):
    """Rows of very different sizes with ties, zeros of both signs, infinities and no numbers among them."""
    values = rng.standard_normal(shape) * 2.0 ** rng.integers(-20, 14, (*shape[:2], 1))
    flat = values.reshape(-1, shape[-1])
    for i, row in enumerate(flat):
        if i % 7 == 1:
            row[:] = rng.integers(-64, 65, row.shape) * 2.0 ** (i % 5)      # many ties
        elif i % 7 == 2:
            row[:] = rng.choice([0.0, -0.0], row.shape)
        elif i % 7 == 3:
            row[rng.integers(row.size)] = rng.choice([np.inf, -np.inf, np.nan])
        elif i % 7 == 4 and dtype != DType.F16:
            row[:] *= rng.choice([2.0 ** -126, 2.0 ** -100, 2.0 ** 100])
        elif i % 7 == 5:
            row[:] = rng.choice([448.0, 449.0, 464.0, 1.75, 1.8], row.shape) * 2.0 ** (i % 4)
    with np.errstate(over="ignore"):
        return rounded(values, dtype)


# ------------------------------------------------------------------ storing and reading back

COPIES = [
    # rows, heads, width, page_tokens, start, dtype, view of the rows
    (1, 8, 128, 16, 0, DType.BF16, "dense"), (1, 1, 4, 1, 2, DType.F32, "dense"), (37, 8, 128, 16, 5, DType.BF16, "dense"),
    (700, 4, 128, 16, 21, DType.F32, "dense"), (65, 2, 64, 48, 47, DType.F16, "dense"), (33, 3, 256, 32, 0, DType.BF16, "dense"),
    (9, 2, 512, 16, 7, DType.F32, "dense"), (20, 5, 132, 3, 1, DType.F16, "dense"), (12, 2, 20, 5, 4, DType.BF16, "dense"),
    (50, 8, 128, 16, 3, DType.BF16, "heads first"), (21, 2, 64, 16, 0, DType.F32, "every other"),
    (30, 4, 128, 16, 9, DType.F16, "of wider rows"), (30, 4, 128, 16, 9, DType.BF16, "odd offset"),
]


def rows_view(backend, values, dtype, form):
    """`values` [T, H, D] through a view; and what its whole storage holds, to see what else is written."""
    t, h, d = values.shape
    if form == "heads first":
        return upload(backend, values.transpose(1, 0, 2), dtype).permute([1, 0, 2])
    shape, offset, strides = {"dense": ((t, h, d), 0, None), "every other": ((t, h, 2 * d), 1, (2 * h * d, 2 * d, 2)),
                              "of wider rows": ((t, h + 2, d), d, ((h + 2) * d, d, 1)),
                              "odd offset": ((t * h * d + 3,), 3, (h * d, d, 1))}[form]
    whole = np.full(int(np.prod(shape)), 7.0, np.float32)
    layout = Layout.contiguous(dtype, 0, (t, h, d), whole.size * dtype.byte_size) if strides is None else \
        Layout(dtype, offset, (t, h, d), strides, whole.size * dtype.byte_size)
    at = np.lib.stride_tricks.as_strided(whole[layout.offset:], (t, h, d), [4 * s for s in layout.strides])
    at[...] = values
    return upload(backend, whole, dtype).with_layout(layout)


def shuffled_table(rng, pages, physical, longer=0):
    order = rng.permutation(physical)[:pages]
    table = np.zeros((pages + longer, 2), np.uint32)
    table[:, 1] = 0xffffffff
    table[:pages] = np.stack([order, 11 + order], 1)
    return table


@pytest.mark.parametrize("rows,heads,width,pt,start,dtype,form", COPIES)
def test_rows_into_pages_and_out(hip, rows, heads, width, pt, start, dtype, form):
    rng = np.random.default_rng(rows * width)
    values = hard_rows(rng, (rows, heads, width), dtype)
    pages = -(-(start + rows) // pt)
    physical, w = pages + 3, padded(pt) // 4
    table = shuffled_table(rng, pages, physical, longer=2)
    codes = rng.integers(0, 256, (physical, pt, heads, width), dtype=np.uint8)
    scales = rng.integers(0, 248, (physical, 2, heads, 4 * w), dtype=np.uint8)
    codes_t, scales_t = (upload(hip, a.view(np.uint32), DType.U32) for a in (codes, scales))
    table_t, gens = upload(hip, table, DType.U32), upload(hip, 11 + np.arange(physical), DType.U32)
    plane = rows % 2
    run(hip, Op.paged_quant_copy(INTO_PAGES, start, pt), [rows_view(hip, values, dtype, form), table_t, gens],
        [codes_t, plane_of(scales_t, plane)])
    position = start + np.arange(rows)
    page, slot = table[position // pt, 0], position % pt
    codes[page, slot], scales[page, plane, :, slot] = quant_cache.encode_rows(values)
    got = read_bytes(hip, codes_t).reshape(codes.shape)
    none = (codes & 0x7f) == 0x7f                       # the sign of no number is not told
    assert np.array_equal(got & 0x7f, codes & 0x7f) and np.array_equal(got[~none], codes[~none])
    assert np.array_equal(read_bytes(hip, scales_t).reshape(scales.shape), scales)
    # and out again, in every type
    for out_dtype in (dtype, DType.F32, DType.BF16):
        out = rows_view(hip, np.full(values.shape, 3.0, np.float32), out_dtype, form)
        before = read_bytes(hip, out).copy()
        run(hip, Op.paged_quant_copy(OUT_OF_PAGES, start, pt), [codes_t, plane_of(scales_t, plane), table_t, gens], [out])
        with np.errstate(over="ignore"):
            want = rounded(quant_cache.decode_rows(codes[page, slot], scales[page, plane, :, slot]).astype(np.float32), out_dtype)
        assert np.array_equal(to_f32(hip.read(out), out_dtype).reshape(want.shape), want, equal_nan=True)
        seen = np.zeros(before.size // out_dtype.byte_size, bool)
        np.lib.stride_tricks.as_strided(seen[out.layout.offset:], out.shape, out.layout.strides)[...] = True
        other = np.repeat(~seen, out_dtype.byte_size)
        assert np.array_equal(read_bytes(hip, out)[other], before[other])


def test_copies_of_an_inactive_lane_and_through_refused_entries(hip):
    rng = np.random.default_rng(2)
    values = rng.standard_normal((40, 2, 128)).astype(np.float32)
    table = shuffled_table(rng, 4, 6)
    gens = upload(hip, 11 + np.arange(6), DType.U32)
    codes, scales = hip.alloc(DType.U32, (6, 16, 2, 32)), hip.alloc(DType.U32, (6, 2, 4))
    rows = upload(hip, values, DType.F32)
    zero, one = upload(hip, np.array([0]), DType.U32), upload(hip, np.array([1]), DType.U32)
    run(hip, Op.paged_quant_copy(INTO_PAGES, 3, 16), [rows, upload(hip, table, DType.U32), gens, zero], [codes, scales])
    assert not read_bytes(hip, codes).any() and not read_bytes(hip, scales).any()
    for broken in ((2, 1, 99), (1, 0, 6), (1, 0, 0xffffffff)):      # a stale generation, pages that are not there
        bad = table.copy()
        bad[broken[0], broken[1]] = broken[2]
        for op, inputs, outputs in ((Op.paged_quant_copy(INTO_PAGES, 3, 16), [rows], [codes, scales]),
                                    (Op.paged_quant_copy(OUT_OF_PAGES, 3, 16), [codes, scales], [upload(hip, values, DType.F32)])):
            with pytest.raises(BackendError) as info:
                run(hip, op, inputs + [upload(hip, bad, DType.U32), gens, one], outputs)
            assert info.value.status == Status.DEVICE_ERROR_FLAG and info.value.index == broken[0]
        position = 3 + np.arange(40)
        whole = position // 16 != broken[0]
        got = to_f32(hip.read(outputs[0]), DType.F32).reshape(values.shape)
        assert np.array_equal(got[~whole], values[~whole])                    # left as they were
        assert np.array_equal(got[whole], quant_cache.decode_rows(*quant_cache.encode_rows(values[whole])).astype(np.float32))


# ------------------------------------------------------------------ attention

class Batch:
    """A ragged batch over an 8-bit cache: numpy arrays, and the tensors of a backend made from them.  Slots that hold no
    key are codes of no number, with a scale byte that makes them so large as they can be."""

    def __init__(self, contexts, counts, hq, hkv, pt, width=128, value_width=None, dtype=DType.BF16, out_dtype=None, seed=1,
                 activity=None, spread=0, make=None):
        rng = np.random.default_rng(seed)
        value_width = width if value_width is None else value_width
        self.contexts, self.counts, self.pt, self.dtype = contexts, counts, pt, dtype
        self.out_dtype = dtype if out_dtype is None else out_dtype
        self.hq, self.hkv, self.activity = hq, hkv, activity
        lanes, tokens = len(contexts), sum(counts)
        need = [-(-(c + n) // pt) for c, n in zip(contexts, counts)]
        self.physical = sum(need) + 3
        order = rng.permutation(self.physical)
        self.tables = np.zeros((lanes, max(need) + 2, 2), np.uint32)
        self.tables[:, :, 1] = 0xffffffff
        at = 0
        for lane, n in enumerate(need):
            self.tables[lane, :n] = np.stack([order[at:at + n], 11 + order[at:at + n]], 1)
            at += n
        self.cu = np.concatenate([[0], np.cumsum(counts)])
        make = make or (lambda what, shape: rng.standard_normal(shape) * 2.0 ** rng.integers(-spread, spread + 1, (*shape[:2], 1)))
        self.q, self.k_new, self.v_new = (rounded(make(what, shape), dtype) for what, shape in (
            ("q", (tokens, hq, width)), ("k", (tokens, hkv, width)), ("v", (tokens, hkv, value_width))))
        self.codes = [np.full((self.physical, pt, hkv, d), 0x7f, np.uint8) for d in (width, value_width)]
        self.scales = np.full((self.physical, 2, hkv, padded(pt)), 247, np.uint8)
        for lane, context in enumerate(contexts):
            page, slot = self.where(lane, np.arange(context))
            for plane, (what, d) in enumerate((("k", width), ("v", value_width))):
                rows = quant_cache.encode_rows(make(what, (context, hkv, d)))
                self.codes[plane][page, slot], self.scales[page, plane, :, slot] = rows

    def where(self, lane, position):
        return self.tables[lane, position // self.pt, 0], position % self.pt

    def upload(self, hip):
        u32 = lambda a: upload(hip, np.ascontiguousarray(a), DType.U32)  # noqa: E731
        self.out = upload(hip, np.full((*self.q.shape[:2], self.v_new.shape[2]), 5.0, np.float32), self.out_dtype)
        self.cache = [u32(a.view(np.uint32)) for a in (*self.codes, self.scales)]
        self.inputs = [upload(hip, a, self.dtype) for a in (self.q, self.k_new, self.v_new)]
        self.inputs += [u32(self.tables), u32(11 + np.arange(self.physical)), u32(self.cu), u32(np.array(self.contexts))]
        if self.activity is not None:
            self.inputs.append(u32(np.array(self.activity)))
        return self

    def attend(self, hip, scale, promise=False, static=False):
        run(hip, Op.paged_quant_attention_ragged(scale, self.pt, promise), self.inputs, [self.out, *self.cache], static)
        return to_f32(hip.read(self.out), self.out_dtype).reshape(*self.q.shape[:2], -1)

    def live(self, lane):
        return self.activity is None or self.activity[lane]

    def store(self):
        """What the cache holds after the batch's rows are in it."""
        for lane, (context, count) in enumerate(zip(self.contexts, self.counts)):
            if not self.live(lane):
                continue
            page, slot = self.where(lane, context + np.arange(count))
            for plane, rows in enumerate((self.k_new, self.v_new)):
                rows = quant_cache.encode_rows(rows[self.cu[lane]:self.cu[lane + 1]])
                self.codes[plane][page, slot], self.scales[page, plane, :, slot] = rows

    def expected(self, scale):
        """(attended rows in 64 bits, how far a result may be off)."""
        self.store()
        out = np.zeros((*self.q.shape[:2], self.v_new.shape[2]))
        bound = np.zeros(out.shape)
        weight = 2.0 ** -8 if self.dtype == DType.BF16 and self.out_dtype != DType.F32 else 2.0 ** -16
        for lane, (context, count) in enumerate(zip(self.contexts, self.counts)):
            if not self.live(lane) or count == 0:
                continue
            page, slot = self.where(lane, np.arange(context + count))
            keys, values = (quant_cache.decode_rows(self.codes[p][page, slot], self.scales[page, p, :, slot]) for p in range(2))
            rows = slice(self.cu[lane], self.cu[lane + 1])
            q = self.q[rows].astype(np.float64)
            o, a, s = quant_cache.attend(q, keys, values, float(np.float32(scale)), context + 1 + np.arange(count))
            z = abs(scale) * np.abs(q).max(-1, keepdims=True) * np.repeat(np.nan_to_num(np.abs(keys)).sum(-1).max(0), self.hq // self.hkv)[:, None]
            delta = 2.0 ** -14 * s + 2.0 ** -18 * z + 2.0 ** -21
            n = context + count
            out[rows] = o
            bound[rows] = (HALF_STEP[self.out_dtype] * (np.abs(o) + weight * a) + (weight + 2 * delta + (n / 4 + 64) * 2.0 ** -23) * a)
        return out, bound

    def check(self, hip, scale, promise=False, static=False):
        got = self.upload(hip).attend(hip, scale, promise, static)
        want, bound = self.expected(scale)
        within(got, want, bound)
        for tensor, array in zip(self.cache, (*self.codes, self.scales)):
            assert np.array_equal(read_bytes(hip, tensor).reshape(array.shape), array)
        return got


BATCHES = [
    # contexts, new rows per lane, query heads, kv heads, page_tokens
    ([17, 64, 130, 511], [1, 1, 1, 1], 16, 8, 16),
    ([300, 1, 2047, 700, 15, 16, 0], [1] * 7, 32, 4, 16),
    ([0], [1], 40, 8, 16), ([0], [1], 1, 1, 16), ([3000], [1], 12, 1, 16), ([900, 3], [1, 1], 64, 2, 32),
    ([40, 0, 100], [1, 5, 3], 8, 2, 16),                     # a decode row between prompt chunks
    ([100, 257, 9], [1, 0, 1], 32, 4, 64),                   # a lane that brings nothing
    ([0, 130, 33, 900], [70, 1, 45, 1], 40, 8, 16),
    ([0, 64], [200, 37], 16, 8, 48),
    ([500, 31], [96, 1], 32, 4, 16),
    ([0, 5], [33, 31], 4, 4, 16),
    ([61, 7], [3, 70], 48, 1, 16),                           # 48 query heads on one
    ([4100, 250], [9, 66], 8, 1, 16),
    ([5000, 100, 2500, 33, 9000], [1] * 5, 8, 8, 16),
    ([(37 * i) % 90 for i in range(300)], [1] * 300, 8, 8, 16),
]


@pytest.mark.parametrize("dtype", [DType.BF16, DType.F32])
@pytest.mark.parametrize("contexts,counts,hq,hkv,pt", BATCHES)
def test_attention(hip, contexts, counts, hq, hkv, pt, dtype):
    Batch(contexts, counts, hq, hkv, pt, dtype=dtype, spread=2, seed=sum(contexts)).check(
        hip, 1.0 / math.sqrt(128), promise=max(counts) == 1 and len(contexts) % 2 == 1)


@pytest.mark.parametrize("dtype,out_dtype", [(DType.F16, DType.F16), (DType.BF16, DType.F32), (DType.F32, DType.BF16),
                                             (DType.BF16, DType.F16)])
@pytest.mark.parametrize("contexts,counts", [([70, 300, 2], [1, 1, 1]), ([70, 300, 0], [1, 60, 40])])
def test_attention_across_types(hip, contexts, counts, dtype, out_dtype):
    Batch(contexts, counts, 16, 4, 16, dtype=dtype, out_dtype=out_dtype, spread=1, seed=3).check(hip, 0.09)


@pytest.mark.parametrize("pt,width,value_width", [
    (16, 64, 64), (64, 64, 64), (16, 256, 256), (32, 256, 256), (1, 128, 128), (3, 128, 128), (20, 64, 64), (16, 96, 96),
    (16, 128, 64), (16, 512, 128), (8, 4, 4), (16, 128, 256)])
@pytest.mark.parametrize("contexts,counts", [([70, 300, 2], [1, 1, 1]), ([70, 0, 130], [1, 60, 5])])
def test_attention_across_widths_and_pages(hip, contexts, counts, pt, width, value_width):
    for dtype in (DType.BF16, DType.F32):
        Batch(contexts, counts, 10, 2, pt, width, value_width, dtype=dtype, seed=5).check(hip, 1.0 / math.sqrt(width))


@pytest.mark.parametrize("scale", [0.0, -0.11, 3.0, 1e-30])
@pytest.mark.parametrize("counts", [[1, 1], [40, 1]])
def test_attention_at_unusual_scales(hip, scale, counts):
    for dtype in (DType.BF16, DType.F32):
        Batch([130, 600], counts, 8, 2, 16, dtype=dtype, seed=9).check(hip, scale)


LENGTHS = list(range(0, 70)) + [94, 95, 96, 127, 128, 129, 159, 160, 161, 255, 256, 1022, 1023, 1024, 1025, 1056, 4000]


@pytest.mark.parametrize("pt,width,hq,hkv", [(16, 128, 16, 8), (16, 128, 20, 1), (48, 128, 5, 1), (64, 64, 8, 2), (16, 256, 4, 2),
                                             (5, 128, 2, 1)])
@pytest.mark.parametrize("chunk", [0, 1, 3, 150])
def test_every_key_counts_once(hip, pt, width, hq, hkv, chunk):
    """Queries of zeros weigh every key alike and values are whole numbers: the sums are exact, whatever their order, and a
    row is its values' mean to a few f32 steps.  Decode rows of many lengths, alone (chunk 0) and beside a chunk."""
    rng = np.random.default_rng(pt)
    scales = 2.0 ** rng.integers(-1, 3, 7)

    def make(what, shape):
        if what == "q":
            return np.zeros(shape)
        return rng.integers(-8, 9, shape) * rng.choice(scales, (*shape[:2], 1))     # 17 * 2^3 * 4000 keys: below 2^24
    contexts = LENGTHS + ([700] if chunk else [])
    counts = [1] * len(LENGTHS) + ([chunk] if chunk else [])
    batch = Batch(contexts, counts, hq, hkv, pt, width, out_dtype=DType.F32, make=make, seed=pt + chunk)
    got = batch.upload(hip).attend(hip, 0.1)
    want = batch.expected(0.1)[0]
    # (the reference's own rounding: 4000 weights of 1/n, each off by 2^-53 of itself, times values of up to 64: below 2^-35)
    within(got, want, 4 * 2.0 ** -24 * np.abs(want) + 2.0 ** -35)


def test_inactive_lanes_and_rows_of_no_lane(hip):
    for counts in ([1, 1, 1], [1, 30, 2]):
        batch = Batch([33, 70, 5], counts, 8, 4, 16, activity=[1, 0, 1], seed=4)
        got = batch.check(hip, 0.09)
        assert not got[batch.cu[1]:batch.cu[2]].any()
        # rows behind the last lane belong to none: zeros, and nothing is stored
        batch = Batch([33, 70, 5], counts, 8, 4, 16, seed=4)
        batch.cu = batch.cu.copy()
        batch.cu[3] = batch.cu[2]
        batch.counts = [*counts[:2], 0]
        got = batch.check(hip, 0.09)
        assert not got[batch.cu[3]:].any() and got[:batch.cu[3]].any()


@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 30, 2]])
@pytest.mark.parametrize("width", [128, 96])
def test_refused_pages_batches_and_promises(hip, counts, width):
    def refused(batch, promise=False):
        batch.upload(hip)
        with pytest.raises(BackendError) as info:
            batch.attend(hip, 0.09, promise)
        assert info.value.status == Status.DEVICE_ERROR_FLAG
        return info.value.index, to_f32(hip.read(batch.out), batch.out_dtype).reshape(*batch.q.shape[:2], -1)

    for entry, value, index in (((1, 2, 1), 3, 2), ((1, 0, 0), 0xfffffff0, 0)):
        batch = Batch([33, 70, 5], counts, 8, 4, 16, width, seed=6)
        want, bound = Batch([33, 70, 5], counts, 8, 4, 16, width, seed=6).expected(0.09)
        batch.tables[entry] = value
        at, got = refused(batch)
        assert at == index
        assert not got[batch.cu[1]:batch.cu[2]].any()
        for lane in (0, 2):
            rows = slice(batch.cu[lane], batch.cu[lane + 1])
            within(got[rows], want[rows], bound[rows])
    # a lane whose rows pass its table
    batch = Batch([33, 70, 5], counts, 8, 4, 16, width, seed=6)
    batch.tables = batch.tables[:, :5]                      # 80 tokens
    batch.contexts = [33, 80, 5]
    at, got = refused(batch)
    assert at == 5 and not got[batch.cu[1]:batch.cu[2]].any() and got[0].any()
    # token ranges that run backwards or past the batch: zeros, and the cache is left alone
    for cu, index in (([0, 2, 1, 3], 1), ([0, 1, 2, sum(counts) + 1], 2), ([5, 1, 2, 3], 0)):
        batch = Batch([33, 70, 5], counts, 8, 4, 16, width, seed=6)
        batch.cu = np.array(cu)
        at, got = refused(batch)
        assert at == index and not got.any()
        for tensor, array in zip(batch.cache, (*batch.codes, batch.scales)):
            assert np.array_equal(read_bytes(hip, tensor).reshape(array.shape), array)
    # the promise of one row a lane
    if max(counts) > 1:
        batch = Batch([33, 70, 5], counts, 8, 4, 16, width, seed=6)
        at, got = refused(batch, promise=True)
        # the lane's rows read zero, and nothing of it is stored
        assert at == batch.cu[1] and not got[1:].any() and got[0].any()
        page, slot = batch.where(1, 70 + np.arange(30))
        assert (read_bytes(hip, batch.cache[0]).reshape(batch.codes[0].shape)[page, slot] == 0x7f).all()


def test_no_numbers_stay_in_the_rows_that_attend_them(hip):
    """A key or value of no number in one head of one lane; an infinite query is no number in its own row alone."""
    for counts in ([1, 1, 1], [20, 1, 33]):
        for where in ("k", "v", "q"):
            batch = Batch([40, 33, 70], counts, 8, 2, 16, seed=8)
            if where == "q":
                batch.q[batch.cu[1], 5, 3] = np.inf
            else:
                page, slot = batch.where(2, np.array([35]))
                batch.codes["kv".index(where)][page[0], slot[0], 1, 7] = 0x7f
            got = batch.upload(hip).attend(hip, 0.09)
            bad = np.isnan(got)
            assert not bad[:batch.cu[1]].any()
            if where == "q":
                assert bad[batch.cu[1], 5].all() and bad.sum() == 128
            else:
                rows = bad[batch.cu[2]:]
                assert not rows[:, :4].any() and not bad[batch.cu[1]].any()
                assert rows[:, 4:].all() if where == "k" else (rows[:, 4:, 7].all() and rows.sum() == rows[:, 4:, 7].size)


@pytest.mark.parametrize("dtype,hq,hkv,width", [(DType.BF16, 8, 2, 128), (DType.F32, 16, 1, 128), (DType.BF16, 5, 1, 64),
                                                (DType.F16, 4, 4, 64), (DType.BF16, 6, 2, 96)])
def test_no_numbers_among_new_rows_reach_no_row_before_them(hip, dtype, hq, hkv, width):
    """What a causal mask hides may be anything: rows before it are as they are without it, those from it on have what they
    attend of it, in its columns."""
    batch = Batch([40, 3, 70], [100, 1, 37], hq, hkv, 16, width, dtype=dtype, seed=18)
    rng = np.random.default_rng(19)
    for token in (17, 63, 64, 99, 100, 120):
        batch.v_new[token, rng.integers(hkv), rng.integers(width, size=3)] = rng.choice([np.nan, np.inf, -np.inf], 3)
    batch.k_new[80, 0, 5] = np.inf
    got = batch.upload(hip).attend(hip, 0.09)
    want, bound = batch.expected(0.09)
    assert np.isnan(want).any(axis=2).sum() < 0.9 * want[:, :, 0].size
    assert np.array_equal(np.isnan(got), np.isnan(want))
    number = ~np.isnan(want)
    within(got[number], want[number], bound[number])


def test_a_cache_does_not_depend_on_how_its_sequence_came(hip):
    """A prompt in one chunk, in several, and by PagedQuantCopy: the same codes and scales; and reading them back gives what
    attention reads.  Then decode steps."""
    rng = np.random.default_rng(12)
    hq, hkv, pt, n = 8, 2, 16, 150
    q, k, v = (rounded(rng.standard_normal((n, h, 128)), DType.BF16) for h in (hq, hkv, hkv))
    table = shuffled_table(rng, 10, 12)
    held, outs = [], []
    for cuts in ([n], [37, 64, 1, 48], "copy"):
        gens = upload(hip, 11 + np.arange(12), DType.U32)
        cache = [hip.alloc(DType.U32, s) for s in ((12, pt, hkv, 32), (12, pt, hkv, 32), (12, 2, hkv, pt // 4))]
        tables = upload(hip, table[None], DType.U32)
        if cuts == "copy":
            for plane, rows in enumerate((k, v)):
                for at in range(0, n, 50):
                    run(hip, Op.paged_quant_copy(INTO_PAGES, at, pt),
                        [upload(hip, rows[at:at + 50], DType.BF16), upload(hip, table, DType.U32), gens],
                        [cache[plane], plane_of(cache[2], plane)])
        else:
            at, rows_out = 0, []
            for cut in cuts:
                out = hip.alloc(DType.F32, (cut, hq, 128))
                run(hip, Op.paged_quant_attention_ragged(0.09, pt),
                    [*(upload(hip, a[at:at + cut], DType.BF16) for a in (q, k, v)), tables, gens,
                     upload(hip, np.array([0, cut]), DType.U32), upload(hip, np.array([at]), DType.U32)], [out, *cache])
                rows_out.append(to_f32(hip.read(out), DType.F32).reshape(cut, hq, 128))
                at += cut
            outs.append(np.concatenate(rows_out))
        held.append([read_bytes(hip, t).tobytes() for t in cache])
        for plane, rows in enumerate((k, v)):
            back = hip.alloc(DType.F32, (n, hkv, 128))
            run(hip, Op.paged_quant_copy(OUT_OF_PAGES, 0, pt),
                [cache[plane], plane_of(cache[2], plane), upload(hip, table, DType.U32), gens], [back])
            want = quant_cache.decode_rows(*quant_cache.encode_rows(rows))
            assert np.array_equal(to_f32(hip.read(back), DType.F32).reshape(want.shape), want)
    assert held[0] == held[1] == held[2]
    keys, values = (quant_cache.decode_rows(*quant_cache.encode_rows(rows)) for rows in (k, v))
    want, spread, _ = quant_cache.attend(q.astype(np.float64), keys, values, 0.09, 1 + np.arange(n))
    for got in outs:      # two bf16 pieces a weight; scores of a few units in f32
        within(got, want, 2.0 ** -12 * spread)


@pytest.mark.parametrize("contexts,counts", [([700, 33, 1500, 5], [1, 1, 1, 1]), ([0, 700, 33], [70, 1, 45])])
def test_static_submissions_give_the_same_bits(hip, contexts, counts):
    for dtype in (DType.BF16, DType.F32):
        outs = []
        for static in (False, True, False):
            batch = Batch(contexts, counts, 16, 4, 16, dtype=dtype, seed=21)
            outs.append(batch.check(hip, 0.09, promise=max(counts) == 1, static=static))
        assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])


def test_layers_of_one_submission_share_their_lanes(hip):
    """Several layers in one list, and a list whose starts change between two of them: each attends as its own."""
    layers = [Batch([70, 300, 5], [1, 1, 1], 16, 8, 16, seed=s) for s in (31, 32, 33)]
    commands = CommandList()
    for layer in layers:
        layer.tables, layer.upload(hip)
        layer.inputs[3:] = layers[0].inputs[3:]
        commands.dispatch_many(Op.paged_quant_attention_ragged(0.09, 16, True), layer.inputs, [layer.out, *layer.cache])
    for layer in layers[1:]:
        own, layer.tables = layer.tables, layers[0].tables
        codes, scales = [c.copy() for c in layer.codes], layer.scales.copy()
        for lane, context in enumerate(layer.contexts):      # the layer's rows under the first one's table
            position = np.arange(context)
            to, slot = layer.where(lane, position)
            at = own[lane, position // 16, 0]
            for plane in range(2):
                layer.codes[plane][to, slot] = codes[plane][at, slot]
                layer.scales[to, plane, :, slot] = scales[at, plane, :, slot]
        for tensor, array in zip(layer.cache, (*layer.codes, layer.scales)):
            hip.write(tensor, array.tobytes())
    later = Batch([9, 2, 64], [1, 1, 1], 16, 8, 16, seed=34).upload(hip)
    commands.dispatch(Op.copy(), [later.inputs[6]], layers[0].inputs[6])
    commands.dispatch(Op.copy(), [later.inputs[3].narrow(1, 0, 7)], layers[0].inputs[3].narrow(1, 0, 7))
    later.inputs[3], later.inputs[6] = layers[0].inputs[3], layers[0].inputs[6]
    later.inputs[4] = layers[0].inputs[4]
    hip.submit(commands).wait()
    for layer in layers:
        got = to_f32(hip.read(layer.out), DType.BF16).reshape(3, 16, 128)
        want, bound = layer.expected(0.09)
        within(got, want, bound)


def test_pages_beyond_32_bits(hip):
    """Pools of over 4 GiB, keys in their last pages."""
    pt, hkv, physical = 64, 8, 70000
    cache = [hip.alloc(DType.U32, s) for s in ((physical, pt, hkv, 32), (physical, pt, hkv, 32), (physical, 2, hkv, pt // 4))]
    try:
        batch = Batch([150, 300], [1, 40], 8, 8, pt, seed=41)
        first = physical - batch.physical
        u32 = lambda a: upload(hip, np.ascontiguousarray(a), DType.U32)  # noqa: E731
        batch.upload(hip)
        tables = batch.tables.copy()
        tables[:, :, 0] += first
        gens = np.zeros(physical, np.uint32)
        gens[first:] = 11 + np.arange(batch.physical)
        for tensor, array in zip(cache, (*batch.codes, batch.scales)):
            hip.write(tensor.narrow(0, first, batch.physical), array.tobytes())
        out = hip.alloc(DType.BF16, (41, 8, 128))
        run(hip, Op.paged_quant_attention_ragged(0.09, pt), [*batch.inputs[:3], u32(tables), u32(gens), *batch.inputs[5:]], [out, *cache])
        got = to_f32(hip.read(out), DType.BF16).reshape(41, 8, 128)
        want, bound = batch.expected(0.09)
        within(got, want, bound)
        back = hip.alloc(DType.F32, (190, 8, 128))
        run(hip, Op.paged_quant_copy(OUT_OF_PAGES, 150, pt),
            [cache[1], plane_of(cache[2], 1), u32(tables[1]), u32(gens)], [back.narrow(0, 0, 190)])
        page, slot = batch.where(1, 150 + np.arange(190))
        want = quant_cache.decode_rows(batch.codes[1][page, slot], batch.scales[page, 1, :, slot])
        assert np.array_equal(to_f32(hip.read(back), DType.F32).reshape(want.shape), want)
    finally:
        for tensor in cache:
            hip.release(tensor)


@pytest.mark.parametrize("lanes,several", [(3000, 0), (4096, 0), (2500, 40), (4097, 0), (4100, 3)])
def test_as_many_lanes_as_there_may_be(hip, lanes, several):
    """More units than the plan keeps beside it, and more lanes than it takes."""
    contexts = [(41 * i) % 70 for i in range(lanes)]
    counts = [1 + (i % 23 if i % (lanes // several) == 5 else 0) if several else 1 for i in range(lanes)]
    Batch(contexts, counts, 2, 1, 16, 64, seed=lanes).check(hip, 0.125, promise=lanes == 4096)


@pytest.mark.parametrize("hq,hkv", [(128, 1), (129, 1), (33, 1), (200, 2)])
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 30, 3]])
def test_many_query_heads_on_one(hip, hq, hkv, counts):
    for dtype in (DType.BF16, DType.F32):
        Batch([70, 5, 600], counts, hq, hkv, 16, 64, dtype=dtype, seed=hq).check(hip, 0.125)


@pytest.mark.parametrize("contexts,counts,promise", [([70, 300, 2], [1, 1, 1], True), ([70, 300, 2], [1, 1, 1], False),
                                                     ([70, 0, 130], [1, 60, 5], False)])
@pytest.mark.parametrize("of_q,of_k,of_v", [("dense", "every other", "dense"), ("of wider rows", "of wider rows", "odd offset"),
                                            ("odd offset", "dense", "of wider rows"), ("heads first", "heads first", "heads first")])
def test_rows_as_they_lie_in_other_tensors(hip, contexts, counts, promise, of_q, of_k, of_v):
    """Queries and new rows through views that the wide loads take and that they do not, two layers of a submission."""
    for dtype in (DType.BF16, DType.F32):
        batch = Batch(contexts, counts, 8, 2, 16, dtype=dtype, seed=51).upload(hip)
        batch.inputs[:3] = [rows_view(hip, values, dtype, form)
                            for values, form in ((batch.q, of_q), (batch.k_new, of_k), (batch.v_new, of_v))]
        second = [upload(hip, np.zeros(a.shape[:-1] + (a.shape[-1] // 4,)), DType.U32) for a in (*batch.codes, batch.scales)]
        for tensor, array in zip(second, (*batch.codes, batch.scales)):
            hip.write(tensor, array.tobytes())
        again = upload(hip, np.full((*batch.q.shape[:2], 128), 5.0, np.float32), dtype)
        commands = CommandList()
        for out, cache in ((batch.out, batch.cache), (again, second)):
            commands.dispatch_many(Op.paged_quant_attention_ragged(0.09, 16, promise), batch.inputs, [out, *cache])
        hip.submit(commands).wait()
        want, bound = batch.expected(0.09)
        for out, cache in ((batch.out, batch.cache), (again, second)):
            within(to_f32(hip.read(out), dtype).reshape(want.shape), want, bound)
            for tensor, array in zip(cache, (*batch.codes, batch.scales)):
                assert np.array_equal(read_bytes(hip, tensor).reshape(array.shape), array)


def test_two_backends_at_once():
    """Submissions of two backends in turns, none waited for in between: plans and partial results are a backend's own."""
    from forja_amd.hip_backend import HipBackend
    backends = [HipBackend(0), HipBackend(0)]
    batches = [Batch([700, 33, 1500], counts, 16, 4, 16, seed=61).upload(b) for b, counts in zip(backends, ([1, 1, 1], [1, 70, 9]))]
    waiting = []
    for _ in range(4):
        for backend, batch in zip(backends, batches):
            commands = CommandList()
            commands.dispatch_many(Op.paged_quant_attention_ragged(0.09, 16), batch.inputs, [batch.out, *batch.cache])
            waiting.append(backend.submit(commands))
    for submission in waiting:
        submission.wait()
    for backend, batch in zip(backends, batches):
        got = to_f32(backend.read(batch.out), DType.BF16).reshape(*batch.q.shape)
        want, bound = batch.expected(0.09)
        within(got, want, bound)
        backend.close()


@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 30, 3]])
@pytest.mark.parametrize("width", [64, 128])
def test_queries_of_any_size(hip, counts, width):
    """Rows down to the smallest numbers of bf16, whose elements do not come down to one code each: every key then weighs alike,
    and a row is nearly the mean of its values.  And rows of 2^100 under a scale that takes them back."""
    for dtype, out_dtype in ((DType.BF16, DType.BF16), (DType.BF16, DType.F16), (DType.F32, DType.F32)):
        batch = Batch([70, 5, 600], counts, 8, 2, 16, width, dtype=dtype, out_dtype=out_dtype, seed=71)
        sizes = np.arange(-133, -109)
        sizes = np.resize(sizes, batch.q.shape[:2])[..., None]       # every size, with each element's own bits
        batch.q = rounded(np.ldexp(batch.q / np.abs(batch.q).max(-1, keepdims=True), sizes), dtype)
        got = batch.check(hip, 1.0)
        assert np.abs(got).max() > 0
        batch = Batch([70, 5, 600], counts, 8, 2, 16, width, dtype=dtype, out_dtype=out_dtype, seed=72)
        batch.q = rounded(batch.q * 2.0 ** 100, dtype)
        batch.check(hip, 0.09 * 2.0 ** -100)


@pytest.mark.parametrize("hq,hkv,pt,width", [(8, 4, 16, 128), (20, 4, 16, 128), (16, 1, 64, 64), (8, 4, 16, 96), (9, 3, 48, 128)])
@pytest.mark.parametrize("context,count,first", [(70, 30, 80), (0, 200, 96), (3000, 160, 3088), (3000, 160, 2496), (40, 9, 48)])
@pytest.mark.parametrize("past", [False, True])
def test_rows_before_a_refused_page_are_attended(hip, hq, hkv, pt, width, context, count, first, past):
    """A chunk of which a page is stale, or whose rows pass the lane's table, from about position `first` on: rows that attend
    nothing of it are as without it, those that do are zeros, and what has a page of its own is stored."""
    page = -(-first // pt)
    position = context + np.arange(count)
    lost = position[position >= page * pt if past else position // pt == page]
    reached = np.zeros(count + 4, bool)
    reached[1:1 + count] = position + 1 > page * pt
    # (strange: values of no number among the new rows)
    for dtype, strange in ((DType.BF16, False), (DType.BF16, True), (DType.F32, True)):
        batch, whole = (Batch([33, context, 5], [1, count, 3], hq, hkv, pt, width, dtype=dtype, seed=81) for _ in range(2))
        for b in (batch, whole):
            if strange:
                b.v_new[1 + count // 3, 0, 5] = b.v_new[count, hkv - 1, 0] = np.nan
        if past and reached.any():
            batch.tables = batch.tables[:, :page]
        else:
            batch.tables[1, page, 1] ^= 1
        batch.upload(hip)
        if reached.any():
            with pytest.raises(BackendError) as info:
                batch.attend(hip, 0.09)
            assert info.value.status == Status.DEVICE_ERROR_FLAG and info.value.index == page
        else:
            batch.attend(hip, 0.09)
        got = to_f32(hip.read(batch.out), dtype).reshape(*batch.q.shape[:2], -1)
        want, bound = whole.expected(0.09)
        assert not got[reached].any()
        got, want, bound = got[~reached], want[~reached], bound[~reached]
        number = ~np.isnan(want)
        assert np.array_equal(np.isnan(got), ~number)
        within(got[number], want[number], bound[number])
        at, slot = whole.where(1, lost)
        for held, first_held in zip(whole.codes, batch.codes):
            held[at, slot] = first_held[at, slot]
        whole.scales[at, :, :, slot] = batch.scales[at, :, :, slot]
        for tensor, array in zip(batch.cache, (*whole.codes, whole.scales)):
            got = read_bytes(hip, tensor).reshape(array.shape)
            none = (array & 0x7f) == 0x7f                   # the sign of no number is not told
            assert np.array_equal(got & 0x7f, array & 0x7f) and np.array_equal(got[~none], array[~none])


@pytest.mark.parametrize("contexts,counts", [([0, 300, 20], [600, 1, 40]), ([(37 * i) % 50 for i in range(650)], [1] * 650)])
def test_static_batches_whose_splits_do_not_fit(hip, contexts, counts):
    """A partial row for every token of these batches is more than a static submission's 36 MiB: they are attended unsplit."""
    assert sum(counts) * 128 * 128 * 4 > 36 << 20
    Batch(contexts, counts, 128, 8, 16, seed=91).check(hip, 0.09, static=True)


@pytest.mark.parametrize("static", [False, True])
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 30, 3]])
def test_lanes_that_change_between_layers(hip, counts, static):
    """A list that writes the lanes' starts and tables between two layers: each is attended, and stored, by its own."""
    first, later = (Batch(contexts, counts, 16, 8, 16, seed=seed) for contexts, seed in (([70, 300, 5], 31), ([9, 2, 64], 34)))
    pages = max(b.tables.shape[1] for b in (first, later))
    physical = max(b.physical for b in (first, later))
    for batch in (first, later):
        empty = np.tile(np.array([0, 0xffffffff], np.uint32), (3, pages - batch.tables.shape[1], 1))
        batch.tables = np.concatenate([batch.tables, empty], 1)
        more = physical - batch.physical
        batch.codes = [np.concatenate([c, np.full((more, *c.shape[1:]), 0x7f, np.uint8)]) for c in batch.codes]
        batch.scales = np.concatenate([batch.scales, np.full((more, *batch.scales.shape[1:]), 247, np.uint8)])
        batch.physical = physical
        batch.upload(hip)
    commands = CommandList()
    op = Op.paged_quant_attention_ragged(0.09, 16, max(counts) == 1)
    held = first.inputs[3:]                                   # what both layers name
    commands.dispatch_many(op, first.inputs, [first.out, *first.cache])
    for index in (3, 6):
        commands.dispatch(Op.copy(), [later.inputs[index]], held[index - 3])
    commands.dispatch_many(op, later.inputs[:3] + held, [later.out, *later.cache])
    if static:
        hip.submit_static(commands)
    else:
        hip.submit(commands).wait()
    for batch in (first, later):
        want, bound = batch.expected(0.09)
        within(to_f32(hip.read(batch.out), DType.BF16).reshape(want.shape), want, bound)
        for tensor, array in zip(batch.cache, (*batch.codes, batch.scales)):
            assert np.array_equal(read_bytes(hip, tensor).reshape(array.shape), array)


@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 40, 3]])
def test_one_channel_that_dominates_the_scores(hip, width, counts):
    """Keys and queries with one channel hundreds of times as large as the others', which almost every key has alike: what tells
    keys apart is the rest.  A product of two codes is exact; summed by a scaled product of the matrix cores, terms end
    2^-11.9 of the sum of all sizes from the exact sum at worst (measured: 64 and 128 terms of sizes spread over 2^34, and one large one
    beside small ones, 2^-12 and 2^-12.7); the second pieces add terms of at most 2^-4 of the first ones' sizes, so that a score of bf16
    queries may be off by 2^-11.5 S where the other forms' are by 2^-14 S (see the head of this file)."""
    scale = 0.02

    def rows(rng):
        def make(what, shape):
            values = rng.standard_normal(shape) * 0.3
            if what != "v":
                values[..., 7] = 20.0 + rng.integers(-1, 2, shape[:-1])
            return values
        return make

    for dtype, sums in ((DType.BF16, 2.0 ** -11.5), (DType.F32, 0.0)):
        batch = Batch([70, 300, 600], counts, 8, 2, 16, width, dtype=dtype, make=rows(np.random.default_rng(101)), seed=101)
        got = batch.upload(hip).attend(hip, scale)
        want, bound = batch.expected(scale)
        for lane, (context, count) in enumerate(zip(batch.contexts, counts)):
            page, slot = batch.where(lane, np.arange(context + count))
            keys, values = (quant_cache.decode_rows(batch.codes[p][page, slot], batch.scales[page, p, :, slot]) for p in range(2))
            at = slice(batch.cu[lane], batch.cu[lane + 1])
            o, a, s = quant_cache.attend(batch.q[at].astype(np.float64), keys, values, float(np.float32(scale)), context + 1 + np.arange(count))
            assert s.min() > 6
            bound[at] += 2 * sums * s * a
        within(got, want, bound)


@pytest.mark.parametrize("width", [64, 128])
def test_decode_weights_hold_16_bits(hip, width):
    """Rows of bf16 with few keys, to f16: the bound of a decode batch with weights of 2^-16, and scores as the scaled products sum
    them (2^-11.5 S: see the test of a dominating channel; S is small here)."""
    batch = Batch([i % 7 for i in range(200)], [1] * 200, 8, 2, 16, width, out_dtype=DType.F16, seed=111)
    got = batch.upload(hip).attend(hip, 0.004)
    want, bound = batch.expected(0.004)
    for lane, context in enumerate(batch.contexts):
        page, slot = batch.where(lane, np.arange(context + 1))
        keys, values = (quant_cache.decode_rows(batch.codes[p][page, slot], batch.scales[page, p, :, slot]) for p in range(2))
        o, a, s = quant_cache.attend(batch.q[lane:lane + 1].astype(np.float64), keys, values, float(np.float32(0.004)), [context + 1])
        assert s.max() < 1
        bound[lane] = (HALF_STEP[DType.F16] * np.abs(o) + (2.0 ** -16 + 2 * (2.0 ** -11.5 * s + 2.0 ** -18 * s + 2.0 ** -21)
                                                         + (context / 4 + 64) * 2.0 ** -23) * a + 2.0 ** -25)[0]   # (f16's smallest step)
    within(got, want, bound)


@pytest.mark.parametrize("counts,activity,lead,behind", [([1, 700, 3, 40], [1, 0, 1, 1], 0, 900), ([1, 5, 1, 2], [1, 1, 0, 1], 70, 1200),
                                                         ([1, 1, 1, 1], [1, 1, 1, 0], 0, 300), ([600, 1, 300, 1], [0, 0, 0, 0], 5, 0)])
def test_padded_batches(hip, counts, activity, lead, behind):
    """Rows in front of the first lane, behind the last and of inactive lanes, more of them than the plan has threads: all read zero."""
    batch = Batch([40, 0, 700, 3], counts, 8, 2, 16, activity=activity, seed=121)
    shift = lambda a: np.concatenate([np.ones((lead, *a.shape[1:]), np.float32), a, np.ones((behind, *a.shape[1:]), np.float32)])  # noqa: E731
    batch.q, batch.k_new, batch.v_new = (shift(a) for a in (batch.q, batch.k_new, batch.v_new))
    batch.cu = batch.cu + lead
    got = batch.check(hip, 0.09)
    live = np.zeros(len(got), bool)
    for lane, active in enumerate(activity):
        live[batch.cu[lane]:batch.cu[lane + 1]] = active
    assert not got[~live].any() and got[live].any(axis=(1, 2)).all()
