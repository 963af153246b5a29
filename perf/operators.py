"""Cases for timing the operators of the paged key/value cache that is held in 8 bits: storing rows into its
pages and reading them back (`Op.paged_quant_copy`), and the ragged attention of a packed batch that stores the
batch's new rows and attends through them (`Op.paged_quant_attention_ragged`), each through `Backend.submit`.

The cache holds a row (one token, one kv head) as e4m3 codes c_i with one scale 2^e of its own:

    e    = the smallest whole number with max_i |x_i| <= 448 * 2^e, at least -126
    c_i  = x_i / 2^e rounded to e4m3, ties to even;  the row stands for c_i * 2^e

Four codes are a u32 word, a scale is the byte e + 127: codes [pages, page_tokens, kv heads, dim / 4], scales
[pages, 2 (keys, values), kv heads, page_tokens / 4].  A case is a plain dict.  `kind` "write" and "read" move
`rows` rows of one sequence from position `start` on; "attend" is one layer's attention of a packed batch:

  q_heads, kv_heads, dim   head layout; `dtype` that of queries, new rows and output; `page_tokens` the page size
  lanes, ctx_lo, ctx_hi    decode rows, one per sequence, with cached contexts spread log-uniformly
  rows, chunks, prefix     prompt rows, the ragged chunks they are cut into, cached tokens in front of each

Head layouts are those of the shapes in forja_amd/model.py (16 query heads on 8, 32 on 4, 40 on 8, of 128), with
generic ones among the drawn cases.
"""
import collections
import math

import numpy as np
import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IN_FLIGHT = 4      # submissions a program has enqueued before it waits for the oldest


def _copy(name, kind, rows, start, kv_heads, dim, dtype, page_tokens=16):
    return {"name": name, "kind": kind, "rows": rows, "start": start, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page_tokens": page_tokens}


def _attend(name, q_heads, kv_heads, dtype, lanes, ctx_lo, ctx_hi, rows=0, chunks=0, prefix=0, dim=128, page_tokens=16):
    return {"name": name, "kind": "attend", "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page_tokens": page_tokens, "lanes": lanes, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "rows": rows, "chunks": chunks,
            "prefix": prefix}


def listed():
    return [
        # One new token of one sequence is stored: the time of a call.
        _copy("write_1", "write", 1, 400, 8, 128, "bf16"),
        # A long prompt's keys go into the cache at once.
        _copy("write_32749", "write", 32749, 0, 8, 128, "bf16"),
        # A shared prefix is taken out of the cache, from the middle of a page on.
        _copy("read_700", "read", 700, 21, 8, 128, "bf16"),
        # A sequence of the mixture model's engine leaves the device in that engine's f32.
        _copy("read_16384", "read", 16384, 0, 4, 128, "f32"),
        # One user chats with the small model: latency.
        _attend("chat_1", 16, 8, "bf16", 1, 400, 400),
        # One coding assistant far into a long context: one sequence has to fill the device.
        _attend("long_1", 32, 4, "bf16", 1, 30011, 30011),
        # The engine's own dtypes, the most lanes that it batches.
        _attend("engine_8", 32, 4, "f32", 8, 256, 32768),
        # A decode batch of the dense model.
        _attend("dense_48", 40, 8, "bf16", 48, 128, 4096),
        # The headline batch: 128 lanes of very different contexts.
        _attend("coder_128", 32, 4, "bf16", 128, 256, 32768),
        # A prompt of 512 tokens from scratch in the engine's dtypes.
        _attend("engine_prompt_512", 32, 4, "f32", 0, 1, 1, 512, 1, 0),
        # Continued prompts of a mixture model beside a decode batch.
        _attend("coder_prompt_2048", 32, 4, "bf16", 32, 256, 8192, 2048, 3, 1024),
        # A full prefill chunk of the dense model with its decode rows.
        _attend("dense_prefill_8256", 40, 8, "bf16", 64, 128, 4096, 8192, 6, 0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "decode", "prompt", "prompt"])
    pages = rng.choice([16, 16, 32, 64])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    dim = rng.choice([128, 128, 128, 64])
    if kind in ("write", "read"):
        case = _copy("", kind, _log_uniform(rng, 1, 32768), _log_uniform(rng, 1, 5000) - 1, rng.choice([1, 2, 4, 8]), dim,
                     dtype, pages)
    else:
        q_heads, kv_heads = rng.choice([(16, 8), (32, 4), (32, 4), (40, 8), (8, 8), (12, 1)])
        ctx_lo = _log_uniform(rng, 1, 1000)
        ctx_hi = _log_uniform(rng, ctx_lo, 8192 if kv_heads == 8 or kind == "prompt" else 32768)
        if kind == "decode":
            case = _attend("", q_heads, kv_heads, dtype, _log_uniform(rng, 1, 128), ctx_lo, ctx_hi, dim=dim,
                           page_tokens=pages)
        else:
            rows = _log_uniform(rng, 24, 2000 if dtype == "f32" else 6000)
            case = _attend("", q_heads, kv_heads, dtype, rng.randint(0, 64), ctx_lo, ctx_hi, rows,
                           rng.randint(1, min(6, rows // 12)), rng.choice([0, 0, _log_uniform(rng, 1, 8000)]), dim, pages)
    del case["name"]
    return case


def _batch(case):
    """Cached tokens and new rows of every lane of an "attend" case: decode lanes, then prompt chunks, whose lengths
    go in proportion 2 : 3 : 4 : .., the last taking the rest."""
    n, chunks, rows = case["lanes"], case["chunks"], case["rows"]
    lo, hi = math.log(case["ctx_lo"]), math.log(case["ctx_hi"])
    contexts = [int(round(math.exp(lo + (hi - lo) * (i * 37 % n + 0.5) / n))) for i in range(n)] if math.gcd(37, n) == 1 else \
        [int(round(math.exp(lo + (hi - lo) * (i + 0.5) / n))) for i in range(n)]
    counts = [1] * n
    if chunks:
        total = sum(range(2, chunks + 2))
        parts = [max(1, rows * (i + 2) // total) for i in range(chunks - 1)]
        counts += parts + [rows - sum(parts)]
        contexts += [case["prefix"]] * chunks
    return contexts, counts


# ---------------------------------------------------------------- inputs, the same on both sides

def _e4m3(rows):
    """Rows [.., dim] as (codes u8, scale bytes u8) of the cache's format."""
    x = rows.float()
    most = x.abs().amax(-1, keepdim=True)
    fraction, exponent = torch.frexp(most)                 # most = fraction * 2^exponent, 1/2 <= fraction < 1
    e = (exponent - 9 + (fraction > 0.875).int()).clamp(min=-126)     # 448 = 0.875 * 2^9
    e = torch.where(most == 0, torch.full_like(e, -126), e)
    codes = (x * _power(-e)).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, (e + 127).to(torch.uint8).squeeze(-1)


def _power(e):
    """2^e in f32, e from -126 to 127."""
    return ((e + 127) << 23).view(torch.float32)


def _randn(generator, *shape):
    return torch.randn(shape, generator=generator, device="cuda")


def _gains(generator, heads, dim):
    """Sizes of a head's channels: most alike, a few several times larger, as trained keys have them."""
    gains = torch.exp(0.3 * _randn(generator, heads, dim))
    return torch.where(torch.rand((heads, dim), generator=generator, device="cuda") < 0.03, gains * 4.0, gains)


def _rows(generator, rows, heads, dim, dtype, gains):
    return (_randn(generator, rows, heads, dim) * gains).to(dtype)


class _State:
    pass


def _inputs(case, seed):
    """Everything a pass needs, as torch tensors: the cache with its tables, and the batch."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = _State()
    s.kind, pt, heads, dim = case["kind"], case["page_tokens"], case["kv_heads"], case["dim"]
    s.page_tokens, dtype = pt, TORCH[case["dtype"]]
    if s.kind == "attend":
        s.contexts, s.counts = _batch(case)
    else:
        s.contexts, s.counts = [case["start"]], [case["rows"]]
    pages = [-(-(c + n) // pt) for c, n in zip(s.contexts, s.counts)]
    total, most = sum(pages) + 8, max(pages) + 1
    order = torch.randperm(total, generator=g, device="cuda")
    s.generations = torch.arange(11, 11 + total, device="cuda")
    s.tables = torch.zeros((len(pages), most, 2), dtype=torch.int64, device="cuda")
    s.tables[:, :, 1] = 0xffffffff
    at = 0
    for lane, n in enumerate(pages):
        s.tables[lane, :n, 0] = order[at:at + n]
        s.tables[lane, :n, 1] = s.generations[order[at:at + n]]
        at += n
    gains = _gains(g, heads, dim)
    planes = [gains, torch.ones_like(gains)] if s.kind == "attend" else [gains]
    s.codes, scales = [], []
    for plane in planes:
        codes, bytes_ = _e4m3(_rows(g, total * pt, heads, dim, torch.bfloat16, plane))
        s.codes.append(codes.view(total, pt, heads, dim))
        scales.append(bytes_.view(total, pt, heads).transpose(1, 2))
    s.scales = torch.stack(scales, 1).contiguous()            # [pages, planes, heads, page_tokens]
    rows = sum(s.counts)
    if s.kind == "read":
        s.out = torch.zeros((rows, heads, dim), dtype=dtype, device="cuda")
    else:
        s.new = [_rows(g, rows, heads, dim, dtype, plane) for plane in planes]
    if s.kind == "attend":
        group = case["q_heads"] // heads
        # a query asks for channels as its head's keys have them; scores of a few units
        s.q = (_randn(g, rows, case["q_heads"], dim) * 1.5 / gains.repeat_interleave(group, 0)).to(dtype)
        s.scale = 1.0 / math.sqrt(dim)
        s.out = torch.zeros((rows, case["q_heads"], dim), dtype=dtype, device="cuda")
        s.cu = np.concatenate([[0], np.cumsum(s.counts)])
    # where the batch's rows go: page and slot of each
    lanes = torch.repeat_interleave(torch.arange(len(s.counts), device="cuda"), torch.tensor(s.counts, device="cuda"))
    first = torch.tensor(np.concatenate([[0], np.cumsum(s.counts)])[:-1], device="cuda")
    s.starts = torch.tensor(s.contexts, device="cuda")
    position = s.starts[lanes] + torch.arange(rows, device="cuda") - first[lanes]
    s.position = position
    s.page, s.slot = s.tables[lanes, position // pt, 0], position % pt
    return s


# ---------------------------------------------------------------- the framework's side

_backend = None
_submitted = collections.deque()


def _the_backend():
    """One backend for the process, as a serving host has."""
    global _backend
    if _backend is None:
        from forja_amd.hip_backend import HipBackend
        _backend = HipBackend(0)
    return _backend


class _Buffer:
    """A tensor of the framework and the memory under it, as torch takes it; released with the last tensor over it."""

    def __init__(self, backend, dtype, shape):
        self.backend, self.tensor = backend, backend.alloc(dtype, tuple(shape))
        bytes_ = self.tensor.layout.buffer_len
        self.__cuda_array_interface__ = {"shape": (bytes_,), "typestr": "|u1", "strides": None, "version": 2,
                                         "data": (backend.device_address(self.tensor), False)}

    def __del__(self):
        if self.backend._handle is not None:
            self.backend.release(self.tensor)


class _Device:
    """The state in the framework's tensors, and the recorded command list.  torch's own stream here is the null stream, which
    comes after what the backend has been given, and before what it is given next."""

    def __init__(self, case, s):
        from forja_amd.core import INTO_PAGES, OUT_OF_PAGES, CommandList, DType, Op
        self.backend, self.buffers, self.kind = _the_backend(), [], s.kind
        dtype = {"bf16": DType.BF16, "f16": DType.F16, "f32": DType.F32}[case["dtype"]]
        planes, (total, pt, heads, dim) = len(s.codes), s.codes[0].shape
        u32 = lambda t: self._put(DType.U32, t.shape, t.to(torch.int32))[0]  # noqa: E731
        words = lambda t: self._put(DType.U32, (*t.shape[:-1], t.shape[-1] // 4), t)  # noqa: E731
        floats = lambda t: self._put(dtype, t.shape, t)  # noqa: E731
        pools, codes = words(torch.cat(s.codes))
        pools = [pools.narrow(0, plane * total, total) for plane in range(planes)]
        all_scales, scales = words(s.scales)
        plane_scales = [all_scales.reshape((total, planes * heads, pt // 4)).narrow(1, plane * heads, heads) for plane in range(planes)]
        # where the pass's rows lie, [plane, row, head]: the row's codes, and its scale
        plane = torch.arange(planes, device="cuda")[:, None]
        self.codes, self.scales = codes.view(-1, heads, dim), scales.view(-1)
        self.rows = ((plane * total + s.page) * pt + s.slot).flatten()
        self.places = ((((s.page * planes + plane) * heads)[..., None] + torch.arange(heads, device="cuda")) * pt + s.slot[:, None]).flatten()
        self.shape = planes, len(s.page), heads, dim
        generations = u32(s.generations)
        commands = CommandList()
        if s.kind == "attend":
            tables, cu, starts = u32(s.tables), u32(torch.from_numpy(s.cu)), u32(s.starts)
            out, self.out = floats(s.out)
            commands.dispatch_many(
                Op.paged_quant_attention_ragged(s.scale, pt, one_row_per_lane=case["rows"] == 0),
                [floats(s.q)[0], *(floats(t)[0] for t in s.new), tables, generations, cu, starts], [out, *pools, all_scales])
            # what the stored rows stand for: of few sequences as the framework reads them back, a dispatch a sequence and plane
            self.read_back = len(s.counts) <= 8
            if self.read_back:
                rows, self.stored = self._put(DType.F32, self.shape, torch.zeros(self.shape, device="cuda"))
                for plane in range(planes):
                    for lane, (context, count) in enumerate(zip(s.contexts, s.counts)):
                        commands.dispatch_many(
                            Op.paged_quant_copy(OUT_OF_PAGES, context, pt),
                            [pools[plane], plane_scales[plane], tables.narrow(0, lane, 1).reshape(tables.shape[1:]), generations],
                            [rows.narrow(0, plane, 1).reshape(self.shape[1:]).narrow(0, int(s.cu[lane]), count)])
        else:
            table = u32(s.tables[0])
            if s.kind == "write":
                commands.dispatch_many(Op.paged_quant_copy(INTO_PAGES, case["start"], pt),
                                       [floats(s.new[0])[0], table, generations], [pools[0], plane_scales[0]])
                out, self.out = self._put(DType.F32, self.shape[1:], torch.zeros(self.shape[1:], device="cuda"))
            else:
                out, self.out = floats(s.out)
            commands.dispatch_many(Op.paged_quant_copy(OUT_OF_PAGES, case["start"], pt),
                                   [pools[0], plane_scales[0], table, generations], [out])
        self.encoded = self.backend.encode(commands)

    def _put(self, dtype, shape, values):
        """The framework's tensor of `values`, and torch's over the same memory."""
        buffer = _Buffer(self.backend, dtype, shape)
        self.buffers.append(buffer)
        held = torch.as_tensor(buffer, device="cuda").view(values.dtype).view(values.shape)
        held.copy_(values)
        return buffer.tensor, held

    def run(self):
        """One pass, and its outputs whole: the output rows where the framework has put them, and what the rows that it has
        stored stand for."""
        _submitted.append(self.backend.submit(self.encoded))
        if len(_submitted) > IN_FLIGHT:
            _submitted.popleft().wait()
        if self.kind == "read":
            return {"out": self.out}
        if self.kind == "attend" and self.read_back:
            return {"out": self.out, "keys": self.stored[0], "values": self.stored[1]}
        exponents = self.scales.index_select(0, self.places).int()
        if self.kind == "write":
            return {"rows": self.out, "exponents": exponents.sub_(127).view(self.shape[1:3])}
        rows = self.codes.index_select(0, self.rows).view(torch.float8_e4m3fn).float().view(self.shape)
        rows *= (exponents << 23).view(torch.float32).view(*self.shape[:3], 1)
        return {"out": self.out, "keys": rows[0], "values": rows[1]}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s.device = _Device(case, s)
        for name in ("codes", "scales", "new", "q", "out", "tables", "generations"):
            s.__dict__.pop(name, None)
    return s


# ---------------------------------------------------------------- one pass

class _Outputs(dict):
    """The pass's outputs: buffers of the state.  Looking one up reads it (a program that goes on with the next layer on
    the device reads none): the output rows, and of the cache what the rows that the pass has stored stand for."""

    def __init__(self, s):
        names = {"read": ["out"], "write": ["rows", "exponents"], "attend": ["out", "keys", "values"]}[s.kind]
        super().__init__((name, None) for name in names)
        self.s = s

    def __getitem__(self, name):
        s = self.s
        if name == "out":
            return s.device.read(s.device.out, s.dtype).view(s.shapes[2]) if hasattr(s, "device") else s.out
        plane = 1 if name == "values" else 0
        if hasattr(s, "device"):
            codes = s.device.read(s.device.codes[plane], torch.uint8).view(s.shapes[0][plane])
            scales, page, slot = s.device.read(s.device.scales, torch.uint8).view(s.shapes[1]), s.host["page"], s.host["slot"]
        else:
            codes, scales, page, slot = s.codes[plane], s.scales, s.page, s.slot
        exponents = scales[page, plane, :, slot].int() - 127
        return exponents if name == "exponents" else _decoded(codes[page, slot], exponents)


def _decoded(codes, exponents):
    return codes.contiguous().view(torch.float8_e4m3fn).float() * _power(exponents[..., None])


def _store(s):
    """The batch's rows into the cache."""
    for plane, rows in enumerate(s.new):
        codes, bytes_ = _e4m3(rows)
        s.codes[plane][s.page, s.slot] = codes
        s.scales[s.page, plane, :, s.slot] = bytes_


def _attend_lanes(s, lanes, row0, rows):
    """Causal attention of `lanes` (a range) of the batch, padded to the longest: `rows` new rows at most, from packed
    row row0 of each."""
    longest = max(s.contexts[lane] + s.counts[lane] for lane in lanes)
    pages = -(-longest // s.page_tokens)
    index = torch.tensor(list(lanes), device="cuda")
    page = s.tables[index, :pages, 0]
    kv = []
    for plane in range(2):
        exponents = s.scales[page, plane].int() - 127                        # [lanes, pages, heads, page_tokens]
        values = _decoded(s.codes[plane][page], exponents.transpose(2, 3))   # [lanes, pages, page_tokens, heads, dim]
        kv.append(values.flatten(1, 2).permute(0, 2, 1, 3).contiguous())     # [lanes, heads, keys, dim]
    heads, dim = kv[0].shape[1], kv[0].shape[3]
    first = torch.tensor([row0[lane] for lane in lanes], device="cuda")
    count = torch.tensor([s.counts[lane] for lane in lanes], device="cuda")
    step = torch.arange(rows, device="cuda")
    packed = first[:, None] + torch.minimum(step, count[:, None] - 1)        # [lanes, rows]
    q = s.q[packed].float()                                                  # [lanes, rows, q heads, dim]
    group = q.shape[2] // heads
    q = q.view(len(lanes), rows, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(len(lanes), heads, rows * group, dim)
    scores = torch.matmul(q, kv[0].transpose(2, 3)) * s.scale                # [lanes, heads, rows * group, keys]
    limit = s.position[packed].repeat_interleave(group, 1)                   # the last key that a row attends
    key = torch.arange(scores.shape[3], device="cuda")
    scores.masked_fill_(key > limit[:, None, :, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(weights, kv[1]) / weights.sum(-1, keepdim=True)
    out = out.view(len(lanes), heads, rows, group, dim).permute(0, 2, 1, 3, 4).reshape(len(lanes), rows, heads * group, dim)
    live = step < count[:, None]
    s.out[packed[live]] = out[live].to(s.out.dtype)


def run(state):
    s = state
    if own:
        return s.device.run()
    elif s.kind == "read":
        s.out.copy_(_decoded(s.codes[0][s.page, s.slot], s.scales[s.page, 0, :, s.slot].int() - 127))
    else:
        _store(s)
        if s.kind == "attend":
            single = sum(n == 1 for n in s.counts)          # decode lanes come first
            if single:
                _attend_lanes(s, range(single), s.cu, 1)
            if single < len(s.counts):
                _attend_lanes(s, range(single, len(s.counts)), s.cu, max(s.counts[single:]))
    return _Outputs(s)


def work(case):
    size, heads, dim = TORCH[case["dtype"]].itemsize, case["kv_heads"], case["dim"]
    if case["kind"] != "attend":
        elements = case["rows"] * heads * dim
        return {"bytes": elements * (size + 1) + case["rows"] * heads, "flops": 2.0 * elements}
    contexts, counts = _batch(case)
    rows, q_heads = sum(counts), case["q_heads"]
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(contexts, counts))
    cached, new = sum(contexts), rows
    return {"bytes": (cached + new) * 2 * heads * (dim + 1) + new * 2 * heads * dim * size + 2 * rows * q_heads * dim * size,
            "flops": 4.0 * q_heads * dim * pairs}


# ---------------------------------------------------------------- the definition, in 64 bits

def _nearest(rows):
    """The format by its definition: the nearest of the 253 values, ties to the even code; (values, exponents)."""
    x = rows.double()
    most = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(most.clamp(min=2.0 ** -200) / 448.0))
    e = torch.where(most > 448.0 * torch.exp2(e), e + 1, e)               # log2 next to a whole number
    e = torch.where(most <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
    table = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (k - 7) for k in range(1, 16) for m in range(8)]
    table = torch.tensor(table[:127], dtype=torch.float64, device=x.device)
    y = (x / torch.exp2(e)).contiguous()
    between = (table[1:] + table[:-1]) / 2
    below, above = torch.searchsorted(between, y.abs()), torch.searchsorted(between, y.abs(), right=True)
    code = torch.where(below % 2 == 0, below, above)                      # equal but on a tie
    return torch.copysign(table[code] * torch.exp2(e), y), e.squeeze(-1)


def exact(case, seed):
    s = _inputs(case, seed)
    if s.kind == "read":
        codes = s.codes[0][s.page, s.slot].view(torch.float8_e4m3fn).double()
        return {"out": codes * torch.exp2(s.scales[s.page, 0, :, s.slot].double() - 127)[..., None]}
    stored = [_nearest(rows) for rows in s.new]
    if s.kind == "write":
        return {"rows": stored[0][0], "exponents": stored[0][1].int()}
    out = torch.zeros(s.out.shape, dtype=torch.float64, device="cuda")
    group = case["q_heads"] // case["kv_heads"]
    for lane, (context, count) in enumerate(zip(s.contexts, s.counts)):
        at = int(s.cu[lane])
        token = torch.arange(context, device="cuda")
        page, slot = s.tables[lane, token // s.page_tokens, 0], token % s.page_tokens
        limit = context + torch.arange(count, device="cuda")
        hidden = torch.arange(context + count, device="cuda") > limit[:, None]
        for head in range(case["kv_heads"]):
            kv = []
            for plane in range(2):
                cached = s.codes[plane][page, slot, head].view(torch.float8_e4m3fn).double()
                cached = cached * torch.exp2(s.scales[page, plane, head, slot].double() - 127)[:, None]
                kv.append(torch.cat([cached, stored[plane][0][at:at + count, head]]))
            for query in range(head * group, (head + 1) * group):
                scores = s.q[at:at + count, query].double() @ kv[0].T * s.scale
                scores = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
                out[at:at + count, query] = scores @ kv[1]
    return {"out": out, "keys": stored[0][0], "values": stored[1][0]}
