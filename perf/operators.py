"""Workloads of the 8-bit row operators: the RMS norm that ends an encoder layer and writes 8-bit rows,
the product of 8-bit rows with an 8-bit projection, and the cache of 8-bit rows that token vectors are
written to and read back from.

An 8-bit row is a row of int8 values with one float32 scale (the cache: one scale for each group of the row,
such as a head); it stands for value * scale. With `own` false every operator is computed from elementary
torch operations in 32 bits; with `own` true by jhq_gpu_b200.
"""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
PAGE = 32                       # cache slots a page

# The largest work of one case: multiply-adds of a product, values of a norm or of a cache pass.
MOST_MACS = 32768 * 8192 * 8192
MOST_NORM = 65536 * 4096
MOST_CACHE = 65536 * 2048


def listed():
    return [
        # the last norm of one query token
        norm("norm_token", 1, 4096, "bfloat16", "same"),
        # a search batch of 256 embeddings of 1024 dimensions, no residual stream
        norm("norm_batch", 256, 1024, "float16", "none"),
        # rows that are slices of a wider float32 buffer, of no round width
        norm("norm_ragged", 4099, 1001, "float32", "same", pad=7),
        # the tokens of a large indexing batch, residual stream kept in float32
        norm("norm_index", 65536, 4096, "bfloat16", "float32"),
        # one token through a large square projection: the weights' bytes count
        matmul("matmul_token", 1, 8192, 8192, "bfloat16"),
        # a serving batch of 64 tokens through the same projection
        matmul("matmul_batch", 64, 8192, 8192, "bfloat16"),
        # packed rows of odd length, so that no row but the first starts on a boundary
        matmul("matmul_ragged", 1000, 999, 1001, "float32", bias=True, packed=True),
        # a large indexing batch: the multiply-adds count
        matmul("matmul_index", 32768, 8192, 8192, "bfloat16"),
        # a decoding step: one token's keys and values (8 heads each) written, 2048 tokens read back
        cache("cache_token", 1, 2048, 16, 128, "bfloat16"),
        # a prompt of 32768 tokens written behind as many older ones and all of them read back
        cache("cache_prompt", 32768, 65536, 16, 128, "bfloat16"),
        # a batch of 256 query tokens: norm, then the projection to 1024-dimensional embeddings
        embed("embed_query", 256, 1024, 4096, "bfloat16"),
        # the same head over an indexing batch of 65536 tokens
        embed("embed_index", 65536, 1024, 4096, "bfloat16"),
    ]


def norm(name, rows, dim, dtype, residual, pad=0):
    """residual: "none", "same" (the type of x) or "float32"."""
    return dict(name=name, op="norm", rows=rows, dim=dim, type=dtype, residual=residual, pad=pad)


def matmul(name, tokens, channels, depth, dtype, bias=False, packed=False):
    """packed: rows follow one another; else each begins at a multiple of 16 bytes."""
    return dict(name=name, op="matmul", tokens=tokens, channels=channels, depth=depth, type=dtype, bias=bias, packed=packed)


def cache(name, new, read, groups, dim, dtype):
    return dict(name=name, op="cache", new=new, read=read, groups=groups, dim=dim, type=dtype)


def embed(name, tokens, channels, depth, dtype):
    return dict(name=name, op="embed", tokens=tokens, channels=channels, depth=depth, type=dtype)


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _width(rng, low, high):
    """A width: half of them multiples of 80, the others odd."""
    n = _log(rng, low, high)
    return n | 1 if rng.random() < 0.5 or n < 80 else n // 80 * 80


def draw(rng):
    op = rng.choice(["norm", "norm", "matmul", "matmul", "matmul", "cache", "cache", "embed"])
    dtype = rng.choice(sorted(TYPES))
    while True:
        if op == "norm":
            c = norm("", _log(rng, 1, 65536), _width(rng, 16, 16384), dtype, rng.choice(["none", "same", "float32"]), rng.choice([0, 0, rng.randint(1, 40)]))
            cost, most = c["rows"] * c["dim"], MOST_NORM
        elif op == "matmul":
            c = matmul("", _log(rng, 1, 32768), _width(rng, 16, 16384), _width(rng, 16, 16384), dtype, rng.random() < 0.5, rng.random() < 0.3)
            cost, most = c["tokens"] * c["channels"] * c["depth"], MOST_MACS
        elif op == "cache":
            new = _log(rng, 1, 32768)
            c = cache("", new, new + _log(rng, 1, 32768), rng.randint(1, 32), _width(rng, 16, 1024), dtype)
            cost, most = c["read"] * c["groups"] * c["dim"], MOST_CACHE
        else:
            c = embed("", _log(rng, 1, 65536), _width(rng, 64, 4096), _width(rng, 64, 8192), dtype)
            cost, most = c["tokens"] * c["depth"] * max(c["channels"], 1024), 65536 * 4096 * 1024
        if cost <= most:
            del c["name"]
            return c


# ---- inputs ---------------------------------------------------------------------------------------------

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rows(values, pad, dtype):
    """`values` as rows of a buffer that is `pad` wider."""
    n, d = values.shape
    buf = torch.zeros(n, d + pad, dtype=dtype, device="cuda")
    buf[:, :d] = values
    return buf[:, :d]


def _hidden(g, rows, dim):
    """Hidden states: normal, a few channels an order of magnitude larger, about one row in 50 all zero."""
    x = _normal(g, rows, dim)
    x *= 1 + 9 * (torch.rand(dim, generator=g, device="cuda") < 0.01)
    return x * (torch.rand(rows, 1, generator=g, device="cuda") >= 0.02)


def _bytes_buffer(rows, dim, packed=False):
    return torch.empty(rows, dim if packed else -(-dim // 16) * 16, dtype=torch.int8, device="cuda")[:, :dim]


def _q8_rows(g, rows, dim, spread, packed=False):
    q = _bytes_buffer(rows, dim, packed)
    for i in range(0, rows, 8192):
        n = min(8192, rows - i)
        q[i:i + n] = (_normal(g, n, dim) * spread).round().clamp(-127, 127).to(torch.int8)
    return q, torch.rand(rows, generator=g, device="cuda") * 0.02 + 0.002


def _slots(g, tokens):
    """Cache slots of a sequence: whole pages anywhere in a cache twice as large, one entry in 32 padding (-1)."""
    pages = -(-tokens // PAGE)
    at = torch.randperm(2 * pages, generator=g, device="cuda")[:pages]
    slots = (at[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)[:tokens]
    return torch.where(torch.rand(tokens, generator=g, device="cuda") < 1 / 32, -1, slots), 2 * pages * PAGE


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    s = dict(op=case["op"], dtype=dtype)
    if case["op"] in ("norm", "embed"):
        rows, dim = (case["rows"], case["dim"]) if case["op"] == "norm" else (case["tokens"], case["depth"])
        kind, pad = case.get("residual", "same"), case.get("pad", 0)
        s["x"] = _rows(_hidden(g, rows, dim), pad, dtype)
        s["weight"] = (1 + 0.2 * _normal(g, dim)).to(dtype)
        s["residual"] = s["residual_out"] = None
        if kind != "none":
            s["residual"] = _rows(_hidden(g, rows, dim), pad, dtype if kind == "same" else torch.float32)
            s["residual_out"] = torch.empty_like(s["residual"], memory_format=torch.contiguous_format)
        s["q"], s["scale"] = _bytes_buffer(rows, dim), torch.empty(rows, device="cuda")
        if case["op"] == "norm":
            s["out"] = torch.empty(rows, dim, dtype=dtype, device="cuda")
        else:
            s["w"], s["w_scale"] = _q8_rows(g, case["channels"], dim, 40.0)
            s["bias"], s["out"] = None, torch.empty(rows, case["channels"], device="cuda")
    elif case["op"] == "matmul":
        s["q"], s["scale"] = _q8_rows(g, case["tokens"], case["depth"], 30.0, case["packed"])
        s["w"], s["w_scale"] = _q8_rows(g, case["channels"], case["depth"], 40.0, case["packed"])
        s["bias"] = _normal(g, case["channels"]) if case["bias"] else None
        s["out"] = torch.empty(case["tokens"], case["channels"], dtype=dtype, device="cuda")
    else:
        groups, dim = case["groups"], case["dim"]
        s["groups"], s["dim"] = groups, dim
        s["slots"], room = _slots(g, case["read"])
        s["new_slots"] = s["slots"][case["read"] - case["new"]:]
        s["x"] = _hidden(g, case["new"], groups * dim).to(dtype)
        s["q"], _ = _q8_rows(g, room, groups * dim, 40.0)
        s["scale"] = torch.rand(room, groups, generator=g, device="cuda") * 0.02 + 0.002
        s["out"] = torch.empty(case["read"], groups * dim, dtype=dtype, device="cuda")
    return s


# ---- the operators --------------------------------------------------------------------------------------

def _quantise(y):
    """Whole numbers in -127 .. 127 and the largest magnitude of each row (last axis) of float32 `y`."""
    top = y.abs().amax(-1, keepdim=True)
    return torch.round(y * torch.where(top > 0, 127 / top, 0)), top


def _norm_plain(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
        s["residual_out"].copy_(h)
    q, top = _quantise(h * s["weight"].float())
    return q, top * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) / 127


def _matmul_plain(q, scale, s):
    y = (q @ s["w"].float().T) * scale * s["w_scale"]
    return (y if s["bias"] is None else y + s["bias"]).to(s["out"].dtype)


def _cache_plain(s):
    x = s["x"].float().view(-1, s["groups"], s["dim"])
    q, top = _quantise(x)
    kept = s["new_slots"] >= 0
    to = s["new_slots"][kept]
    s["q"][to] = q.view(len(x), -1)[kept].to(torch.int8)
    s["scale"][to] = (top / 127)[kept, :, 0]
    at = s["slots"].clamp(min=0)
    back = s["q"][at].float().view(-1, s["groups"], s["dim"]) * s["scale"][at][:, :, None]
    return torch.where(s["slots"][:, None] >= 0, back.view(len(at), -1), 0).to(s["dtype"])


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "norm":
        q, step = _norm_plain(s)
        return dict(values=(q * step).to(s["dtype"]), residual=s["residual_out"])
    if s["op"] == "matmul":
        return dict(out=_matmul_plain(s["q"].float(), s["scale"][:, None], s))
    if s["op"] == "embed":
        q, step = _norm_plain(s)
        return dict(out=_matmul_plain(q, step, s), residual=s["residual_out"])
    return dict(values=_cache_plain(s))


def _run_own(s):
    import jhq_gpu_b200 as J
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "cache":
        rows = J.Q8Rows.of(s["q"], s["scale"], groups=s["groups"])
        J.q8_write(J.View.of(s["x"]), rows, slots=s["new_slots"].data_ptr(), stream=stream)
        J.q8_read(rows, J.View.of(s["out"]), slots=s["slots"].data_ptr(), stream=stream)
        return dict(values=s["out"])
    rows, out = J.Q8Rows.of(s["q"], s["scale"]), J.View.of(s["out"])
    if s["op"] in ("norm", "embed"):
        residual = residual_out = None
        if s["residual"] is not None:
            residual, residual_out = J.View.of(s["residual"]), J.View.of(s["residual_out"])
        J.q8_rms_norm(J.View.of(s["x"]), rows, weight=J.View.of(s["weight"]), residual=residual, residual_out=residual_out, eps=EPS, stream=stream)
        if s["op"] == "norm":
            J.q8_read(rows, out, stream=stream)
            return dict(values=s["out"], residual=s["residual_out"])
    bias = None if s["bias"] is None else J.View.of(s["bias"])
    J.q8_matmul(rows, J.Q8Rows.of(s["w"], s["w_scale"]), out, bias=bias, stream=stream)
    return dict(out=s["out"], residual=s["residual_out"]) if s["op"] == "embed" else dict(out=s["out"])


# ---- what a pass cannot do without, and what it returns in 64 bits -------------------------------------------

def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "cache":
        new, read = case["new"], case["read"]
        values, scales = case["groups"] * case["dim"], 4 * case["groups"]
        return dict(bytes=new * (values * (size + 1) + scales + 8) + read * (values * (1 + size) + scales + 8),
                    flops=3 * new * values + read * values)
    nbytes = flops = 0
    if case["op"] in ("norm", "embed"):
        rows, dim = (case["rows"], case["dim"]) if case["op"] == "norm" else (case["tokens"], case["depth"])
        wide = {"none": 0, "same": size, "float32": 4}[case.get("residual", "same")]
        nbytes += rows * dim * (size + 2 * wide + 1) + 4 * rows + dim * size
        flops += 6 * rows * dim
        if case["op"] == "norm":                                       # the rows read back
            nbytes += rows * dim * (1 + size) + 4 * rows
    if case["op"] in ("matmul", "embed"):
        t, n, k = case["tokens"], case["channels"], case["depth"]
        out = 4 if case["op"] == "embed" else size
        nbytes += (t + n) * (k + 4) + t * n * out + (4 * n if case.get("bias") else 0)
        flops += 2 * t * n * k
    return dict(bytes=nbytes, flops=flops)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "cache":
        groups, dim = s["groups"], s["dim"]
        q, scale = s["q"].clone(), s["scale"].double()
        for i in range(0, case["new"], 4096):
            x = s["x"][i:i + 4096].double().view(-1, groups, dim)
            to = s["new_slots"][i:i + 4096]
            step = x.abs().amax(2) / 127
            whole = torch.round(x / torch.where(step > 0, step, 1)[:, :, None]).view(len(to), -1).to(torch.int8)
            q[to[to >= 0]], scale[to[to >= 0]] = whole[to >= 0], step[to >= 0]
        out = torch.zeros(case["read"], groups * dim, dtype=torch.float64, device="cuda")
        for i in range(0, case["read"], 4096):
            at = s["slots"][i:i + 4096]
            there = (at >= 0).nonzero()[:, 0]
            v = q[at[there]].double().view(-1, groups, dim) * scale[at[there]][:, :, None]
            out[i + there] = v.view(len(there), -1)
        return dict(values=out)
    got = {}
    if s["op"] in ("norm", "embed"):
        n = len(s["x"])
        got["residual"] = None
        if s["residual"] is not None:
            got["residual"] = torch.empty(s["residual_out"].shape, dtype=torch.float64, device="cuda")
        values = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
        for i in range(0, n, 8192):
            h = s["x"][i:i + 8192].double()
            if s["residual"] is not None:
                h += s["residual"][i:i + 8192].double()
                got["residual"][i:i + 8192] = h
            y = h / (h.square().mean(1, keepdim=True) + EPS).sqrt() * s["weight"].double()
            step = y.abs().amax(1, keepdim=True) / 127
            values[i:i + 8192] = torch.round(y / torch.where(step > 0, step, 1)) * step
        if s["op"] == "norm":
            return dict(values=values, **got)
        left = values
    else:
        left = s["q"].double() * s["scale"].double()[:, None]
    got["out"] = left @ (s["w"].double() * s["w_scale"].double()[:, None]).T
    if s["bias"] is not None:
        got["out"] += s["bias"].double()
    return got
