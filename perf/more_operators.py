"""Measured cases of the operators that serve a transformer's layer over microscaled 4-bit rows.

  write     new tokens' keys and values into a cache of microscaled rows (mi355x_mx4_cache_write),
            and the cache's values read back
  attend    attention over such a cache, prompts and single tokens, with a sliding window and a
            few first tokens that stay visible (mi355x_mx4_attention)
  adapters  a FullyConnected over microscaled weights with a low-rank adapter of each row's own
            beside it (mi355x_mx4_fc_adapters)

A microscaled row of `cols` values is P = ceil(cols / 128) times 64 bytes of codes (E2M1, two
to a byte, the even column in the low half), P times 4 scale bytes (E8M0, one for each 32
columns) and zeros up to a multiple of 16 bytes; what is past `cols` is zero. A cache holds a
row of kv_heads * dim columns for each token, in pages of as many tokens; a sequence's pages
stand in a table, or follow each other where there is none.

`own` chooses between the plain form, elementary torch operations in 32 bits, and the
library's calls. Both work on the same state.
"""
import functools

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2, "mx4": 3}
MOST_TOKENS = 4 * 131072         # in a cache
MOST_VALUES = MOST_TOKENS * 1024
MOST_FLOPS = 2 * 4096 * (4096 * 4096 + 64 * 8192)
EPSILON = 1e-30


def listed():
    return [
        # The first answer of a small model to one request: the call itself.
        dict(name="attend_one", op="attend", sequences=1, longest=200, shortest=200, new=1, pad=0, heads=8, kv_heads=2,
             dim=64, page=0, window=0, sinks=0, type="f16"),
        # A batch of conversations of all lengths, a token each, in a padded batch.
        dict(name="attend_step", op="attend", sequences=61, longest=4096, shortest=1, new=1, pad=3, heads=32, kv_heads=8,
             dim=128, page=16, window=0, sinks=0, type="bf16"),
        # A few very long documents: bound by the cache.
        dict(name="attend_long", op="attend", sequences=4, longest=131072, shortest=100003, new=1, pad=0, heads=32,
             kv_heads=8, dim=128, page=64, window=0, sinks=0, type="f16"),
        # Conversations that see their last 4096 tokens and the first four.
        dict(name="attend_window", op="attend", sequences=64, longest=8191, shortest=100, new=1, pad=0, heads=32, kv_heads=8,
             dim=128, page=32, window=4096, sinks=4, type="bf16"),
        # Two prompts from their first token: bound by the matrix cores.
        dict(name="attend_prompt", op="attend", sequences=2, longest=4096, shortest=4096, new=4096, pad=0, heads=32,
             kv_heads=8, dim=128, page=64, window=0, sinks=0, type="bf16"),
        # A long prompt through a window.
        dict(name="attend_prompt_window", op="attend", sequences=1, longest=16384, shortest=16384, new=16384, pad=0,
             heads=32, kv_heads=8, dim=128, page=128, window=1024, sinks=4, type="f16"),
        # Prompts of odd lengths, each behind a part that is in the cache, in 32 bits.
        dict(name="attend_prompt_ragged", op="attend", sequences=7, longest=1009, shortest=61, new=415, pad=0, heads=12,
             kv_heads=4, dim=64, page=16, window=0, sinks=0, type="f32"),
        # A token's keys and values of each of a batch.
        dict(name="write_step", op="write", sequences=64, longest=32, shortest=1, new=1, pad=0, kv_heads=8, dim=128, page=16,
             type="bf16"),
        # Keys and values of prompts of odd lengths.
        dict(name="write_prompt", op="write", sequences=5, longest=4001, shortest=509, new=4001, pad=11, kv_heads=8,
             dim=128, page=64, type="f16"),
        # A token of each of many requests, most with an adapter of their own.
        dict(name="adapters_step", op="adapters", M=64, K=4096, N=4096, rank=16, count=64, requests=64, input="bf16",
             output="bf16", type="bf16", bias=False, relu=False),
        # A small layer whose sizes are odd.
        dict(name="adapters_ragged", op="adapters", M=61, K=415, N=509, rank=5, count=3, requests=9, input="f32",
             output="f32", type="f32", bias=True, relu=True),
        # The prompts of a few requests.
        dict(name="adapters_prompt", op="adapters", M=4096, K=4096, N=4096, rank=64, count=8, requests=6, input="f16",
             output="f16", type="f16", bias=False, relu=False),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "adapters", "adapters"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "adapters":
        M, K, N, rank = _log(rng, 1, 4096), _log(rng, 16, 8192), _log(rng, 16, 8192), _log(rng, 1, 64)
        while 2 * M * (K * N + rank * (K + N)) > MOST_FLOPS:
            M, N = max(1, M // 2), max(16, N * 3 // 4)
        return dict(op=op, M=M, K=K, N=N, rank=rank, count=_log(rng, 1, 64), requests=_log(rng, 1, min(M, 100)),
                    input=rng.choice([kind, "mx4"]), output=kind, type=kind, bias=rng.random() < 0.5,
                    relu=rng.random() < 0.3)
    kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
    c = dict(op=op, kv_heads=kv_heads, dim=dim, page=rng.choice([0, 16, 32, 64, 256]), pad=rng.choice([0, 0, 1, 7]),
             type=kind)
    if op == "write":
        sequences = _log(rng, 1, 64)
        longest = _log(rng, 1, max(1, 20000 // sequences))
        return dict(c, sequences=sequences, longest=longest, shortest=_log(rng, 1, longest),
                    new=longest if rng.random() < 0.5 else _log(rng, 1, min(longest, 64)))
    window = rng.choice([0, 0, _log(rng, 1, 8192)])
    c.update(heads=kv_heads * rng.choice([1, 2, 3, 4, 8]), window=window, sinks=rng.choice([0, 4, 7]) if window else 0)
    how = rng.choice(["step", "step", "draft", "prompt"])
    if how == "prompt":
        sequences = _log(rng, 1, 8)
        longest = _log(rng, 1, 4096)
        while sequences * longest * longest * c["heads"] * dim > 2 * 4096 * 4096 * 4096:
            longest = longest * 3 // 4
        new = longest if rng.random() < 0.7 else _log(rng, 1, longest)
    else:
        sequences = _log(rng, 1, 128)
        longest = _log(rng, 1, min(131072, MOST_TOKENS // sequences))
        new = 1 if how == "step" else min(longest, rng.randint(2, 8))
    return dict(c, sequences=sequences, longest=longest, shortest=_log(rng, 1, longest), new=new)


# ---- microscaled rows ----------------------------------------------------------------

def row_bytes(cols):
    groups = -(-cols // 128)
    return -(-groups * 68 // 16) * 16


def _to_mx4(x):
    """The values that the rows of x [.., cols] stand for as microscaled rows, scaled to their
    blocks, and the blocks' exponents: both [.., blocks, 32] and [.., blocks, 1], 32 bits."""
    cols = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -cols % 32)).unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    e = (((most.view(torch.int32) >> 23) & 255) - 127 - 2).clamp(-127, 127)
    # by the power of two in two factors: 2^127 and 2^-127 are no normal numbers' inverses
    half = e >> 1
    v = torch.ldexp(torch.ldexp(x, -half), -(e - half))
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    v = (torch.round(v / step) * step).clamp(-6, 6)   # (round() takes ties to even)
    return v, torch.where(most == 0, -127, e)


def _rounded(x):
    """x [.., cols] with every value replaced by what its microscaled form stands for."""
    v, e = _to_mx4(x)
    half = e >> 1
    return torch.ldexp(torch.ldexp(v, half), e - half).flatten(-2)[..., :x.shape[-1]]


def _packed(x):
    """x [rows, cols] as microscaled rows, uint8 [rows, row_bytes(cols)]."""
    rows, cols = x.shape
    v, e = _to_mx4(x)
    size = (v.abs() * 2).int()                        # 0 1 2 3 4 6 8 12
    code = torch.where(size < 4, size, torch.where(size < 8, 2 + size // 2, 4 + size // 4))
    code = (code + torch.where(v < 0, 8, 0)).flatten(-2)
    out = torch.zeros(rows, row_bytes(cols), dtype=torch.uint8, device=x.device)
    groups = -(-cols // 128)
    out[:, :code.shape[1] // 2] = (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)
    out[:, 64 * groups:64 * groups + e.shape[1]] = (e[..., 0] + 127).to(torch.uint8)
    return out


def _unpacked(rows, cols):
    """What microscaled rows stand for, float32 [rows, cols]."""
    groups = -(-cols // 128)
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=rows.device)
    b = rows[:, :64 * groups]
    v = table[torch.stack((b & 15, b >> 4), -1).flatten(1).int()]
    e = rows[:, 64 * groups:68 * groups].int() - 127
    v = v.unflatten(1, (-1, 32))
    return torch.ldexp(v, e.unsqueeze(-1)).flatten(1)[:, :cols]


# ---- states --------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _lengths(c):
    """Tokens of each sequence, and how many of them are new."""
    n, lo, hi = c["sequences"], c["shortest"], c["longest"]
    # spread evenly between the two, the longest first, in no order
    lengths = [hi - int((hi - lo) * (i * 0.6180339887 % 1.0)) for i in range(n)]
    return lengths, [min(t, c["new"]) for t in lengths]


def _page_tokens(c):
    return c["page"] or -(-c["longest"] // 16) * 16


def _cache(c, g):
    """A cache's memory, its table and what says which rows of the batch are whose."""
    lengths, new = _lengths(c)
    C, page = c["kv_heads"] * c["dim"], _page_tokens(c)
    per = -(-c["longest"] // page)
    if c["page"]:
        # pages are given out as sequences grow: what belongs to one lies anywhere
        used = [-(-t // page) for t in lengths]
        order = torch.randperm(sum(used), generator=g, device="cuda").int()
        table = torch.full((len(lengths), per), -1, dtype=torch.int32, device="cuda")
        done = 0
        for i, k in enumerate(used):
            table[i, :k] = order[done:done + k]
            done += k
        n_pages = sum(used)
    else:
        table, n_pages = None, per * len(lengths)
    starts = [0]
    for k in new:
        starts.append(starts[-1] + k)
    # keys have columns that stand out, the same for all tokens
    loud = torch.exp(0.5 * _randn(g, 1, C))
    keys, values = (torch.empty(n_pages * page, row_bytes(C), dtype=torch.uint8, device="cuda") for _ in range(2))
    for start in range(0, n_pages * page, 32768):
        part = slice(start, min(n_pages * page, start + 32768))
        keys[part] = _packed(_randn(g, part.stop - part.start, C) * loud)
        values[part] = _packed(_randn(g, part.stop - part.start, C))
    device = dict(dtype=torch.int32, device="cuda")
    return dict(c, keys=keys, values=values, table=table, page_tokens=page, per=per, loud=loud, used=starts[-1],
                rows=starts[-1] + c["pad"], starts=torch.tensor(starts, **device),
                lengths=torch.tensor(lengths, **device))


def _row_adapters(c, g):
    """The adapter of each row: rows of a request stand together, every eighth request has none."""
    M, n, count = c["M"], c["requests"], c["count"]
    order = torch.randperm(count, generator=g, device="cuda").tolist()
    cuts = [M * i // n for i in range(n + 1)]
    ids, mine = [], 0
    for i in range(n):
        a = -1
        if i % 8 != 5:
            a, mine = order[mine % count], mine + 1
        ids.append((cuts[i], cuts[i + 1], a))
    return ids


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] == "adapters":
        M, K, N, rank, kind = c["M"], c["K"], c["N"], c["rank"], TYPES[c["type"]]
        # rows of different sizes, and a few columns that stand out, as activations have
        x = _randn(g, M, K) * torch.exp(0.5 * _randn(g, M, 1)) * torch.exp(0.7 * _randn(g, 1, K))
        ids = _row_adapters(c, g)
        of_row = torch.cat([torch.full((b - a,), i, dtype=torch.int32) for a, b, i in ids]).cuda()
        return dict(c, x=_packed(x) if c["input"] == "mx4" else x.to(TYPES[c["input"]]),
                    w=_packed(_randn(g, N, K) * K ** -0.5), b=_randn(g, N) if c["bias"] else None,
                    down=(_randn(g, c["count"], rank, K) * K ** -0.5).to(kind),
                    up=(_randn(g, c["count"], N, rank) * 0.5 * rank ** -0.5).to(kind),
                    scales=torch.exp(0.5 * _randn(g, c["count"])), ids=ids, of_row=of_row,
                    out=torch.empty(M, N, dtype=TYPES[c["output"]], device="cuda"))
    s = _cache(c, g)
    C, kind = c["kv_heads"] * c["dim"], TYPES[c["type"]]
    if c["op"] == "write":
        # keys and values as they leave one projection: columns of the same rows
        both = (_randn(g, s["rows"], 2 * C) * torch.cat((s["loud"], torch.ones_like(s["loud"])), 1)).to(kind)
        total = s["keys"].shape[0]
        return dict(s, both=both, outs=[torch.empty(total, C, dtype=kind, device="cuda") for _ in range(2)])
    width = c["heads"] * c["dim"]
    return dict(s, q=(1.5 * _randn(g, s["rows"], width)).to(kind),
                out=torch.zeros(s["rows"], width, dtype=kind, device="cuda"))


# ---- the plain form ------------------------------------------------------------------

def _cache_rows(s, sequence, token):
    """The row of the cache where a sequence's token lies."""
    page = token // s["page_tokens"]
    at = s["table"][sequence, page] if s["table"] is not None else sequence * s["per"] + page
    return at.long() * s["page_tokens"] + token % s["page_tokens"]


def _write_plain(s):
    C, n = s["kv_heads"] * s["dim"], s["used"]
    row = torch.arange(n, device="cuda")
    sequence = (row[:, None] >= s["starts"][None, 1:]).sum(1)
    count = s["starts"][1:] - s["starts"][:-1]
    token = s["lengths"][sequence] - count[sequence] + row - s["starts"][sequence]
    at = _cache_rows(s, sequence, token)
    outs = []
    for cache, x in ((s["keys"], s["both"][:n, :C]), (s["values"], s["both"][:n, C:])):
        cache[at] = _packed(x)
        outs.append(_unpacked(cache, C).to(x.dtype))
    return outs


def _attend_plain(s):
    kv, dim, per_kv = s["kv_heads"], s["dim"], s["heads"] // s["kv_heads"]
    longest, S, most = s["longest"], s["sequences"], min(s["new"], s["longest"])
    out = torch.zeros(s["rows"], kv, per_kv, dim, device="cuda")
    token = torch.arange(longest, device="cuda")
    step = max(1, (1 << 28) // (longest * kv * dim))
    for first in range(0, S, step):
        seq = torch.arange(first, min(S, first + step), device="cuda")
        begin, length = s["starts"][seq].long(), s["lengths"][seq].long()
        count = s["starts"][seq + 1] - begin
        i = torch.arange(most, device="cuda")[None]
        there = i < count[:, None]                                   # [sequences, rows]
        row = (begin[:, None] + i).clamp(max=s["rows"] - 1)
        position = (length - count)[:, None] + i
        rows = torch.where(token < length[:, None], _cache_rows(s, seq[:, None], token[None]), 0).flatten()
        K, V = (_unpacked(t[rows], kv * dim).view(len(seq), longest, kv, dim) for t in (s["keys"], s["values"]))
        seen = (token <= position[..., None]) & (token < length[:, None, None])
        if s["window"]:
            seen &= (token > position[..., None] - s["window"]) | (token < s["sinks"])
        q = s["q"][row].float().view(len(seq), most, kv, per_kv, dim)
        for h in range(kv):
            a = q[:, :, h].flatten(1, 2) @ K[:, :, h].transpose(1, 2).contiguous() * dim ** -0.5
            a = torch.where(seen.repeat_interleave(per_kv, 1), a, float("-inf"))
            p = torch.exp(a - a.amax(-1, keepdim=True).clamp(min=-3e38))
            o = p @ V[:, :, h].contiguous() / p.sum(-1, keepdim=True).clamp(min=EPSILON)
            out[row[there], h] = o.unflatten(1, (most, per_kv))[there]
    return out.flatten(1).to(s["q"].dtype)


def _adapters_plain(s):
    M, K, N, rank = s["M"], s["K"], s["N"], s["rank"]
    x = _unpacked(s["x"], K) if s["input"] == "mx4" else s["x"].float()
    y = (x if s["input"] == "mx4" else _rounded(x)) @ _unpacked(s["w"], K).t()
    if s["requests"] * 4 > M:                        # few rows of each: as a batch of single rows
        some = (s["of_row"] >= 0)[:, None]
        of_row = s["of_row"].clamp(min=0)
        low = (s["down"][of_row].float() * x[:, None]).sum(-1) * s["scales"][of_row][:, None]
        y = y + torch.where(some, (s["up"][of_row].float() * low[:, None]).sum(-1), 0)
    else:
        for a, b, i in s["ids"]:
            if i >= 0:
                y[a:b] += x[a:b] @ s["down"][i].float().t() @ (s["up"][i].float() * s["scales"][i]).t()
    if s["b"] is not None:
        y = y + s["b"]
    return (y.clamp(min=0) if s["relu"] else y).to(TYPES[s["output"]])


# ---- the library's calls -------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _capi():
    from glow_amd import capi
    capi.init(0)
    return capi


def _workspace(s, ask):
    """Scratch memory that the program keeps with its buffers; `ask` says how much."""
    if "workspace" not in s:
        n = ask()
        s["workspace"] = (torch.empty(n, dtype=torch.uint8, device="cuda") if n else None, n)
    t, n = s["workspace"]
    return (t.data_ptr() if n else 0), n


def _address(t):
    return 0 if t is None else t.data_ptr()


def _handle(s, make):
    """The description of a cache or of adapters that a program keeps with them."""
    if "handle" not in s:
        s["handle"] = make()
    return s["handle"]


def _run_own(s):
    capi, op = _capi(), s["op"]
    if op == "adapters":
        M, K, N, kind, x, out = s["M"], s["K"], s["N"], CODES[s["input"]], s["x"], s["out"]
        adapters = _handle(s, lambda: capi.Mx4Adapters(s["down"].data_ptr(), s["up"].data_ptr(), s["scales"].data_ptr(),
                                                       s["count"], s["rank"], CODES[s["type"]]))
        capi.launch_mx4_fc_adapters(
            out.data_ptr(), CODES[s["output"]], N * out.element_size(), x.data_ptr(), kind, x.shape[1] * x.element_size(),
            s["w"].data_ptr(), s["w"].shape[1], _address(s["b"]), adapters, s["of_row"].data_ptr(), M, K, N,
            capi.ACT_RELU if s["relu"] else capi.ACT_NONE,
            *_workspace(s, lambda: capi.mx4_fc_adapters_workspace_bytes(M, K, N, kind, s["rank"])))
        return out
    C = s["kv_heads"] * s["dim"]
    cache = _handle(s, lambda: capi.Mx4Cache(s["keys"].data_ptr(), s["values"].data_ptr(), s["keys"].shape[1],
                                             _address(s["table"]), s["keys"].shape[0] // s["page_tokens"],
                                             s["page_tokens"], s["per"], s["kv_heads"], s["dim"]))
    kind = CODES[s["type"]]
    if op == "write":
        both, size = s["both"], s["both"].element_size()
        capi.launch_mx4_cache_write(cache, both.data_ptr(), both.data_ptr() + C * size, kind, 2 * C * size,
                                    s["starts"].data_ptr(), s["lengths"].data_ptr(), s["sequences"], s["rows"])
        for t, out in zip((s["keys"], s["values"]), s["outs"]):
            capi.launch_mx4_dequantize(out.data_ptr(), kind, C * size, t.data_ptr(), t.shape[1], t.shape[0], C)
        return s["outs"]
    q, out = s["q"], s["out"]
    pitch = q.shape[1] * q.element_size()
    capi.launch_mx4_attention(
        out.data_ptr(), kind, pitch, q.data_ptr(), kind, pitch, s["heads"], cache, s["starts"].data_ptr(),
        s["lengths"].data_ptr(), s["sequences"], s["rows"], s["longest"], s["dim"] ** -0.5, s["window"], s["sinks"],
        *_workspace(s, lambda: capi.mx4_attention_workspace_bytes(cache, s["heads"], s["sequences"], s["rows"],
                                                                  s["longest"])))
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend_plain, "write": _write_plain, "adapters": _adapters_plain}[state["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------

def _size(kind):
    return 4 if kind == "f32" else 2


def _seen(c):
    """Tokens that some row of their sequence sees, and pairs of a row and a token that it sees."""
    tokens = pairs = 0
    w, sinks = c["window"], c["sinks"]
    for length, new in zip(*_lengths(c)):
        first = length - new
        if not w:
            tokens += length
            pairs += new * first + new * (new + 1) // 2
        else:
            begin = max(0, first - w + 1)
            tokens += length - begin + min(sinks, begin)
            for p in range(first, length):
                pairs += min(p + 1, w + min(sinks, max(0, p + 1 - w)))
    return tokens, pairs


def work(case):
    c, op = case, case["op"]
    if op == "adapters":
        M, K, N, rank = c["M"], c["K"], c["N"], c["rank"]
        with_one = sum(i % 8 != 5 for i in range(c["requests"]))
        rows = sum(M * (i + 1) // c["requests"] - M * i // c["requests"] for i in range(c["requests"]) if i % 8 != 5)
        x = M * (row_bytes(K) if c["input"] == "mx4" else K * _size(c["input"]))
        return dict(bytes=x + N * row_bytes(K) + M * N * _size(c["output"]) + (4 * N if c["bias"] else 0) + 4 * M +
                    min(with_one, c["count"]) * rank * (K + N) * _size(c["type"]),
                    flops=2 * M * K * N + 2 * rows * rank * (K + N))
    C, (lengths, new) = c["kv_heads"] * c["dim"], _lengths(c)
    if op == "write":
        page = _page_tokens(c)
        total = sum(-(-t // page) for t in lengths) * page if c["page"] else page * len(lengths)
        # the packed rows are written and read: they are what the calls hand on
        return dict(bytes=2 * (sum(new) * (C * _size(c["type"]) + row_bytes(C)) + total * (C * _size(c["type"]) + row_bytes(C))),
                    flops=4 * C * (sum(new) + total))
    tokens, pairs = _seen(c)
    width = c["heads"] * c["dim"]
    return dict(bytes=2 * tokens * C * 17 // 32 + 2 * sum(new) * width * _size(c["type"]),
                flops=4 * width * pairs)


# ---- the definitions in 64 bits ----------------------------------------------------------

_BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)     # between neighbours of the E2M1 values
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx4_exact(x):
    """Each value of x (64 bits) as the nearest E2M1 value times its block's power of two; on a
    border the one with the even code."""
    parts = []
    for block in x.split(32, -1):
        most = block.abs().amax(-1, keepdim=True)
        _, e = torch.frexp(most)                        # most = m * 2^e, 0.5 <= m < 1
        unit = torch.exp2((e.double() - 3).clamp(-127, 127))
        size = block.abs() / unit
        low, high = (torch.bucketize(size, torch.tensor(_BORDERS, dtype=torch.float64, device=x.device), right=r)
                     for r in (False, True))
        code = torch.where(low % 2 == 0, low, high)     # on a border `low` is the lower code
        value = torch.tensor(_VALUES, dtype=torch.float64, device=x.device)[code]
        parts.append(torch.where(most == 0, 0.0, torch.copysign(value * unit, block)))
    return torch.cat(parts, -1)


def _rows_exact(rows, cols):
    """The values of microscaled rows, column by column of their bytes."""
    groups = (cols + 127) // 128
    column = torch.arange(cols, device=rows.device)
    code = (rows[:, column // 2].long() >> (4 * (column % 2))) & 15
    scale = rows[:, 64 * groups + column // 32].double()
    value = torch.tensor(_VALUES, dtype=torch.float64, device=rows.device)[code & 7]
    return torch.where(code >= 8, -value, value) * torch.exp2(scale - 127)


def _places(s, sequence, length):
    """Where the tokens of a sequence lie, page by page."""
    page, places = s["page_tokens"], []
    for k in range(-(-length // page)):
        at = int(s["table"][sequence, k]) if s["table"] is not None else sequence * s["per"] + k
        places.append(torch.arange(at * page, at * page + min(page, length - k * page), device="cuda"))
    return torch.cat(places)


def _attend_exact(s):
    kv, dim = s["kv_heads"], s["dim"]
    group = s["heads"] // kv
    out = torch.zeros(s["rows"], s["heads"], dim, dtype=torch.float64, device="cuda")
    lengths, news = _lengths(s)
    if s["table"] is not None:
        s = dict(s, table=s["table"].cpu())
    row = 0
    for i, (length, new) in enumerate(zip(lengths, news)):
        places = _places(s, i, length)
        K, V = (_rows_exact(t[places], kv * dim).view(length, kv, dim).transpose(0, 1).contiguous()
                for t in (s["keys"], s["values"]))
        q = s["q"][row:row + new].double().view(new, kv, group, dim)
        for first in range(0, new, 1024):
            last = min(new, first + 1024)
            position = torch.arange(length - new + first, length - new + last, device="cuda")[:, None]
            begin = max(0, length - new + first - s["window"] + 1) if s["window"] else 0
            see = [t for t in range(min(s["sinks"], begin))] if s["window"] else []
            token = torch.cat((torch.tensor(see, dtype=torch.int64, device="cuda"),
                               torch.arange(begin, length - new + last, device="cuda")))
            hidden = token > position
            if s["window"]:
                hidden |= (token <= position - s["window"]) & (token >= s["sinks"])
            for h in range(kv):
                a = torch.einsum("rgd,td->rgt", q[first:last, h], K[h, token]) / dim ** 0.5
                p = torch.softmax(a.masked_fill(hidden[:, None], float("-inf")), -1)
                out[row + first:row + last, h * group:(h + 1) * group] = torch.einsum("rgt,td->rgd", p, V[h, token])
        row += new
    return out.flatten(1)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "attend":
        return _attend_exact(s)
    if op == "write":
        C, (lengths, news) = s["kv_heads"] * s["dim"], _lengths(s)
        outs = [_rows_exact(t, C) for t in (s["keys"], s["values"])]
        row = 0
        for i, (length, new) in enumerate(zip(lengths, news)):
            places = _places(s, i, length)[length - new:]
            for k, out in enumerate(outs):
                out[places] = _mx4_exact(s["both"][row:row + new, k * C:(k + 1) * C].double())
            row += new
        return outs
    x = _rows_exact(s["x"], s["K"]) if s["input"] == "mx4" else s["x"].double()
    y = torch.mm(x if s["input"] == "mx4" else _mx4_exact(x), _rows_exact(s["w"], s["K"]).T.contiguous())
    for a, b, i in s["ids"]:
        if i >= 0:
            low = torch.mm(x[a:b], s["down"][i].double().T.contiguous()) * s["scales"][i].double()
            y[a:b] += torch.mm(low, s["up"][i].double().T.contiguous())
    if s["b"] is not None:
        y += s["b"].double()
    return torch.relu(y) if s["relu"] else y
