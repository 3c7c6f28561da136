"""A decoder's attention layer over a key-value cache held in 4 bits: what is timed and compared.

Four operators, in the order in which a layer runs them between its projections:

  rope       queries and keys of each head normed (RMS, gamma) and rotated by position in one pass
  store      keys and values quantised into the cache's pages, and read back as the values that they now stand for
  read       a cache's positions as numbers
  attention  softmax(scale Q K^T) V over the cache, causal, for one new token a sequence, some, or whole prompts;
             optionally a window, and the result gated: Y * sigmoid(G)

The cache is a pool of pages of 64 positions. A page holds, for each key-value head, a tile of 68 * pitch bytes,
pitch = the head's dimension rounded up to a multiple of 64 with zeros past it, nb = pitch / 32 blocks:

  key codes     [64 positions][pitch / 2]        dimension 2j in the low half of byte j, 2j + 1 in the high half
  value codes   [nb][4 q][16 r][4 g][4 i]        position 16 g + 4 q + i, dimensions 32 b + r (low half), 32 b + 16 + r
  key scales    [nb][16 n][4 g]                  position 16 g + n
  value scales  [nb][4 q][4 g][4 i]              position 16 g + 4 q + i

A code is e2m1 (sign, then 0, 1/2, 1, 3/2, 2, 3, 4, 6), a scale the e8m0 byte of a power of two for 32 dimensions of
one position: the smallest from 2^-125 to 2^125 with the block's largest magnitude at most 6 scales, 1 for a block of
zeros; 255 marks a block that had a value which is not finite, and stands for 32 NaN.

A sequence's new tokens are rows starts[s] to starts[s + 1] and its last positions; lengths[s] counts its positions
with them; table[s] names its pages in order.

``listed()`` names the fixed cases, ``draw`` makes more of the same ranges, ``prepare`` builds a program's inputs
(library buffers when the library is called, plain tensors otherwise; the same values), ``run`` is one pass, ``work``
the bytes and operations it cannot do without, ``exact`` the same results in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-6
PAGE = 64
TYPES = ["f32", "bf16"]
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---------------------------------------------------------------- the cases
# new, length: the longest sequence's; the others have some less of both, by `ragged` (0: all alike).
def _attention(**c):
    return dict(dict(kind="attention", seqs=1, new=1, ragged=0.0, window=0, gate=False), **c)


def listed():
    return [
        # One token's queries, beside their gates in the projection's rows, and its keys: the smallest call.
        dict(name="rope_token", kind="rope", tokens=1, heads=24, kv=2, dim=256, rotary=64, gate=True, type="f32"),
        # The same of a prompt.
        dict(name="rope_prompt", kind="rope", tokens=4096, heads=24, kv=2, dim=256, rotary=64, gate=True, type="bf16"),
        # A decode step of 32 sequences.
        dict(name="store_step", kind="store", seqs=32, new=1, length=4000, ragged=0.8, kv=8, dim=128, type="f32"),
        # A long prompt behind a few tokens that were there.
        dict(name="store_prompt", kind="store", seqs=1, new=8192, length=8229, ragged=0.0, kv=8, dim=128, type="bf16"),
        # A few short sequences taken out of the cache, as a session is saved.
        dict(name="read_short", kind="read", seqs=5, length=333, ragged=0.9, kv=2, dim=256, type="f32"),
        # Long ones.
        dict(name="read_long", kind="read", seqs=4, length=16384, ragged=0.3, kv=2, dim=256, type="bf16"),
        # One token of one session.
        _attention(name="decode_token", length=2048, heads=24, kv=2, dim=256, gate=True, type="f32"),
        # A step of a batch of sequences of all lengths.
        _attention(name="decode_batch32", seqs=32, length=8192, ragged=0.9, heads=32, kv=8, dim=128, type="bf16"),
        # One token over a very long context.
        _attention(name="decode_long", length=131072, heads=24, kv=2, dim=256, gate=True, type="bf16"),
        # Short prompts of a batch, heads that fill no block, a sliding window.
        _attention(name="prompt_ragged", seqs=5, new=333, length=500, ragged=0.9, heads=12, kv=4, dim=80, window=200,
                   type="f32"),
        # A chunk late in a long prompt.
        _attention(name="chunk_late", new=512, length=32768, heads=24, kv=2, dim=256, gate=True, type="bf16"),
        # A whole prompt at once: the largest call.
        _attention(name="prompt", new=8192, length=8192, heads=32, kv=8, dim=128, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _heads(rng):
    """(heads, key-value heads, dimension)"""
    return rng.choice([(24, 2, 256), (24, 2, 256), (32, 8, 128), (32, 8, 128), (16, 16, 64), (8, 1, 128), (12, 4, 80), (20, 4, 96),
                       (40, 2, 64), (6, 2, 192), (5, 5, 40)])


def draw(rng):
    kind = rng.choice(["rope", "store", "read", "attention", "attention", "attention"])
    heads, kv, dim = _heads(rng)
    c = dict(kind=kind, kv=kv, dim=dim, type=rng.choice(TYPES))
    if kind == "rope":
        rotary = rng.choice([dim, max(2, dim // 4 // 2 * 2), dim // 2])
        return dict(c, tokens=_log(rng, 1, min(8192, (1 << 25) // ((heads + kv) * dim))), heads=heads, rotary=rotary, gate=rng.random() < 0.5)
    c["seqs"] = _log(rng, 1, 48)
    c["ragged"] = rng.choice([0.0, 0.5, 0.9])
    if kind == "store":
        c["new"] = rng.choice([1, _log(rng, 2, 8), _log(rng, 9, max(9, 16384 // c["seqs"]))])
        return dict(c, length=c["new"] + _log(rng, 1, 8192) - 1)
    if kind == "read":
        return dict(c, length=_log(rng, 1, 65536 // c["seqs"]))
    c.update(heads=heads, window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]), gate=rng.random() < 0.3)
    how = rng.choice(["token", "token", "few", "prompt", "prompt"])
    if how == "prompt":
        c["new"] = _log(rng, 9, max(9, 4096 // c["seqs"]))
        past = min(131072 // c["seqs"], (1 << 30) // (heads * c["seqs"] * c["new"]))
        return dict(c, length=c["new"] + rng.choice([0, _log(rng, 1, past)]))
    c["new"] = 1 if how == "token" else rng.randint(2, 8)
    return dict(c, length=c["new"] + _log(rng, 1, 131072 // c["seqs"]) - 1)


def _spread(n, ragged, k):
    """n, or up to `ragged` of it less for the sequence k: the first has it whole."""
    return max(1, round(n * (1 - ragged * ((0.6180339887 * k) % 1.0))))


def _sequences(case):
    """(new tokens, length) of each sequence."""
    found = []
    for k in range(case["seqs"]):
        length = _spread(case["length"], case["ragged"], k)
        new = length if case["kind"] == "read" else min(length, _spread(case["new"], case["ragged"], 3 * k))
        found.append((new, length))
    return found


# ------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, seed, sigma=1.0):
    return torch.randn(shape, generator=_gen(seed), device="cuda") * sigma


def _dtype(case):
    return torch.bfloat16 if case["type"] == "bf16" else torch.float32


def _pitch(dim):
    return -(-dim // 64) * 64


def _keys(shape, seed):
    """Keys [.., heads, dim] as a layer has them: normal around a channel's own mean, some channels larger."""
    channels = shape[-2:]
    return _normal(shape, seed) * torch.exp(_normal(channels, seed + 1, 0.4)) + _normal(channels, seed + 2, 0.6)


def _codes(x):
    """(code bytes, scale bytes) of x [.., dim] in f32, dim a multiple of 32."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e, 1/2 <= m < 1; at most 6 2^s for s = e - 3, one more past 3/4
    s = torch.where(amax > 0, (e - 3 + (m > 0.75)).clamp(-125, 125), 0)
    y = torch.ldexp(b, -s[..., None])
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    v = torch.round(a / step) * step  # ties to even, as e2m1's last bit is the step's count
    code = torch.where(v < 2, 2 * v, torch.where(v < 4, v + 2, v / 2 + 4)).clamp(max=7)
    code = torch.where(y.signbit(), code + 8, code)
    bad = ~amax.isfinite()
    code = torch.where(bad[..., None], 0.0, code)
    return code.to(torch.uint8).view(x.shape), torch.where(bad, 255, s + 127).to(torch.uint8)


def _tiles(pool, kv, dim):
    """The pool's four parts as views: key codes [P, kv, 64, pitch / 2], value codes [P, kv, nb, 4 q, 16 r, 4 g, 4 i],
    key scales [P, kv, nb, 16 n, 4 g], value scales [P, kv, nb, 4 q, 4 g, 4 i]."""
    pitch = _pitch(dim)
    t, nb = pool.view(-1, kv, 68 * pitch), pitch // 32
    parts = torch.split(t, [32 * pitch, 32 * pitch, 2 * pitch, 2 * pitch], -1)
    return (parts[0].unflatten(-1, (64, pitch // 2)), parts[1].unflatten(-1, (nb, 4, 16, 4, 4)),
            parts[2].unflatten(-1, (nb, 16, 4)), parts[3].unflatten(-1, (nb, 4, 4, 4)))


def _put_codes(pool, kv, dim, page, at, k, ks, v, vs):
    """Codes [T, kv, pitch] and scales [T, kv, nb] of keys and values into positions `at` of pages `page`."""
    tk, tv, tks, tvs = _tiles(pool, kv, dim)
    g, q, i, n = at // 16, at // 4 % 4, at % 4, at % 16
    tk[page, :, at] = k[..., 0::2] | k[..., 1::2] << 4
    tks[page, :, :, n, g] = ks
    v = v.unflatten(-1, (-1, 2, 16))
    tv[page, :, :, q, :, g, i] = v[..., 0, :] | v[..., 1, :] << 4
    tvs[page, :, :, q, g, i] = vs


def _numbers(codes, scales):
    """What codes [.., pitch] and scales [.., nb] stand for, in f32."""
    table = torch.tensor(VALUES + [-v for v in VALUES], device=codes.device)
    s = torch.where(scales == 255, math.nan, torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127))
    return (table[codes.int()].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _pages(pool, kv, dim, table):
    """Keys and values [.., 64 * pages, kv, dim] of the pages in table [.., pages]."""
    pitch = _pitch(dim)
    tk, tv, tks, tvs = _tiles(pool.view(-1, kv * 68 * pitch)[table], kv, dim)
    k = torch.stack([tk & 15, tk >> 4], -1).flatten(-2)  # [P, kv, 64, pitch]
    v = torch.stack([tv & 15, tv >> 4], 3)  # [P, kv, nb, half, q, r, g, i]
    v = v.permute(0, 1, 6, 4, 7, 2, 3, 5).reshape(k.shape)
    ks = tks.permute(0, 1, 4, 3, 2).flatten(2, 3)  # [P, kv, 64, nb]
    vs = tvs.permute(0, 1, 4, 3, 5, 2).flatten(2, 4)
    shape = (*table.shape[:-1], 64 * table.shape[-1], kv, pitch)
    out = [_numbers(c, s).transpose(1, 2).reshape(shape)[..., :dim] for c, s in ((k, ks), (v, vs))]
    return out[0], out[1]


def _pad(x, dim):
    return torch.nn.functional.pad(x, (0, _pitch(dim) - dim))


def _batch(case, seed):
    """The sequences' starts, lengths and tables, and how many pages there are: theirs in any order, and two more."""
    seqs = _sequences(case)
    need = [-(-n // PAGE) for _, n in seqs]
    width, pages = max(need), sum(need) + 2
    order = torch.randperm(pages, generator=_gen(seed), device="cuda").int()
    table = torch.zeros((len(seqs), width), dtype=torch.int32, device="cuda")
    first = 0
    for s, n in enumerate(need):
        table[s, :n] = order[first:first + n]
        first += n
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    return {"starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "lengths": torch.tensor([n for _, n in seqs], dtype=torch.int32, device="cuda"), "table": table}, pages


def _filled(case, pages, seed):
    """A pool of pages whose every position holds a key and a value."""
    kv, dim = case["kv"], case["dim"]
    pool = torch.zeros(pages * kv * 68 * _pitch(dim), dtype=torch.uint8, device="cuda")
    at = torch.arange(pages * PAGE, device="cuda")
    k, v = _keys((pages * PAGE, kv, dim), seed), _normal((pages * PAGE, kv, dim), seed + 5)
    _put_codes(pool, kv, dim, at // PAGE, at % PAGE, *_codes(_pad(k, dim)), *_codes(_pad(v, dim)))
    return pool


def _tables(case, context):
    """Cosines and sines [context, rotary / 2], the angles in 64 bits."""
    half = case["rotary"] // 2
    speed = torch.exp(torch.arange(half, dtype=torch.float64, device="cuda") * (-2 * math.log(1e7) / case["rotary"]))
    angle = torch.arange(context, dtype=torch.float64, device="cuda")[:, None] * speed
    return angle.cos().float(), angle.sin().float()


def _context(case):
    return 2 * case["tokens"] + 1000


def _inputs(case, seed):
    """The pass's inputs by name, and the pool's pages."""
    kind, kv, dim, seed = case["kind"], case["kv"], case["dim"], 100 * seed
    if kind == "rope":
        n, heads = case["tokens"], case["heads"]
        first = torch.randint(0, _context(case) - n, (1,), generator=_gen(seed + 1), device="cuda")
        cos, sin = _tables(case, _context(case))
        return {"Q": (3 * _keys((n, heads, (2 if case["gate"] else 1) * dim), seed + 2)).to(_dtype(case)),
                "K": (3 * _keys((n, kv, dim), seed + 10)).to(_dtype(case)), "q_gamma": 1 + _normal((dim,), seed + 20, 0.1),
                "k_gamma": 1 + _normal((dim,), seed + 21, 0.1), "cos": cos, "sin": sin,
                "positions": (first + torch.arange(n, device="cuda")).int()}, 0
    t, pages = _batch(case, seed + 1)
    n = sum(new for new, _ in _sequences(case))
    t["pool"] = _filled(case, pages, seed + 2)
    if kind == "store":
        t["K"] = _keys((n, kv, dim), seed + 10).to(_dtype(case))
        t["V"] = _normal((n, kv, dim), seed + 20).to(_dtype(case))
    if kind == "attention":
        heads = case["heads"]
        t["Q"] = (_normal((n, heads, dim), seed + 10) + _normal((heads, dim), seed + 11, 0.5)).to(_dtype(case))
        if case["gate"]:  # queries and gates side by side, as the projection leaves them
            t["G"] = _normal((n, heads, 2 * dim), seed + 20).to(_dtype(case))
    return t, pages


# ------------------------------------------------------------------ prepare
_held = {}


def _backend():
    """The program's one context on the GPU."""
    if "backend" not in _held:
        import stratacuda_amd as sm

        _held["backend"] = sm.Backend(0)
    return _held["backend"]


class _Owned:
    """A library buffer freed with its last user, readable as a torch tensor of bytes."""

    def __init__(self, nbytes):
        self.buf = _backend().alloc_bytes(nbytes)
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (self.buf.handle, False),
                                         "version": 2, "strides": None}

    def __del__(self):
        try:
            _backend().free(self.buf)
        except Exception:
            pass


def _empty(shape, dtype):
    """(buffer, tensor over it); the tensor keeps the buffer."""
    nbytes = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
    held = _Owned(nbytes)
    return held.buf, torch.as_tensor(held, device="cuda").view(dtype).view(shape)


def _put(t):
    buf, view = _empty(t.shape, t.dtype)
    view.view(torch.uint8).copy_(t.contiguous().view(torch.uint8))
    return buf, view


def prepare(case, seed):
    t, pages = _inputs(case, seed)
    s = {"case": case, "pages": pages, "longest": max((new for new, _ in _sequences(case)), default=0) if pages else 0}
    if not own:
        return dict(s, **{"in": t})
    # The library takes the buffers that it allocated: the same inputs there,
    # and the outputs and workspace that a program keeps.
    import stratacuda_amd as sm

    s["in"] = {k: _put(v) for k, v in t.items()}
    kind, kv, dim = case["kind"], case["kv"], case["dim"]
    if kind == "rope":
        s["Q"] = _empty((case["tokens"], case["heads"], dim), _dtype(case))
        s["K"] = _empty((case["tokens"], kv, dim), _dtype(case))
    else:
        new = [n for n, _ in _sequences(case)]
        b = {k: s["in"][k][0] for k in ("starts", "lengths", "table")}
        s["sequences"] = sm.Sequences(count=len(new), tokens=sum(new), longest=s["longest"], starts=b["starts"],
                                      lengths=b["lengths"], table=b["table"], table_pages=t["table"].shape[1])
        if kind == "attention":
            s["Y"] = _empty((sum(new), case["heads"], dim), _dtype(case))
            s["workspace"] = _empty((max(1, _backend().kv4_attention_workspace_bytes(s["sequences"], case["heads"], kv, dim)),),
                                    torch.uint8)
        else:
            s["K"], s["V"] = _empty((sum(new), kv, dim), _dtype(case)), _empty((sum(new), kv, dim), _dtype(case))
    torch.cuda.synchronize()  # the library's stream starts from finished inputs
    return s


# ---------------------------------------------------------------------- run
def _run_own(s):
    be, c = _backend(), s["case"]
    t = {k: v[0] for k, v in s["in"].items()}
    kind, kv, dim = c["kind"], c["kv"], c["dim"]
    if kind == "rope":
        heads, wide = c["heads"], (2 if c["gate"] else 1) * dim
        be.qk_norm_rope(t["Q"], t["K"], c["tokens"], heads, kv, dim, t["q_gamma"], t["k_gamma"], EPS, t["cos"], t["sin"],
                        c["rotary"], _context(c), t["positions"], s["Q"][0], s["K"][0], q_view=(heads * wide, wide, 0),
                        type=c["type"])
        return {"Q": s["Q"][1], "K": s["K"][1]}
    seqs, pool = s["sequences"], t["pool"]
    if kind == "attention":
        be.kv4_attention(t["Q"], seqs, pool, s["pages"], c["heads"], kv, dim, dim ** -0.5, s["Y"][0], s["workspace"][0],
                         window=c["window"], gate=t.get("G"), gate_view=(c["heads"] * 2 * dim, 2 * dim, dim), type=c["type"])
        return {"Y": s["Y"][1]}
    if kind == "store":
        be.kv4_write(t["K"], t["V"], seqs, pool, s["pages"], kv, dim, type=c["type"])
    be.kv4_read(pool, s["pages"], kv, dim, seqs, s["K"][0], s["V"][0], type=c["type"])
    return {"K": s["K"][1], "V": s["V"][1]}


def _rows(t, tokens):
    """For each token its sequence and its position there."""
    row = torch.arange(tokens, device="cuda")
    s = torch.searchsorted(t["starts"][1:].long(), row, right=True)
    return s, (t["lengths"] - t["starts"][1:])[s] + row


def _norm_rope(x, gamma, cos, sin, rotary, positions):
    x = x.float()
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma
    c, s = cos[positions.long()][:, None], sin[positions.long()][:, None]
    a, b = n[..., :rotary // 2], n[..., rotary // 2:rotary]
    return torch.cat([a * c - b * s, b * c + a * s, n[..., rotary:]], -1)


def run(state):
    if own:
        return _run_own(state)
    c, t = state["case"], state["in"]
    kind, kv, dim, to = c["kind"], c["kv"], c["dim"], _dtype(c)
    if kind == "rope":
        q = _norm_rope(t["Q"][..., :dim], t["q_gamma"], t["cos"], t["sin"], c["rotary"], t["positions"])
        k = _norm_rope(t["K"], t["k_gamma"], t["cos"], t["sin"], c["rotary"], t["positions"])
        return {"Q": q.to(to), "K": k.to(to)}
    if kind == "store":
        s, at = _rows(t, t["K"].shape[0])
        page = t["table"][s, at // PAGE].long()
        _put_codes(t["pool"], kv, dim, page, at % PAGE, *_codes(_pad(t["K"].float(), dim)), *_codes(_pad(t["V"].float(), dim)))
    if kind != "attention":
        tokens = t["K"].shape[0] if kind == "store" else sum(n for n, _ in _sequences(c))
        s, at = _rows(t, tokens)
        # whole pages from a sequence's first wanted one on, as many for all
        first = (t["lengths"] - t["starts"].diff()) // PAGE
        many = min(t["table"].shape[1], (state["longest"] + 62) // PAGE + 1)
        cols = (first[:, None] + torch.arange(many, device="cuda")).clamp(max=t["table"].shape[1] - 1)
        k, v = _pages(t["pool"], kv, dim, t["table"].gather(1, cols.long()).long())
        at = at - PAGE * first[s]
        return {"K": k[s, at].to(to), "V": v[s, at].to(to)}
    q, heads = t["Q"].float(), c["heads"]
    s, at = _rows(t, q.shape[0])
    k, v = _pages(t["pool"], kv, dim, t["table"].long())  # [S, L, kv, dim]
    # queries to [S, kv, longest * group, dim], a row for each token's heads
    group, most, count = heads // kv, state["longest"], c["seqs"]
    i = torch.arange(q.shape[0], device="cuda") - t["starts"][s]
    padded = torch.zeros((count, most, heads, dim), device="cuda")
    padded[s, i] = q
    where = torch.full((count, most), -1, dtype=torch.long, device="cuda")
    where[s, i] = at.long()
    padded = padded.view(count, most, kv, group, dim).transpose(1, 2).reshape(count, kv, most * group, dim)
    scores = padded @ k.permute(0, 2, 3, 1).contiguous() * dim ** -0.5
    there = torch.arange(k.shape[1], device="cuda") <= where[..., None]
    if c["window"]:
        there &= torch.arange(k.shape[1], device="cuda") > where[..., None] - c["window"]
    there = there.repeat_interleave(group, 1)[:, None]
    scores = scores.masked_fill_(~there, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    y = p @ v.transpose(1, 2).contiguous() / torch.where(total > 0, total, 1.0)
    y = y.view(count, kv, most, group, dim).transpose(1, 2).reshape(count, most, heads, dim)[s, i]
    if c["gate"]:
        y = y / (1 + torch.exp(-t["G"][..., dim:].float()))
    return {"Y": y.to(to)}


# ---------------------------------------------------------------- the bound
def work(case):
    kind, kv, dim, size = case["kind"], case["kv"], case["dim"], 2 if case["type"] == "bf16" else 4
    if kind == "rope":
        n = case["tokens"] * (case["heads"] + kv) * dim
        return {"bytes": 2 * n * size + case["tokens"] * case["rotary"] * 4 + 8 * dim, "flops": 8 * n}
    seqs = _sequences(case)
    held = lambda positions: 2 * positions * kv * (dim // 2 + -(-dim // 32))  # noqa: E731
    n = sum(new for new, _ in seqs)
    if kind != "attention":
        values = 2 * n * kv * dim
        passes = 2 if kind == "store" else 1
        return {"bytes": passes * (values * size + held(n)), "flops": passes * 2 * values}
    window, heads = case["window"], case["heads"]
    read = pairs = 0
    for new, length in seqs:
        first = length - new  # position of the first query
        if window:
            read += length - max(0, first - window + 1)
            full = max(0, length - max(first, window - 1))  # queries with a whole window
            short = new - full
            pairs += full * window + short * (first + 1) + short * (short - 1) // 2
        else:
            read += length
            pairs += new * (first + 1) + new * (new - 1) // 2
    values = n * heads * dim * size
    return {"bytes": held(read) + values * (3 if case["gate"] else 2), "flops": 4 * pairs * heads * dim}


# ------------------------------------------------------------------ 64 bits
def _exact_rope(x, gamma, case, positions, cos, sin):
    x, half = x.double(), case["rotary"] // 2
    x = x * gamma.double() / (x.square().sum(-1, keepdim=True) / case["dim"] + EPS).sqrt()
    turn = torch.complex(cos.double(), sin.double())[positions.long()][:, None]
    z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)


def _exact_rounded(x):
    """x's nearest values in 4 bits, by the distance to each."""
    x = x.double()
    table = torch.tensor(VALUES, dtype=torch.float64, device="cuda")
    b = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / 6))
    e = e + (amax > 6 * torch.exp2(e)).double() - (amax <= 6 * torch.exp2(e - 1)).double()
    scale = torch.exp2(torch.where(amax > 0, e.clamp(-125, 125), torch.zeros_like(e)))
    a = b.abs() / scale
    low = (torch.searchsorted(table, a.contiguous(), right=True) - 1).clamp(max=6)
    up, down = table[low + 1] - a, a - table[low]
    index = torch.where((up < down) | ((up == down) & (low % 2 == 1)), low + 1, low)
    return (table[index] * b.sign() * scale).flatten(-2)[..., : x.shape[-1]]


def _exact_positions(pool, case, row, first, last):
    """Keys and values of a sequence's positions [first, last) in f64, read byte by byte from where the layout has them."""
    kv, dim, pitch = case["kv"], case["dim"], _pitch(case["dim"])
    p = torch.arange(first, last, device="cuda")
    tile = (row[p // PAGE].long()[:, None] * kv + torch.arange(kv, device="cuda")) * (68 * pitch)  # [n, kv]
    tile, at, d = tile[..., None], (p % PAGE)[:, None, None], torch.arange(dim, device="cuda")
    g, n, q, i, b = at // 16, at % 16, at // 4 % 4, at % 4, d // 32
    table = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64, device="cuda")
    number = lambda byte, high, scale: table[(byte.long() >> (4 * high)) & 15] * torch.exp2(scale.double() - 127)  # noqa: E731
    k = number(pool[tile + at * (pitch // 2) + d // 2], d % 2, pool[tile + 64 * pitch + b * 64 + n * 4 + g])
    v = number(pool[tile + 32 * pitch + b * 1024 + q * 256 + d % 16 * 16 + g * 4 + i], d // 16 % 2,
               pool[tile + 66 * pitch + b * 64 + q * 16 + g * 4 + i])
    return k, v


def exact(case, seed):
    t, _ = _inputs(case, seed)
    kind, kv, dim = case["kind"], case["kv"], case["dim"]
    if kind == "rope":
        return {"Q": _exact_rope(t["Q"][..., :dim], t["q_gamma"], case, t["positions"], t["cos"], t["sin"]),
                "K": _exact_rope(t["K"], t["k_gamma"], case, t["positions"], t["cos"], t["sin"])}
    if kind == "store":
        return {"K": _exact_rounded(t["K"]), "V": _exact_rounded(t["V"])}
    found, row, group = [], 0, case.get("heads", kv) // kv
    for s, (new, length) in enumerate(_sequences(case)):
        if kind == "read":
            found.append(_exact_positions(t["pool"], case, t["table"][s], 0, length))
            continue
        k, v = _exact_positions(t["pool"], case, t["table"][s], 0, length)
        out = torch.empty((new, case["heads"], dim), dtype=torch.float64, device="cuda")
        for lo in range(0, new, 512):  # some rows at a time
            hi = min(new, lo + 512)
            q = t["Q"][row + lo:row + hi].double().view(hi - lo, kv, group, dim)
            own_at = length - new + torch.arange(lo, hi, device="cuda")
            p = torch.arange(length, device="cuda")
            hidden = p > own_at[:, None]
            if case["window"]:
                hidden |= p <= own_at[:, None] - case["window"]
            for h in range(kv):
                score = (q[:, h].reshape(-1, dim) @ k[:, h].T.contiguous()).view(hi - lo, group, length) / math.sqrt(dim)
                w = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), -1)
                out[lo:hi, h * group:(h + 1) * group] = (w.view(-1, length) @ v[:, h].contiguous()).view(hi - lo, group, dim)
        if case["gate"]:
            out = out * torch.sigmoid(t["G"][row:row + new, :, dim:].double())
        found.append(out)
        row += new
    if kind == "read":
        return {"K": torch.cat([k for k, _ in found]), "V": torch.cat([v for _, v in found])}
    return {"Y": torch.cat(found)}
