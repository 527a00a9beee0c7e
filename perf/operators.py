"""The key/value cache in 8 bits as cases that can be timed and checked: what is written to it, read back from it, and attention over it.

A token's key and value of one key/value head are held as ``d`` whole numbers from -127 to 127 and one float32 scale each:
``scale = max(largest / 127, 2^-126)`` with ``largest`` the row's largest magnitude rounded to float32, ``code = x / scale``
rounded to the nearest whole number (halves to the even one).  Three kinds of pass:

* ``store``: a step's rows q|k|v are rotated, the queries go out, keys and values into the cache; then the pages that the
  step wrote to are read back, as the values that their codes stand for.
* ``read``: all pages that some requests hold, as values.
* ``attend``: attention of a step's queries over the cache; ``step`` lists what each request brings ("1*29,333*3": 29
  requests with a single token and three with 333).

Requests are ``longest`` tokens long at most after the step, the others between what they bring and that (``ragged``: spread
evenly over that range, the first one shortest; else all alike).  Their pages lie anywhere in the pool.
"""
import math
from types import SimpleNamespace

import torch

own = False

DEVICE = "cuda"
BLOCK = 16                      # tokens a page, the engine's own choice
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    small = dict(H=14, G=2, d=64, dtype="bf16")               # the heads of the 0.5B configuration
    large = dict(H=28, G=4, d=128, dtype="bf16")              # ... of the 7B one
    wide = dict(H=32, G=8, d=128, dtype="bf16")               # ... of the benchmark's width of 4,096
    plain = dict(window=0, sinks=False, cap=0.0, slopes=False)
    return [
        # a reply's next token, one user: the call whose cost is its launches
        dict(small, name="store one token", op="store", step="1*1", longest=700, ragged=False, n_rot=64, pairing="half"),
        # a prompt's portion, as long as the scheduler cuts it
        dict(large, name="store a prompt", op="store", step="2048*1", longest=4096, ragged=False, n_rot=128, pairing="half"),
        # the float32 run, odd portions, part of a head rotated, neighbours turned together
        dict(name="store in float32", op="store", step="37*5,1*3", longest=500, ragged=True, n_rot=32, pairing="interleaved", H=8, G=8, d=80, dtype="fp32"),
        # one request's cache looked at
        dict(small, name="read one request", op="read", step="1*1", longest=1000, ragged=False),
        # several conversations handed on
        dict(large, name="read long requests", op="read", step="1*4", longest=32768, ragged=True),
        # one user's next token behind a short chat
        dict(small, **plain, name="decode one", op="attend", step="1*1", longest=700, ragged=False),
        # a few users with long documents
        dict(large, **plain, name="decode eight long", op="attend", step="1*8", longest=32768, ragged=True),
        # a full batch, requests from their second token on
        dict(large, **plain, name="decode many", op="attend", step="1*64", longest=8192, ragged=True),
        # a few tokens each at once: ends of prompts, drafts to be looked over
        dict(wide, **plain, name="few tokens each", op="attend", step="5*16", longest=8192, ragged=True),
        # a long prompt's last portion
        dict(large, **plain, name="prompt portion", op="attend", step="2048*1", longest=8192, ragged=False),
        # prompts beside single tokens, in a windowed layer with sinks and capped scores
        dict(name="mixed step", op="attend", step="1*29,333*3", longest=4000, ragged=True, H=16, G=4, d=64, dtype="bf16", window=1024, sinks=True, cap=30.0, slopes=False),
        # the float32 run, heads that no tile fits, a bias linear in the distance
        dict(name="attend in float32", op="attend", step="3*5,1*2", longest=900, ragged=True, H=8, G=2, d=80, dtype="fp32", window=0, sinks=False, cap=0.0, slopes=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["store", "read", "attend", "attend", "attend"])
    d, r = rng.choice([64, 128, 64, 128, 80, 32, 256]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12])
    G = rng.choice([1, 2, 4, 8])
    case = dict(op=op, G=G, d=d, H=G * r, dtype="fp32" if rng.random() < 0.15 else "bf16", ragged=rng.random() < 0.7)
    tiled = case["dtype"] == "bf16" and d in (64, 128)
    if op == "store":
        n, q = log(1, 64), log(1, 512)
        return bounded(dict(case, step="%d*%d" % (q, n), longest=q + log(1, 2000), n_rot=rng.choice([0, d // 2, d]), pairing=rng.choice(["half", "interleaved"])))
    if op == "read":
        return bounded(dict(case, step="1*%d" % log(1, 16), longest=log(1, 12000)))
    case.update(window=rng.choice([0, 0, log(1, 4000)]), sinks=rng.random() < 0.25, cap=rng.choice([0.0, 0.0, 0.0, 30.0]), slopes=rng.random() < 0.2)
    kind = rng.choice(["single", "few", "portion", "mixed"])
    if kind == "single":
        return bounded(dict(case, step="1*%d" % log(1, 64), longest=log(1, 16384 if tiled else 2000)))
    if kind == "few":
        q = rng.randint(2, 16)
        return bounded(dict(case, step="%d*%d" % (q, log(1, 16)), longest=q + log(1, 8000 if tiled else 600)))
    q = log(16, 1500 if tiled else 100)
    longest = q + log(1, 6000 if tiled else 300)
    return bounded(dict(case, step="%d*1" % q if kind == "portion" else "1*%d,%d*1" % (log(1, 24), q), longest=longest))


def bounded(case):
    """The case with histories short enough, and heads few enough, to cost no more than the largest listed ones."""
    most = {n: max(work(c)[n] for c in listed() if c["op"] == case["op"]) for n in ("bytes", "flops")}
    while any(work(case)[n] > most[n] for n in most):
        longest, parts = max(max(lens_of(case)[0]), case["longest"] * 3 // 4), [part.split("*") for part in case["step"].split(",")]
        if longest < case["longest"]:
            case = dict(case, longest=longest)
        elif case["G"] > 1:
            case = dict(case, H=case["H"] // case["G"], G=1)
        else:                                                        # fewer tokens at once
            less = ["%d*%s" % ((int(a) + 1) // 2, n) if int(a) > 16 else "%s*%d" % (a, (int(n) + 1) // 2) for a, n in parts]
            case = dict(case, step=",".join(less), longest=max(lens_of(dict(case, step=",".join(less), longest=0))[0]))
            if ",".join(less) == ",".join("*".join(p) for p in parts):
                break
    return case


# ---- the definition of the cache's numbers -----------------------------------------------------------------------------

def lens_of(case):
    """(tokens each request brings, tokens it holds afterwards)."""
    q = [int(a) for part in case["step"].split(",") for a, n in [part.split("*")] for _ in range(int(n))]
    n = len(q)
    return q, [max(a, case["longest"] if not case["ragged"] or n == 1 else a + (case["longest"] - a) * i // (n - 1)) for i, a in enumerate(q)]


def quantised(x):
    """Codes (int8) and scales (float32) of rows along the last dimension, in 64 bits: a code next to a border is the right one."""
    x = x.double()
    scale = (x.abs().amax(-1).float().double() / 127).float().clamp_min(2.0 ** -126)
    return (x / scale.double()[..., None]).round().to(torch.int8), scale


def record_bytes(bs, d):
    return (2 * bs * d + 8 * bs + 15) // 16 * 16


def packed(k, ks, v, vs):
    """The cache as the framework lays it out, from codes [pages, block, G, d] and scales [pages, block, G]: a record per page and head,
    [pages, G, bytes]: key codes, value codes (a byte is code + 128; the 16-byte pieces of a row stand in an order of their own), key scales,
    value scales."""
    pages, bs, G, d = k.shape
    row = torch.arange(bs, device=k.device)[:, None]
    turn = row & 7 if d % 128 == 0 else (row >> 1) & 3 if d % 64 == 0 else row * 0
    at = torch.arange(d // 16, device=k.device)[None, :] ^ turn                             # where piece c of row r stands; its own inverse
    out = torch.zeros(pages, G, record_bytes(bs, d), dtype=torch.uint8, device=k.device)
    for n, (c, s) in enumerate(((k, ks), (v, vs))):
        b = (c.to(torch.int16) + 128).to(torch.uint8).permute(0, 2, 1, 3).reshape(pages, G, bs, d // 16, 16)
        b = torch.gather(b, 3, at[None, None, :, :, None].expand(pages, G, -1, -1, 16))
        out[..., n * bs * d:(n + 1) * bs * d] = b.reshape(pages, G, bs * d)
        first = 2 * bs * d + 4 * bs * n
        out[..., first:first + 4 * bs] = s.permute(0, 2, 1).contiguous().view(torch.uint8).reshape(pages, G, 4 * bs)
    return out


def rotated(x, table, positions, n_rot, pairing):
    """Rows [T, heads, d] with the first ``n_rot`` of each head turned, in the type of ``x`` and ``table``."""
    if n_rot == 0:
        return x
    cs = table[positions.long()][:, None].to(x.dtype)
    c, s, half = cs[..., 0], cs[..., 1], n_rot // 2
    if pairing == "half":
        a, b = x[..., :half], x[..., half:n_rot]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., n_rot:]], -1)
    a, b = x[..., 0:n_rot:2], x[..., 1:n_rot:2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), x[..., n_rot:]], -1)


# ---- what a program has in hand ------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = SimpleNamespace(case=case, **{k: case[k] for k in ("H", "G", "d", "op")})
    dt, H, G, d = TYPES[case["dtype"]], s.H, s.G, s.d
    randn = lambda *n: torch.randn(*n, generator=g, device=DEVICE)
    q_lens, kv_lens = lens_of(case)
    blocks = [(n + BLOCK - 1) // BLOCK for n in kv_lens]
    spare = 3
    pool = sum(blocks) + spare
    order = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
    s.max_blocks = max(blocks)
    s.block_table = torch.full((len(q_lens), s.max_blocks), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(blocks):
        s.block_table[i, :n] = order[at:at + n]
        at += n
    s.q_lens, s.kv_lens = q_lens, kv_lens
    s.positions = torch.cat([torch.arange(n - q, n, dtype=torch.int32) for q, n in zip(q_lens, kv_lens)]).to(DEVICE)
    s.token_seq = torch.repeat_interleave(torch.arange(len(q_lens), dtype=torch.int32), torch.tensor(q_lens)).to(DEVICE)
    T = s.T = sum(q_lens)
    # some channels of keys are much larger than the rest, and tokens differ in size, as a model's do
    channel = torch.exp(0.5 * randn(G, d)) * torch.where(torch.rand(G, d, generator=g, device=DEVICE) < 0.03, 6.0, 1.0)
    token = lambda *n: torch.exp(0.4 * randn(*n, 1))
    k = randn(pool, BLOCK, G, d) * channel * token(pool, BLOCK, G)
    v = randn(pool, BLOCK, G, d) * token(pool, BLOCK, G)
    (s.k, s.ks), (s.v, s.vs) = quantised(k.to(dt)), quantised(v.to(dt))
    s.cache = packed(s.k, s.ks, s.v, s.vs)
    del k, v
    if s.op == "read":
        s.pages = order[:sum(blocks)].contiguous()
        s.rows = torch.cat([(n - BLOCK * torch.arange(b)).clamp(max=BLOCK) for n, b in zip(kv_lens, blocks)]).to(torch.int32).to(DEVICE)
        s.k_out, s.v_out = (torch.empty(len(s.pages), BLOCK, G, d, dtype=dt, device=DEVICE) for _ in range(2))
    elif s.op == "store":
        s.qkv = torch.cat([randn(T, H, d), randn(T, G, d) * channel, randn(T, G, d)], 1)
        s.qkv = (s.qkv * torch.exp(0.4 * randn(T, H + 2 * G, 1))).reshape(T, -1).to(dt)
        blk = s.positions // BLOCK
        s.slots = (s.block_table[s.token_seq.long(), blk.long()] * BLOCK + s.positions % BLOCK).to(torch.int32)
        n_rot, most = case["n_rot"], max(kv_lens)
        s.table = None
        if n_rot:
            f = 1e6 ** (-torch.arange(0, n_rot, 2, dtype=torch.float64, device=DEVICE) / n_rot)
            angle = torch.arange(most, dtype=torch.float64, device=DEVICE)[:, None] * f
            s.table = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        s.q_out = torch.empty(T, H * d, dtype=dt, device=DEVICE)
        # the pages that the step writes to, and how many of their rows are in use
        touched = [(i, b) for i, (q, n) in enumerate(zip(q_lens, kv_lens)) for b in range((n - q) // BLOCK, blocks[i])]
        i, b = (torch.tensor(x, device=DEVICE) for x in zip(*touched))
        s.pages = s.block_table[i, b].contiguous()
        s.rows = (torch.tensor(kv_lens, device=DEVICE)[i] - BLOCK * b).clamp(max=BLOCK).to(torch.int32)
        s.k_out, s.v_out = (torch.empty(len(s.pages), BLOCK, G, d, dtype=dt, device=DEVICE) for _ in range(2))
    else:
        s.q = (randn(T, H, d) * torch.exp(0.3 * randn(T, H, 1)) / channel.repeat_interleave(H // G, 0).clamp_min(1.0)).reshape(T, H * d).to(dt)
        s.out = torch.empty_like(s.q)
        s.scale = 1.0 / math.sqrt(d)
        s.sinks = randn(H) if case["sinks"] else None
        s.slopes = torch.pow(2.0, -4.0 * torch.arange(1, H + 1, device=DEVICE) / H) * 0.1 if case["slopes"] else None
    if own and s.op == "attend":
        # the plan that a program makes once a step for all of its layers
        from hfcpu_b200 import kernels
        s.tiles = {n: torch.from_numpy(a).to(DEVICE) for n, a in kernels.kv8_step_arrays(q_lens, H // G).items()}
        s.meta = SimpleNamespace(block_table=s.block_table, block_size=BLOCK, max_blocks=s.max_blocks)
        bufs = {}

        def buf(name, shape, dtype):
            key = (name, tuple(shape), dtype)
            if key not in bufs:
                bufs[key] = torch.empty(shape, dtype=dtype, device=DEVICE)
            return bufs[key]
        s.ctx = SimpleNamespace(positions=s.positions, token_seq=s.token_seq, max_q_len=max(q_lens), max_kv_len=max(kv_lens), buf=buf)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        from hfcpu_b200 import kernels
        c = s.case
        if s.op == "attend":
            kernels.paged_attention_kv8(s.q, s.cache, s.meta, s.ctx, s.H, s.G, s.d, c["window"], s.scale, s.out, tiles=s.tiles, sinks=s.sinks,
                                        slopes=s.slopes, softcap=c["cap"])
            return s.out
        if s.op == "store":
            kernels.rope_kv8_write(s.qkv, s.table, c["n_rot"], s.positions, s.slots, s.q_out, s.cache, s.H, s.G, s.d, BLOCK, pairing=c["pairing"])
        kernels.kv8_read(s.cache, s.pages, s.rows, s.k_out, s.v_out)
        return {"k": s.k_out, "v": s.v_out} if s.op == "read" else {"q": s.q_out, "k": s.k_out, "v": s.v_out}
    return {"attend": plain_attend, "store": plain_store, "read": plain_read}[s.op](s)


def plain_read(s):
    used = (torch.arange(BLOCK, device=DEVICE)[None] < s.rows[:, None])[..., None]
    at = s.pages.long()
    values = lambda codes, scales: (codes[at].float() * (scales[at] * used)[..., None]).to(s.k_out.dtype)
    return {"k": values(s.k, s.ks), "v": values(s.v, s.vs)}


def plain_store(s):
    T, H, G, d, c = s.T, s.H, s.G, s.d, s.case
    x = s.qkv.double().view(T, H + 2 * G, d)
    turned = rotated(x[:, :H + G], s.table, s.positions, c["n_rot"], c["pairing"])
    page, row = (s.slots // BLOCK).long(), (s.slots % BLOCK).long()
    s.k[page, row], s.ks[page, row] = quantised(turned[:, H:])
    s.v[page, row], s.vs[page, row] = quantised(x[:, H + G:])
    return {"q": turned[:, :H].reshape(T, H * d).to(s.qkv.dtype), **plain_read(s)}


def plain_attend(s):
    H, G, d, c = s.H, s.G, s.d, s.case
    S, Q, r = len(s.q_lens), max(s.q_lens), H // G
    # every request's queries and keys side by side, filled up to the longest
    first = torch.tensor([0] + s.q_lens[:-1], device=DEVICE).cumsum(0)
    at = s.token_seq.long() * Q + (torch.arange(s.T, device=DEVICE) - first[s.token_seq.long()])
    q = torch.zeros(S * Q, H * d, device=DEVICE).index_copy(0, at, s.q.float()).view(S, Q, G, r, d)
    pos = torch.full((S * Q,), -1, dtype=torch.int64, device=DEVICE).index_copy(0, at, s.positions.long()).view(S, 1, 1, Q, 1)
    table = s.block_table.clamp_min(0).long()
    L = s.max_blocks * BLOCK
    k = (s.k[table].float() * s.ks[table][..., None]).view(S, L, G, d)
    a = torch.einsum("sqgrd,skgd->sgrqk", q, k) * s.scale
    del k
    if c["cap"]:
        a = c["cap"] * torch.tanh(a / c["cap"])
    key = torch.arange(L, device=DEVICE)
    if s.slopes is not None:
        a = a - s.slopes.view(1, G, r, 1, 1) * (pos - key)
    seen = (key <= pos) & (key > pos - c["window"] if c["window"] else key >= 0)
    a = a.masked_fill(~seen, -math.inf)
    top = a.amax(-1, keepdim=True)
    if s.sinks is not None:
        top = torch.maximum(top, s.sinks.view(1, G, r, 1, 1))
    top = top.masked_fill(top == -math.inf, 0.0)
    a = torch.exp(a - top)
    total = a.sum(-1)
    if s.sinks is not None:
        total = total + torch.exp(s.sinks.view(1, G, r, 1) - top[..., 0])
    v = (s.v[table].float() * s.vs[table][..., None]).view(S, L, G, d)
    o = torch.einsum("sgrqk,skgd->sgrqd", a, v) / total.masked_fill(total == 0, 1.0)[..., None]
    return o.permute(0, 3, 1, 2, 4).reshape(S * Q, H * d)[at].to(s.q.dtype)


def seen_keys(case):
    """(keys that some query of a request sees, pairs of a query and a key it sees), over all requests."""
    w, keys, pairs = case.get("window", 0), 0, 0
    for q, n in zip(*lens_of(case)):
        first = n - q
        keys += n - max(0, first - w + 1) if w else n
        full = max(0, min(q, n - max(first, w))) if w else 0         # queries that see a whole window
        part = q - full
        pairs += full * w + part * first + part * (part + 1) // 2
    return keys, pairs


def work(case):
    H, G, d, e = case["H"], case["G"], case["d"], 2 if case["dtype"] == "bf16" else 4
    q_lens, kv_lens = lens_of(case)
    T, held = sum(q_lens), G * (2 * d + 8)                           # bytes of a token in the cache
    if case["op"] == "attend":
        keys, pairs = seen_keys(case)
        return {"bytes": 2 * T * H * d * e + keys * held + 4 * sum(-(-n // BLOCK) for n in kv_lens) + 4 * T, "flops": 4 * H * d * pairs}
    if case["op"] == "read":
        keys = sum(kv_lens)
        out = sum(-(-n // BLOCK) for n in kv_lens) * BLOCK
        return {"bytes": keys * held + out * G * 2 * d * e, "flops": keys * G * 2 * d}
    back = [(n - (n - q) // BLOCK * BLOCK, -(-n // BLOCK) - (n - q) // BLOCK) for q, n in zip(q_lens, kv_lens)]
    rows, pages = sum(a for a, _ in back), sum(b for _, b in back)
    return {"bytes": T * (2 * H + 2 * G) * d * e + T * held + 4 * T * case["n_rot"] + 8 * T + rows * held + pages * BLOCK * G * 2 * d * e,
            "flops": 3 * T * (H + G) * case["n_rot"] + 2 * rows * G * d}


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    H, G, d, B = s.H, s.G, s.d, BLOCK
    k, v = s.k.double() * s.ks.double()[..., None], s.v.double() * s.vs.double()[..., None]
    if s.op != "attend":
        out = {}
        if s.op == "store":
            x = s.qkv.double().view(s.T, H + 2 * G, d).clone()
            n = case["n_rot"]
            pairs = [(i, i + n // 2) if case["pairing"] == "half" else (2 * i, 2 * i + 1) for i in range(n // 2)]
            for i, (a, b) in enumerate(pairs):
                c, sn = (s.table[s.positions.long(), i, j].double()[:, None] for j in (0, 1))
                x[:, :H + G, a], x[:, :H + G, b] = x[:, :H + G, a] * c - x[:, :H + G, b] * sn, x[:, :H + G, a] * sn + x[:, :H + G, b] * c
            out["q"] = x[:, :H].reshape(s.T, H * d)
            for held, new in ((k, x[:, H:H + G]), (v, x[:, H + G:])):
                unit = (new.abs().max(-1, keepdim=True).values.float().double() / 127).float().double().clamp_min(2.0 ** -126)
                held.view(-1, G, d)[s.slots.long()] = torch.round(new / unit) * unit
        k, v = k[s.pages.long()], v[s.pages.long()]
        for p in range(B):
            k[s.rows <= p, p], v[s.rows <= p, p] = 0.0, 0.0
        return {**out, "k": k, "v": v}
    out, t = torch.zeros(s.T, H, d, dtype=torch.float64, device=DEVICE), 0
    for i, (n_q, n_kv) in enumerate(zip(s.q_lens, s.kv_lens)):
        pages = s.block_table[i, :-(-n_kv // B)].long()
        for t0 in range(t, t + n_q, 256):
            t1 = min(t + n_q, t0 + 256)
            pos = s.positions[t0:t1].long()[:, None]
            first = max(0, int(pos[0]) - case["window"] + 1) if case["window"] else 0
            last = int(pos[-1])
            key = torch.arange(first, last + 1, device=DEVICE)
            for g in range(G):
                ki, vi = (x[pages, :, g].reshape(-1, d)[first:last + 1] for x in (k, v))
                for h in range(g * (H // G), (g + 1) * (H // G)):
                    a = s.q.view(s.T, H, d)[t0:t1, h].double() @ ki.T * s.scale
                    if case["cap"]:
                        a = case["cap"] * torch.tanh(a / case["cap"])
                    if s.slopes is not None:
                        a = a - s.slopes[h].double() * (pos - key)
                    hidden = (key > pos) | ((key <= pos - case["window"]) if case["window"] else (key < 0))
                    a = a.masked_fill(hidden, -math.inf)
                    if s.sinks is not None:
                        a = torch.cat([a, s.sinks[h].double().expand(t1 - t0, 1)], 1)
                    p = torch.softmax(a, -1)[:, :last + 1 - first]
                    out[t0:t1, h] = p @ vi
        t += n_q
    return out.reshape(s.T, H * d)
