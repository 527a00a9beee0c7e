"""The cache in 8 bits on the GPU: each operator against 64 bits, together, and in the engine.

Where the tolerances come from.  Codes and scales are those of the definition, bit for bit.  A value read back is one product of two
float32 numbers (half a step of float32, 2^-24) rounded once to the output's type (bfloat16: 2^-8).  Attention in bfloat16: the output's
rounding, 2^-8 of its size; a weight's rounding to float16, 2^-11 of sum p |v|; and scores that are off by e shift weights by up to 2 e
relative to each other, in numerator and denominator: 4 e sum p |v|.  e: a sum of up to 256 products in float32, each at most |q| 255 scale:
256 * 2^-24 = 2^-16 of the largest such sum, and 2^-20 for exponentials, a cap's tanh (a few 1e-7 of the cap) and a bias's product.
A weight is held in float16 as 2^10 times its share of the reference, and float16's smallest step is 2^-24: a weight that is tiny beside
the others' is off by 2^-25 2^-10 = 2^-35 of the largest scale, which n keys with codes up to 127 can add up to 2^-35 n 127 max(scale) (the
sum of the weights is one at least).  (The first run of these tests came without this term: one output in 476,672, of 4e-10 beside
values of one, was off by a twentieth.)
In float32: 2^-24 of the output's size twice, sums of n weights in the order of the keys, n 2^-24 of sum p |v| (warps of n / 8 and their
merge), and the same e.
"""
import math
from types import SimpleNamespace

import pytest
import torch

from kv8_util import EmuKv8, attention, pack, quantised, rotated, unpack, values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def native():
    from hfcpu_b200 import kernels
    return kernels


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def context(buffers=None):
    bufs = {} if buffers is None else buffers

    def buf(name, shape, dtype):
        key = (name, dtype)
        n = math.prod(shape)
        if key not in bufs or bufs[key].numel() < n:
            bufs[key] = torch.empty(n, dtype=dtype, device=DEV)
        return bufs[key][:n].view(*shape)
    return buf


def step(q_lens, kv_lens, bs, G, d, seed=0, spare=2, size=None, scramble=True):
    """A cache with random rows (and rows of stale requests behind the last), the step's index arrays, and queries' places."""
    g = gen(seed)
    blocks = [-(-n // bs) for n in kv_lens]
    pool = sum(blocks) + spare
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(q_lens), max(blocks)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
    x = torch.randn(2, pool, bs, G, d, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(2, pool, bs, G, 1, generator=g, device=DEV))
    if size is not None:
        x *= size
    (k, ks), (v, vs) = quantised(x[0]), quantised(x[1])
    positions = torch.cat([torch.arange(n - q, n) for q, n in zip(q_lens, kv_lens)]).to(torch.int32).to(DEV)
    seq = torch.repeat_interleave(torch.arange(len(q_lens)), torch.tensor(q_lens)).to(torch.int32).to(DEV)
    return SimpleNamespace(k=k, ks=ks, v=v, vs=vs, table=table, positions=positions, seq=seq, q_lens=list(q_lens), kv_lens=list(kv_lens), bs=bs, G=G, d=d,
                           T=sum(q_lens), blocks=blocks, g=g)


def attend(s, q, cache, H, mask=0, tiles=True, settled=False, buf=None, out=None, plan=None, scale=None, **options):
    K = native()
    meta = SimpleNamespace(block_table=s.table, block_size=s.bs, max_blocks=s.table.shape[1])
    ctx = SimpleNamespace(positions=s.positions, token_seq=s.seq, max_q_len=max(s.q_lens), max_kv_len=max(s.kv_lens), buf=buf or context())
    if plan is None and tiles:
        plan = {n: torch.from_numpy(a).to(DEV) for n, a in K.kv8_step_arrays(s.q_lens, H // s.G).items()}
    out = torch.full_like(q, 7.0) if out is None else out
    K.paged_attention_kv8(q, cache, meta, ctx, H, s.G, s.d, mask, 1 / math.sqrt(s.d) if scale is None else scale, out, tiles=plan if tiles else None,
                          settled=settled, **options)
    return out


def check(s, q, cache, got, H, mask=0, scale=None, rows=None, **options):
    scale = 1 / math.sqrt(s.d) if scale is None else scale
    ref, size, worst, far = attention(q, cache, s.table, s.seq, s.positions, s.bs, H, s.G, s.d, mask, scale, **options)
    got = got.double().view(ref.shape)
    hs = options.get("head_scales")
    worst *= float(hs.abs().max()) if hs is not None else 1.0
    e = 2.0 ** -16 * worst + 2.0 ** -20 * (options.get("softcap", 0.0) + worst + (float(options["slopes"].abs().max()) * max(s.kv_lens) if options.get("slopes") is not None else 0))
    if q.dtype == torch.bfloat16:
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -11 + 4 * e) * size + 2.0 ** -35 * far
    else:
        tol = 2.0 ** -23 * ref.abs() + (max(s.kv_lens) * 2.0 ** -24 + 4 * e) * size
    bad = ~((got - ref).abs() <= tol + 1e-30)
    if rows is not None:
        bad = bad[rows]
    assert not bad.any(), (int(bad.sum()), float(((got - ref).abs() / (tol + 1e-30)).nan_to_num(1e9).max()))


# ---- write -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,H,G,d,n_rot,bs,pairing", [
    (1, 14, 2, 64, 64, 16, "half"), (33, 28, 4, 128, 128, 16, "half"), (65, 8, 8, 80, 32, 5, "interleaved"), (7, 6, 3, 16, 16, 1, "half"),
    (40, 4, 4, 256, 128, 64, "interleaved"), (129, 3, 1, 192, 24, 8, "half"), (12, 5, 5, 96, 0, 32, "half"), (9, 2, 2, 48, 6, 3, "interleaved"),
    (31, 4, 2, 112, 10, 128, "half"), (300, 16, 4, 128, 64, 16, "interleaved")])
def test_write_rows_are_the_definitions(T, H, G, d, n_rot, bs, pairing, dtype):
    K, dt, g = native(), DT[dtype], gen(T * d + n_rot)
    pages = T // bs + 5
    wide = (torch.randn(T, (H + 2 * G) * d + 16, generator=g, device=DEV) * torch.exp(torch.randn(T, 1, generator=g, device=DEV) * 3)).to(dt)
    qkv = wide[:, 8:8 + (H + 2 * G) * d] if d % 32 == 0 else wide[:, 3:3 + (H + 2 * G) * d]         # a slice of wider rows, aligned or not
    ang = torch.arange(500, dtype=torch.float64, device=DEV)[:, None] * 10 ** (-torch.arange(n_rot // 2, dtype=torch.float64, device=DEV) / 4)
    table = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    pos = torch.randint(0, 500, (T,), generator=g, device=DEV, dtype=torch.int32)
    slots = torch.randperm(pages * bs, generator=g, device=DEV)[:T].to(torch.int32)
    slots[T // 3] = -1
    before = torch.randint(0, 256, K.kv8_cache(pages, bs, G, d, DEV).shape, generator=g, device=DEV, dtype=torch.uint8)
    cache, q_out = before.clone(), torch.empty(T, H * d, device=DEV, dtype=dt)
    K.rope_kv8_write(qkv, table if n_rot else None, n_rot, pos, slots, q_out, cache, H, G, d, bs, pairing=pairing)
    x = qkv.double().reshape(T, H + 2 * G, d)
    x = torch.cat([rotated(x[:, :H + G], table, pos, n_rot, pairing), x[:, H + G:]], 1)
    # q: two products and a sum in float32 (3 * 2^-24 of their sizes), rounded to the type
    step = torch.finfo(dt).eps / 2
    assert ((q_out.double().view(T, H, d) - x[:, :H]).abs() <= step * x[:, :H].abs() + 2.0 ** -22 * x[:, :H].abs().amax(-1, keepdim=True)).all()
    kc, ks, vc, vs = (y.clone() for y in unpack(before, bs, G, d))
    ok = slots >= 0
    page, row = slots[ok].long() // bs, slots[ok].long() % bs
    kc[page, row], ks[page, row] = (y[ok] for y in quantised(x[:, H:H + G]))
    vc[page, row], vs[page, row] = (y[ok] for y in quantised(x[:, H + G:]))
    want = before.clone()
    want[..., :2 * bs * d + 8 * bs] = pack(kc, ks, vc, vs)[..., :2 * bs * d + 8 * bs]
    assert torch.equal(cache, want)                                   # ... and every other byte is as it was


def test_write_rows_next_to_borders_and_extremes():
    """Values on and beside the halves between two codes, tiny rows, rows of zeros, rows that are no numbers."""
    K, d, G, bs = native(), 128, 1, 16
    rows = []
    for top in (127.0, 254.0, 1.984375, 127.0 * 2.0 ** -20):
        unit = top / 127
        x = (torch.arange(d, device=DEV, dtype=torch.float64) - 64 + 0.5) * unit
        rows += [x, torch.nextafter(x.float(), torch.full((), 1e9, device=DEV)).double(), torch.nextafter(x.float(), torch.full((), -1e9, device=DEV)).double()]
        for r in rows[-3:]:
            r[0] = top
    rows += [torch.zeros(d, device=DEV), torch.full((d,), 1e-45, device=DEV), torch.full((d,), 3e38, device=DEV), torch.full((d,), -2.0 ** -126, device=DEV)]
    bad = torch.ones(3, d, device=DEV)
    bad[0, 5], bad[1, 127], bad[2, 0] = math.inf, math.nan, -math.inf
    k = torch.stack([r.float() for r in rows] + list(bad))
    T = len(k)
    cache = K.kv8_cache(4, bs, G, d, DEV)
    K.kv8_write(k, k.flip(0).contiguous(), torch.arange(T, device=DEV, dtype=torch.int32), cache, G, d, bs)
    kc, ks, vc, vs = (x.flatten(0, 1)[:T, 0] for x in unpack(cache, bs, G, d))
    c, s = quantised(k)
    assert torch.equal(kc, c) and torch.equal(vc, c.flip(0))
    assert torch.equal(ks.nan_to_num(-1), s.nan_to_num(-1)) and torch.equal(vs.nan_to_num(-1), s.flip(0).nan_to_num(-1))
    assert torch.isnan(ks[-3:]).all()
    out = torch.empty(4, bs, G, d, device=DEV), torch.empty(4, bs, G, d, device=DEV)
    K.kv8_read(cache, torch.arange(4, device=DEV, dtype=torch.int32), torch.full((4,), bs, device=DEV, dtype=torch.int32), *out)
    assert torch.isnan(out[0].flatten(0, 1)[T - 3:T]).all() and not torch.isnan(out[0].flatten(0, 1)[:T - 3]).any()


def test_write_reports_slots_and_positions_outside():
    K = native()
    K.check_device_errors()
    cache, q = K.kv8_cache(2, 16, 1, 64, DEV), torch.empty(2, 64, device=DEV, dtype=torch.bfloat16)
    qkv, table = torch.ones(2, 192, device=DEV, dtype=torch.bfloat16), torch.ones(8, 32, 2, device=DEV)
    i = lambda *x: torch.tensor(x, device=DEV, dtype=torch.int32)
    for pos, slots in ((i(0, 8), i(0, 1)), (i(0, -1), i(0, 1)), (i(0, 1), i(0, 32))):
        K.rope_kv8_write(qkv, table, 64, pos, slots, q, cache, 1, 1, 64, 16)
        with pytest.raises(K.DeviceFault):
            K.check_device_errors()
    K.check_device_errors()
    from hfcpu_b200.kernels.native import KernelError
    with pytest.raises(KernelError):                     # a tensor of the host
        K.rope_kv8_write(qkv, table, 64, i(0, 1).cpu(), i(0, 1), q, cache, 1, 1, 64, 16)


def test_queries_alone_are_turned():
    K = native()
    qkv, table = torch.randn(5, 256, device=DEV, generator=gen(1)).bfloat16(), torch.randn(8, 32, 2, device=DEV, generator=gen(2))
    pos = torch.arange(5, device=DEV, dtype=torch.int32)
    cache, q, q2 = K.kv8_cache(1, 16, 1, 64, DEV), torch.empty(5, 128, device=DEV).bfloat16(), torch.empty(5, 128, device=DEV).bfloat16()
    K.rope_kv8_write(qkv, table, 64, pos, None, q, cache, 2, 1, 64, 16)
    assert not cache.any()
    K.rope_kv8_write(qkv, table, 64, pos, pos, q2, cache, 2, 1, 64, 16)
    assert torch.equal(q, q2) and cache.any()


# ---- read ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bs,G,d", [(16, 2, 64), (1, 3, 16), (5, 8, 80), (64, 1, 256), (16, 4, 128), (128, 2, 192), (8, 1, 48)])
def test_read_gives_the_values_codes_stand_for(bs, G, d, dtype):
    K, dt = native(), DT[dtype]
    s = step([1], [bs * 11], bs, G, d, seed=bs + d)
    s.ks[3, bs // 2] = math.nan
    cache = pack(s.k, s.ks, s.v, s.vs)
    pages = torch.tensor([4, 0, -1, 4, 12, 3, 7, 7], device=DEV, dtype=torch.int32)                  # in any order, some twice, one that is none
    rows = torch.tensor([bs, 0, bs, bs // 2, bs, bs // 2, bs, (bs + 1) // 2], device=DEV, dtype=torch.int32)
    k, v = (torch.full((8, bs, G, d), 5.0, device=DEV, dtype=dt) for _ in range(2))
    K.kv8_read(cache, pages, rows, k, v)
    used = (torch.arange(bs, device=DEV)[None] < rows[:, None]) & (pages >= 0)[:, None]
    for got, codes, scales in ((k, s.k, s.ks), (v, s.v, s.vs)):
        want = torch.where(used[..., None, None], (codes[pages.long().clamp_min(0)].float() * scales[pages.long().clamp_min(0)][..., None]).to(dt),
                           torch.zeros((), device=DEV, dtype=dt))
        assert torch.equal(got.nan_to_num(-3), want.nan_to_num(-3)) and not torch.isnan(got).any()
    K.check_device_errors()
    K.kv8_read(cache, pages + 1000, rows, k, v)
    assert not k.any() and not v.any()
    with pytest.raises(K.DeviceFault):
        K.check_device_errors()


# ---- attention -------------------------------------------------------------------------------------------------------------

SHAPES = [                                                   # H, G, d, block
    (14, 2, 64, 16), (28, 4, 128, 16), (32, 8, 128, 16), (4, 4, 64, 8), (8, 1, 128, 32), (12, 1, 64, 64), (17, 1, 64, 16), (40, 2, 128, 8), (64, 2, 64, 32),
    (4, 2, 128, 64), (3, 1, 128, 16)]
OTHER = [(6, 3, 16, 4), (8, 2, 80, 16), (4, 1, 256, 16), (6, 2, 32, 5), (5, 5, 192, 128), (4, 2, 64, 1), (4, 2, 128, 128)]
STEPS = {                                                    # what requests bring, what they hold afterwards
    "single": ([1], [1]), "one": ([1], [700]), "many": ([1] * 9, [1, 2, 63, 64, 65, 127, 128, 129, 900]), "few": ([5, 2, 16, 1, 3], [5, 300, 17, 64, 130]),
    "portion": ([70], [70]), "behind": ([100, 33], [420, 700]), "mixed": ([1, 90, 1, 3, 130, 1], [500, 90, 1, 260, 300, 64])}


@pytest.fixture(autouse=True)
def prompts_kernel_for_small_steps(monkeypatch):
    """Lets small portions reach the kernel for prompts, which otherwise waits for rows enough."""
    monkeypatch.setattr(native(), "KV8_MANY_ROWS", 64)


@pytest.mark.parametrize("name", list(STEPS))
@pytest.mark.parametrize("shape", SHAPES + OTHER, ids=str)
def test_attention(shape, name):
    H, G, d, bs = shape
    s = step(*STEPS[name], bs, G, d, seed=H + d)
    cache = pack(s.k, s.ks, s.v, s.vs)
    q = (torch.randn(s.T, H * d, generator=s.g, device=DEV) * 2).bfloat16()
    got = attend(s, q, cache, H)
    check(s, q, cache, got, H)
    assert torch.equal(got, attend(s, q, cache, H, settled=True))          # whatever came in front, and the same bits again


@pytest.mark.parametrize("shape", [(8, 2, 80, 16), (6, 3, 64, 16), (4, 1, 128, 8), (2, 2, 256, 5)], ids=str)
def test_attention_in_float32(shape):
    H, G, d, bs = shape
    for name in ("many", "few", "mixed"):
        s = step(*STEPS[name], bs, G, d, seed=H + d)
        cache = pack(s.k, s.ks, s.v, s.vs)
        q = torch.randn(s.T, H * d, generator=s.g, device=DEV)
        check(s, q, cache, attend(s, q, cache, H), H)


@pytest.mark.parametrize("mask", [1, 2, 50, 64, 200, -1, -7, -64, -100])
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (8, 2, 128, 8), (8, 2, 80, 16)], ids=str)
def test_masks(shape, mask):
    H, G, d, bs = shape
    for name in ("many", "mixed"):
        s = step(*STEPS[name], bs, G, d, seed=mask + 1000)
        # pages that the mask has passed are gone, as the cache's manager gives them back
        for i, (n_q, n) in enumerate(zip(s.q_lens, s.kv_lens)):
            p = n - n_q
            s.table[i, :(max(0, p - mask + 1) if mask > 0 else p // -mask * -mask) // bs] = -1
        cache = pack(s.k, s.ks, s.v, s.vs)
        q = torch.randn(s.T, H * d, generator=s.g, device=DEV).bfloat16()
        check(s, q, cache, attend(s, q, cache, H, mask=mask), H, mask=mask)
        native().check_device_errors()


@pytest.mark.parametrize("which", ["sinks", "zero_sink", "slopes", "head_scales", "softcap", "all"])
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (28, 4, 128, 16), (24, 2, 64, 8), (8, 2, 80, 16)], ids=str)
def test_options(shape, which):
    H, G, d, bs = shape
    r = lambda: torch.randn(H, device=DEV, generator=gen(H))
    o = {"sinks": dict(sinks=r() * 3), "zero_sink": dict(zero_sink=True), "slopes": dict(slopes=r().abs() * 0.05), "head_scales": dict(head_scales=r()),
         "softcap": dict(softcap=2.0), "all": dict(sinks=r() - 40, slopes=r() * 0.02, head_scales=r(), softcap=20.0)}[which]
    for name, mask in (("many", 0), ("mixed", 70), ("behind", 0)):
        s = step(*STEPS[name], bs, G, d, seed=5)
        cache = pack(s.k, s.ks, s.v, s.vs)
        q = (torch.randn(s.T, H * d, generator=s.g, device=DEV) * 2).bfloat16()
        check(s, q, cache, attend(s, q, cache, H, mask=mask, **o), H, mask=mask, **o)


@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (8, 2, 128, 16), (8, 2, 80, 16)], ids=str)
def test_rows_that_are_no_numbers_where_nothing_is_seen(shape):
    """Rows behind a request's last, rows that a window has passed, later tokens of the same portion, pages of nobody: whatever they hold."""
    H, G, d, bs = shape
    for name, mask in (("many", 0), ("few", 0), ("mixed", 40), ("behind", 0)):
        s = step(*STEPS[name], bs, G, d, seed=8)
        q = torch.randn(s.T, H * d, generator=s.g, device=DEV).bfloat16()
        clean = pack(s.k, s.ks, s.v, s.vs)
        seen = torch.zeros(s.ks.shape[:2], dtype=torch.bool, device=DEV)
        for i, (n_q, n) in enumerate(zip(s.q_lens, s.kv_lens)):
            for p in range(max(0, n - n_q - mask + 1) if mask else 0, n):
                seen[s.table[i, p // bs], p % bs] = True
        for x in (s.ks, s.vs):
            x[~seen] = math.nan
        s.k[~seen] = -128
        cache = pack(s.k, s.ks, s.v, s.vs)
        assert torch.equal(attend(s, q, cache, H, mask=mask), attend(s, q, clean, H, mask=mask))
        # the last token's row: only that token sees it
        s2 = step(*STEPS[name], bs, G, d, seed=8)
        n = s2.kv_lens[0]
        page, row = int(s2.table[0, (n - 1) // bs]), (n - 1) % bs
        for x in (s2.ks, s2.vs):
            x[page, row] = math.nan
        got = attend(s2, q, pack(s2.k, s2.ks, s2.v, s2.vs), H, mask=mask)
        last = sum(s.q_lens[:1]) - 1
        assert torch.isnan(got[last]).all()
        # (what a tile's other tokens see may be rounded relative to another scale)
        check(s, q, clean, got, H, mask=mask, rows=torch.arange(s.T, device=DEV) != last)


@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (4, 2, 128, 64), (8, 2, 80, 16)], ids=str)
def test_pages_that_are_not_there(shape):
    """An entry that names no page raises the error word; its keys count for nothing."""
    K = native()
    H, G, d, bs = shape
    for name in ("many", "behind"):
        s = step(*STEPS[name], bs, G, d, seed=9)
        cache = pack(s.k, s.ks, s.v, s.vs)
        i = len(s.q_lens) - 1
        s.table[i, 1] = -1
        s.table[i, 2] = 1 << 20
        q = torch.randn(s.T, H * d, generator=s.g, device=DEV).bfloat16()
        K.check_device_errors()
        got = attend(s, q, cache, H)
        with pytest.raises(K.DeviceFault):
            K.check_device_errors()
        s.table[i, 1:3] = 0
        check(s, q, cache, got, H, missing=[(i, 1), (i, 2)])


@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (8, 2, 128, 16), (8, 2, 80, 16)], ids=str)
def test_sizes_far_apart(shape):
    """Keys, values and queries of very different sizes beside each other, rows of zeros, a key that stands out."""
    H, G, d, bs = shape
    for seed, name in enumerate(("many", "mixed", "few")):
        s = step(*STEPS[name], bs, G, d, seed=seed)
        pick = torch.randint(0, 6, s.ks.shape, generator=s.g, device=DEV)
        s.vs *= torch.tensor([1.0, 1e-4, 1e3, 1.0, 1e-9, 1.0], device=DEV)[pick]
        s.ks *= torch.tensor([1.0, 1e-3, 0.0, 4.0, 1.0, 1e-6], device=DEV)[pick]
        s.v[pick == 3] = 0
        s.vs[pick == 3] = 2.0 ** -126
        s.ks.clamp_(min=2.0 ** -126)
        cache = pack(s.k, s.ks, s.v, s.vs)
        q = (torch.randn(s.T, H, d, generator=s.g, device=DEV) * 10.0 ** torch.randint(-6, 2, (s.T, H, 1), generator=s.g, device=DEV)).bfloat16().view(s.T, H * d)
        q[0] = 0
        check(s, q, cache, attend(s, q, cache, H), H)
    # the largest and smallest queries that bfloat16 has, with a factor that brings the scores back
    for by in (2.0 ** 100, 2.0 ** -110):
        s = step(*STEPS["mixed"], bs, G, d, seed=3)
        cache = pack(s.k, s.ks, s.v, s.vs)
        q = (torch.randn(s.T, H * d, generator=s.g, device=DEV) * by).bfloat16()
        check(s, q, cache, attend(s, q, cache, H, scale=0.1 / by), H, scale=0.1 / by)


def test_a_row_of_values_of_zeros_still_counts():
    for d in (64, 128, 80):
        s = step([1, 40], [50, 40], 16, 1, d, seed=4)
        s.v[:] = 0
        s.vs[:] = 2.0 ** -126
        q = torch.randn(41, 4 * d, generator=s.g, device=DEV).bfloat16()
        assert not attend(s, q, pack(s.k, s.ks, s.v, s.vs), 4).any()
        page = int(s.table[0, 0])
        s.v[page, 3], s.vs[page, 3] = 100, 0.25
        cache = pack(s.k, s.ks, s.v, s.vs)
        check(s, q, cache, attend(s, q, cache, 4), 4)


def test_tokens_without_a_position_read_nothing():
    for d in (64, 128, 80):
        s = step([1, 1, 1], [40, 50, 60], 16, 2, d, seed=6)
        s.positions[1] = -1
        q = torch.randn(3, 8 * d, generator=s.g, device=DEV).bfloat16()
        got = attend(s, q, pack(s.k, s.ks, s.v, s.vs), 8)
        assert not got[1].any() and got[0].any() and got[2].any()


def test_a_long_request_and_many_tiles():
    """Ranges over many CTAs; more tiles than one launch takes."""
    s = step([1, 3], [40000, 9000], 16, 1, 64, seed=2)
    cache = pack(s.k, s.ks, s.v, s.vs)
    q = torch.randn(4, 8 * 64, generator=s.g, device=DEV).bfloat16()
    check(s, q, cache, attend(s, q, cache, 8), 8)
    n = 2300
    s = step([1] * n, [1 + i % 70 for i in range(n)], 16, 1, 64, seed=3)
    cache = pack(s.k, s.ks, s.v, s.vs)
    q = torch.randn(n, 2 * 64, generator=s.g, device=DEV).bfloat16()
    check(s, q, cache, attend(s, q, cache, 2), 2)


def test_cache_beyond_32_bits():
    """Records behind the first 4 GiB."""
    K = native()
    bs, G, d = 16, 8, 128
    pages = (1 << 32) // (G * K.kv8_record_bytes(bs, d)) + 40
    cache = K.kv8_cache(pages, bs, G, d, DEV)
    T = 96
    far = torch.arange(pages - 10, pages, device=DEV, dtype=torch.int32)
    k, v = (torch.randn(T, G * d, device=DEV, generator=gen(i)).bfloat16() for i in (1, 2))
    slots = (far[torch.arange(T, device=DEV) // bs] * bs + torch.arange(T, device=DEV, dtype=torch.int32) % bs).to(torch.int32)
    K.kv8_write(k, v, slots, cache, G, d, bs)
    small = K.kv8_cache(10, bs, G, d, DEV)
    K.kv8_write(k, v, torch.arange(T, device=DEV, dtype=torch.int32), small, G, d, bs)
    assert torch.equal(cache[-10:], small) and not cache[:-10].any()
    outs = [torch.empty(6, bs, G, d, device=DEV) for _ in range(4)]
    rows = torch.full((6,), bs, device=DEV, dtype=torch.int32)
    K.kv8_read(cache, far[:6].contiguous(), rows, outs[0], outs[1])
    K.kv8_read(small, torch.arange(6, device=DEV, dtype=torch.int32), rows, outs[2], outs[3])
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]) and outs[0].any()
    for q_lens in ([1], [96]):
        s = SimpleNamespace(q_lens=q_lens, kv_lens=[96], bs=bs, G=G, d=d, seq=torch.zeros(q_lens[0], device=DEV, dtype=torch.int32),
                            positions=torch.arange(96 - q_lens[0], 96, device=DEV, dtype=torch.int32))
        q = torch.randn(q_lens[0], 16 * d, device=DEV, generator=gen(3)).bfloat16()
        s.table = far[None, :6].contiguous()
        a = attend(s, q, cache, 16)
        s.table = torch.arange(6, device=DEV, dtype=torch.int32)[None]
        assert torch.equal(a, attend(s, q, small, 16))


@pytest.mark.parametrize("d", [64, 128, 80])
def test_written_read_and_attended_in_one_go_on_another_stream(d):
    """The three together, several times behind one another, on a stream that is not the default one."""
    K, H, G, bs = native(), 8, 2, 16
    n_rot = d if d != 80 else 32
    table = torch.randn(600, n_rot // 2, 2, device=DEV, generator=gen(1))
    cache, side = K.kv8_cache(48, bs, G, d, DEV), torch.cuda.Stream()
    blocks = torch.randperm(48, device=DEV, generator=gen(2))[:40].to(torch.int32)[None].contiguous()
    held, buf = 0, context()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i, n in enumerate((200, 1, 1, 5, 130, 1, 17)):
            pos = torch.arange(held, held + n, device=DEV, dtype=torch.int32)
            qkv = torch.randn(n, (H + 2 * G) * d, device=DEV, generator=gen(10 + i)).bfloat16()
            slots = blocks[0, (pos // bs).long()] * bs + pos % bs
            q = torch.empty(n, H * d, device=DEV).bfloat16()
            K.rope_kv8_write(qkv, table, n_rot, pos, slots, q, cache, H, G, d, bs)
            held += n
            s = SimpleNamespace(q_lens=[n], kv_lens=[held], bs=bs, G=G, d=d, table=blocks, positions=pos, seq=torch.zeros(n, device=DEV, dtype=torch.int32))
            got = attend(s, q, cache, H, buf=buf)
            x = qkv.double().view(n, H + 2 * G, d)
            assert torch.equal(quantised(rotated(x[:, H:H + G], table, pos, n_rot, "half"))[0],
                               unpack(cache, bs, G, d)[0].flatten(0, 1)[slots.long()])
            check(s, q, cache, got, H)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("d", [64, 128, 80])
def test_captured_and_replayed(d):
    """Two graphs of single tokens over the same buffers, replayed in turn beside eager calls, while the requests grow."""
    K, H, G, bs = native(), 8, 2, 16
    s = step([1] * 5, [30, 300, 64, 1, 129], bs, G, d, seed=7, spare=300)
    s.table = torch.cat([s.table, torch.randperm(300, device=DEV, generator=gen(1)).to(torch.int32)[:5 * 40].view(5, 40)], 1)[:, :40].contiguous()
    s.table = torch.randperm(5 * 40, device=DEV, generator=gen(2)).to(torch.int32).view(5, 40)
    cache = pack(s.k[:300], s.ks[:300], s.v[:300], s.vs[:300])
    q, outs, graphs, buf = torch.randn(5, H * d, device=DEV, generator=gen(3)).bfloat16(), [], [], context()
    plan = {n: torch.from_numpy(a).to(DEV) for n, a in K.kv8_step_arrays(s.q_lens, H // G).items()}
    attend(s, q, cache, H, buf=buf, plan=plan)
    for _ in range(2):
        out = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(s, q, cache, H, buf=buf, plan=plan, out=out)
        outs.append(out)
        graphs.append(graph)
    for i in range(6):
        s.positions += torch.tensor([1, 40, 7, 90, 3], device=DEV, dtype=torch.int32)
        s.positions.clamp_(max=639)
        s.kv_lens = [int(x) + 1 for x in s.positions]
        q.copy_(torch.randn(q.shape, device=DEV, generator=gen(20 + i)))
        for o in outs:
            o.zero_()
        graphs[i % 2].replay()
        eager = attend(s, q, cache, H, buf=buf)
        graphs[1 - i % 2].replay()
        check(s, q, cache, outs[0], H)
        assert torch.equal(outs[0], outs[1])
        check(s, q, cache, eager, H)


# ---- in the engine -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_engine_is_as_far_from_the_plain_cache_as_the_definition(tiny_folders, name, dtype):
    """Logits on a cache in 8 bits, however the prompt is cut, graphs and eager.  The stand-in backend in float32 says how far codes take
    them from the float32 cache's (``far``).  Sums in another order flip one code in 10^4 or fewer, which adds the root of that, a
    hundredth of ``far``: a quarter is allowed.  A bfloat16 run adds its own roundings: what they do to the plain cache's logits, twice
    (queries, outputs and keys are rounded at the same places)."""
    from hfcpu_b200.engine import Engine, StepEntry
    from hfcpu_b200.models import load_model
    K = native()
    folder = tiny_folders[name + ("16" if dtype == "bfloat16" else "")]
    prompt = [int(x) for x in torch.randint(0, 500, (150,), generator=torch.Generator().manual_seed(1))]

    def run(engine, cut, decode=6):
        engine.add_request("r")
        at = 0
        for n in cut:
            engine.step([StepEntry("r", prompt[at:at + n], [n - 1])])
            at += n
        out = [engine.step([StepEntry("r", [5 + i], [0])]).clone() for i in range(decode)]
        engine.finish_request("r")
        return torch.cat(out).float()

    def engine_of(dt, kv):
        return Engine(load_model(folder, dt, DEV), block_size=16, max_tokens=512, kv_dtype=kv)
    plain = run(engine_of(torch.float32, "auto"), [150])
    own = float((run(engine_of(DT[dtype], "auto"), [150]) - plain).abs().max())
    real = K.backend()
    try:
        K.set_backend(EmuKv8())
        eng = engine_of(torch.float32, "int8")
        eng.use_graphs = False
        emu = run(eng, [150])
    finally:
        K.set_backend(real)
    far = float((emu - plain).abs().max())
    engine = engine_of(DT[dtype], "int8")
    for cut in ([150], [64, 70, 16], [1, 5, 144]):
        got = run(engine, cut)
        assert float((got - emu).abs().max()) <= (0.25 * far + 1e-4 if dtype == "float32" else far + 2 * own), cut
        assert not torch.equal(got, plain)
    K.check_device_errors()
    first, k, v = engine.read_cache(_add(engine, prompt), 0)
    assert k.shape == v.shape and k.dtype == DT[dtype] and first + k.shape[0] == 150


def _add(engine, prompt):
    from hfcpu_b200.engine import StepEntry
    engine.add_request("again")
    engine.step([StepEntry("again", prompt)])
    return "again"


def test_session_generates_on_8_bits(tiny_folders):
    import hfcpu_b200
    prompts = [[1, 2, 3], list(range(40)), [9] * 130]
    kw = dict(temp=0.0, max_tokens=12, eos_ids=[])
    sess = hfcpu_b200.Session(tiny_folders["C16"], kv_dtype="int8", ctx_max=512, kv_pages=200, batch=50)
    a = sess.generate(prompts, **kw)
    b = sess.generate(prompts, **kw)
    assert [[c.tokens for c in x] for x in a] == [[c.tokens for c in x] for x in b] and all(len(c.tokens) == 12 for x in a for c in x)
    # two completions of one prompt share its pages
    c = sess.generate(prompts[2], n=2, **kw)
    assert c[0].tokens == c[1].tokens
    sess.engine.cache.check()


@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128)])
def test_alike_layers_made_again_give_the_same_bits(heads, monkeypatch):
    """A step through recorded launches against the same step layer by layer, on records of layers that differ in nothing else:
    portions on either kernel, several requests, single tokens."""
    from hfcpu_b200.config import config_from_dict
    from hfcpu_b200.engine import Engine, StepEntry
    from hfcpu_b200.kernels.native import Recording
    from hfcpu_b200.models import random_model
    K, (H, G, d) = native(), heads
    config = config_from_dict(dict(architectures=["Qwen2ForCausalLM"], num_hidden_layers=5, hidden_size=H * d, num_attention_heads=H,
                                   num_key_value_heads=G, intermediate_size=1024, vocab_size=1000, max_position_embeddings=1024,
                                   rms_norm_eps=1e-6, rope_theta=1e6, tie_word_embeddings=False))
    model, made, inner = random_model(config, seed=5, dtype=torch.bfloat16, device=DEV, std=0.08), [], Recording.replay

    def replay(self, tensors):
        made.append(inner(self, tensors))
        return made[-1]
    monkeypatch.setattr(Recording, "replay", replay)
    got = []
    for record in (True, False):
        if not record:
            monkeypatch.setattr(K, "recorder", lambda: None)
        engine = Engine(model, block_size=16, max_tokens=2048, max_requests=4, kv_dtype="int8")
        engine.use_graphs = False
        engine.add_request("a")
        engine.add_request("b")
        got.append(torch.stack([engine.step([StepEntry(r, [(7 * i + n + (r == "b")) % 1000 for i in range(n)], [n - 1]) for r in "ab"]).clone()
                                for n in (300, 40, 3, 1, 1)]))
    assert torch.equal(got[0], got[1]) and torch.isfinite(got[0]).all()
    assert len(made) >= 10 and all(made)
    K.check_device_errors()


# ---- the prompts' kernel: what stands between a CTA's pieces -----------------------------------------------------------------

@pytest.mark.parametrize("shape", [(32, 8, 64, 16), (28, 4, 128, 8)], ids=str)
def test_many_short_pieces_a_cta(shape):
    """Portions of one or two steps each, many more than there are CTAs: a CTA's places for codes go from one piece to the next without a
    pause, and a piece's last copies must not land on the next one's first."""
    H, G, d, bs = shape
    s = step([33 + i % 5 for i in range(60)], [33 + i % 5 + 100 * (i % 3) for i in range(60)], bs, G, d, seed=d)
    assert set(n.split(".")[0] for n in native().kv8_step_arrays(s.q_lens, H // G)) == {"many"}
    cache = pack(s.k, s.ks, s.v, s.vs)
    q = torch.randn(s.T, H * d, generator=s.g, device=DEV).bfloat16()
    got = attend(s, q, cache, H)
    check(s, q, cache, got, H)
    for _ in range(5):
        assert torch.equal(got, attend(s, q, cache, H))
    native().check_device_errors()


def test_second_query_tile_without_tokens():
    """Portions that the first query tile holds alone: the second one's warps walk through hundreds of steps that are not theirs."""
    for d in (64, 128):
        s = step([20] * 6, [20, 5000, 900, 3000, 64, 2000], 16, 2, d, seed=d + 1)
        assert set(n.split(".")[0] for n in native().kv8_step_arrays(s.q_lens, 4)) == {"many"}
        cache = pack(s.k, s.ks, s.v, s.vs)
        q = torch.randn(s.T, 8 * d, generator=s.g, device=DEV).bfloat16()
        got = attend(s, q, cache, 8)
        check(s, q, cache, got, 8)
        assert torch.equal(got, attend(s, q, cache, 8))
        native().check_device_errors()


def test_attention_is_right_again_behind_a_launch_that_gave_up(monkeypatch):
    """Counts that a launch left behind (put there from the host) are gone once its error has been taken: eager and captured launches."""
    import ctypes
    K = native()
    b = K.backend()
    s = step([1, 90, 1], [3000, 2000, 1500], 16, 2, 64, seed=12)
    cache = pack(s.k, s.ks, s.v, s.vs)
    q, buf = torch.randn(s.T, 8 * 64, generator=s.g, device=DEV).bfloat16(), context()
    plan = {n: torch.from_numpy(a).to(DEV) for n, a in K.kv8_step_arrays(s.q_lens, 4).items()}
    assert len(plan) == 6
    right, out = attend(s, q, cache, 8, buf=buf, plan=plan), torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(s, q, cache, 8, buf=buf, plan=plan, out=out)
    for c in (c for of_scratch in b._kv8_counters.values() for c in of_scratch):
        c.fill_(1)
    torch.cuda.synchronize()
    take = b.lib.hfb_error_word_take

    class Lib:
        def __getattr__(self, name):
            return getattr(lib, name)

        @staticmethod
        def hfb_error_word_take(at, stream):
            rc = take(at, stream)
            ctypes.cast(at, ctypes.POINTER(ctypes.c_int32))[0] = 4
            return rc
    lib = b.lib
    b.lib = Lib()
    try:
        with pytest.raises(K.DeviceFault):
            K.check_device_errors()
    finally:
        b.lib = lib
    graph.replay()
    assert torch.equal(out, right) and torch.equal(attend(s, q, cache, 8, buf=buf, plan=plan), right)
    check(s, q, cache, right, 8)
    K.check_device_errors()


@pytest.mark.parametrize("sink", ["learned", "zero"])
@pytest.mark.parametrize("slope", [0.0, 0.01, 0.02, 0.05, 0.2])
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (28, 4, 128, 16)], ids=str)
def test_sinks_beside_keys_far_below_them(shape, slope, sink):
    """Thousands of keys, many pieces a tile: with a bias linear in the distance the oldest keys' scores lie hundreds or thousands below the
    sink, and without one a sink may stand far above (or below) every score."""
    H, G, d, bs = shape
    K = native()
    s = step([40, 300, 96], [8040, 8300, 700], bs, G, d, seed=H)
    assert set(n.split(".")[0] for n in K.kv8_step_arrays(s.q_lens, H // G)) == {"many"}
    cache = pack(s.k, s.ks, s.v, s.vs)
    q = (torch.randn(s.T, H * d, generator=s.g, device=DEV) * 2).bfloat16()
    o = dict(zero_sink=True) if sink == "zero" else dict(sinks=torch.randn(H, device=DEV, generator=gen(2)))
    if slope:
        o["slopes"] = torch.full((H,), slope, device=DEV) * torch.linspace(0.5, 1, H, device=DEV)
    for far in (0.0, 120.0, -120.0) if sink == "learned" else (0.0,):
        if sink == "learned":
            o["sinks"] = torch.randn(H, device=DEV, generator=gen(2)) + far
        got = attend(s, q, cache, H, **o)
        assert torch.isfinite(got).all()
        check(s, q, cache, got, H, **o)
    K.check_device_errors()


# ---- scales far apart --------------------------------------------------------------------------------------------------------
# Nothing that a row does not see may take part in how its numbers are rounded by more than a step, and no value is too small beside its
# neighbours.  Tolerance: the output's rounding 2^-8; a weight's rounding 2^-11, a value's scale's and the value's own, 2^-11 each, of
# sum p |v|; the scores' e as above, with a key's own rounding in the prompts' kernel: 2^-11 of sum |q k|, which the sum |q| 255 scale that e
# is taken of exceeds twofold at least, so 2^-12 of it at most; 4 e.  And float16's smallest step, 2^-24: a weight times its value's
# reference (a power of two, at most twice the value's scale) is held as 2^10 times its share of the largest such product among the keys
# that the row sees, so that each of n keys is off by 127 2^-25 2^-10 2 times the largest p scale of the row.  The row of values that has
# it has a code of 127: 127 p scale is at most the largest sum p |v| of the row.  2^-34 n of that, and nothing of what the row does not
# see.  (The first run came without this last term: numbers of 1e-10 beside ones of 1e12 in the same output row were zeros.)

def check_apart(s, q, got, H, rows=None, mask=0, scale=None, cache=None, size_of_scores=None, least=0.0):
    """``rows``: tokens that are looked at; ``size_of_scores``: sum |q| 255 scale to reckon with instead of that of all keys seen."""
    scale = 1 / math.sqrt(s.d) if scale is None else scale
    rows = torch.arange(s.T, device=DEV) if rows is None else rows
    ref, size, worst, _ = attention(q[rows], cache, s.table, s.seq[rows], s.positions[rows], s.bs, H, s.G, s.d, mask, scale)
    worst = worst if size_of_scores is None else size_of_scores
    e = (2.0 ** -16 + 2.0 ** -20 + (2.0 ** -12 if size_of_scores is None else 0)) * worst
    got = got[rows].double().view(ref.shape)
    assert torch.isfinite(got).all()
    tol = 2.0 ** -8 * ref.abs() + (3 * 2.0 ** -11 + 4 * min(e, 0.02)) * size + 2.0 ** -34 * max(s.kv_lens) * size.amax(-1, keepdim=True)
    off = (got - ref).abs()
    assert float(ref.abs().max()) >= least and (off <= tol + 1e-37).all(), float((off / (tol + 1e-37)).max())


APART = [(14, 2, 64, 16), (28, 4, 128, 16), (8, 2, 80, 16)]
APART_STEPS = {"portion": ([70, 90], [70, 800]), "few": ([5, 3, 16, 1], [5, 300, 90, 200])}


@pytest.mark.parametrize("name", list(APART_STEPS))
@pytest.mark.parametrize("shape", APART, ids=str)
def test_later_tokens_change_nothing_before_them(shape, name):
    """The last tokens of each request bring values, or keys, up to 2^60 times as large as the others."""
    H, G, d, bs = shape
    for by in (2.0 ** 14, 2.0 ** 24, 2.0 ** 40, 2.0 ** 60):
        for of in ("values", "keys"):
            s = step(*APART_STEPS[name], bs, G, d, seed=d)
            q = torch.randn(s.T, H * d, generator=s.g, device=DEV).bfloat16()
            before, at = [], 0
            for i, (n_q, n) in enumerate(zip(s.q_lens, s.kv_lens)):
                late = 0 if n_q == 1 else n_q // 2
                for p in range(n - late, n):
                    (s.vs if of == "values" else s.ks)[s.table[i, p // bs], p % bs] *= by
                before += range(at, at + n_q - late)
                at += n_q
            cache = pack(s.k, s.ks, s.v, s.vs)
            check_apart(s, q, attend(s, q, cache, H), H, rows=torch.tensor(before, device=DEV), cache=cache)


@pytest.mark.parametrize("name", list(APART_STEPS))
@pytest.mark.parametrize("shape", APART, ids=str)
def test_values_of_any_size(shape, name):
    """All values small or large; sizes from 2^-40 to 2^40 side by side; large ones that weigh next to nothing."""
    H, G, d, bs = shape
    for by in (2.0 ** -115, 2.0 ** -95, 2.0 ** 80):
        s = step(*APART_STEPS[name], bs, G, d, seed=d)
        q = torch.randn(s.T, H * d, generator=s.g, device=DEV).bfloat16()
        s.vs *= by
        cache = pack(s.k, s.ks, s.v, s.vs)
        check_apart(s, q, attend(s, q, cache, H), H, cache=cache, least=by)
    s = step(*APART_STEPS[name], bs, G, d, seed=d)
    s.vs *= 2.0 ** torch.randint(-40, 41, s.vs.shape, generator=s.g, device=DEV)
    cache = pack(s.k, s.ks, s.v, s.vs)
    check_apart(s, q, attend(s, q, cache, H), H, cache=cache)
    # every ninth key's score lies about 40 below the others' in the base 2, and its value is 2^30 or 2^-30 as large
    for by in (2.0 ** 30, 2.0 ** -30):
        s = step(*APART_STEPS[name], bs, G, d, seed=d)
        q = (torch.randn(s.T, H * d, generator=s.g, device=DEV) * 0.3 + 0.5).bfloat16()
        s.k[:, ::9], s.ks[:, ::9] = -100, 28 / (100 * 0.5 * math.sqrt(d))
        s.vs[:, ::9] *= by
        cache = pack(s.k, s.ks, s.v, s.vs)
        check_apart(s, q, attend(s, q, cache, H), H, cache=cache)


@pytest.mark.parametrize("name", list(APART_STEPS))
@pytest.mark.parametrize("shape", APART, ids=str)
def test_keys_beside_one_that_is_far_larger(shape, name):
    """A key of each tile 2^22 times as large as the others, whose scores are as far below theirs: it has no weight, and the others have
    theirs."""
    H, G, d, bs = shape
    s = step(*APART_STEPS[name], bs, G, d, seed=d)
    q = (torch.randn(s.T, H * d, generator=s.g, device=DEV) * 0.3 + 1).bfloat16()
    plain = pack(s.k, s.ks, s.v, s.vs)
    _, _, worst, _ = attention(q, plain, s.table, s.seq, s.positions, bs, H, G, d, 0, 1 / math.sqrt(d))
    for i, n in enumerate(s.kv_lens):
        for p in range(3, n, 33):
            s.k[s.table[i, p // bs], p % bs], s.ks[s.table[i, p // bs], p % bs] = -100, 2.0 ** 22 * 0.02
    cache = pack(s.k, s.ks, s.v, s.vs)
    check_apart(s, q, attend(s, q, cache, H), H, cache=cache, size_of_scores=worst)


# ---- what users get without these tests' smaller threshold; other architectures ------------------------------------------------

@pytest.mark.parametrize("mask", [0, 50, -100])
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (28, 4, 128, 16), (32, 8, 128, 16), (40, 2, 128, 8)], ids=str)
def test_steps_below_the_prompts_kernels_threshold(shape, mask, monkeypatch):
    """The choice as it is: steps of up to 512 rows go to the kernel of few queries, several tiles a request, and larger ones to both."""
    H, G, d, bs = shape
    K = native()
    monkeypatch.setattr(K, "KV8_MANY_ROWS", 512)
    for q_lens, kv_lens, kinds in (([9, 1, 14], [309, 200, 14], {"few"}), ([25], [700], {"few"}), ([1, 130, 2], [900, 130, 400], {"few", "many"})):
        s = step(q_lens, kv_lens, bs, G, d, seed=d + len(q_lens))
        assert {n.split(".")[0] for n in K.kv8_step_arrays(s.q_lens, H // G)} == kinds
        cache = pack(s.k, s.ks, s.v, s.vs)
        q = torch.randn(s.T, H * d, generator=s.g, device=DEV).bfloat16()
        o = dict(sinks=torch.randn(H, device=DEV, generator=gen(2)), slopes=torch.full((H,), 0.05, device=DEV)) if mask >= 0 else {}
        got = attend(s, q, cache, H, mask=mask, **o)
        check(s, q, cache, got, H, mask=mask, **o)
        assert torch.equal(got, attend(s, q, cache, H, mask=mask, settled=True, **o))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("arch", ["manapel", "tupalorn"])
def test_other_architectures_on_8_bits(arch, dtype, monkeypatch):
    """Layers with tails of their own (head norms, a norm over the row), windows, caches that later layers read: logits against the
    stand-in backend's, with the tolerances of the engine's test above; prompts on either kernel, graphs and eager steps."""
    import importlib
    from hfcpu_b200.config import config_from_dict
    from hfcpu_b200.engine import Engine, StepEntry
    from hfcpu_b200.models import Model
    from hfcpu_b200.weights.random_init import RandomSource
    K = native()
    monkeypatch.setattr(K, "KV8_MANY_ROWS", 512)
    cfg = config_from_dict(importlib.import_module(arch + "_util").WIDE)
    cpu = torch.device("cpu")
    source = RandomSource(Model(cfg, torch.float32, cpu).tensor_specs(), 5, torch.float32, cpu, std=0.05)
    weights = {t.name: source[t.name].to(DT[dtype]) for t in Model(cfg, torch.float32, cpu).tensor_specs()}
    ids = [int(x) for x in torch.randint(0, 1000, (400,), generator=torch.Generator().manual_seed(1))]

    def run(kv, dt, device, cuts):
        model = Model(cfg, dt, torch.device(device)).bind({n: w.to(device) for n, w in weights.items()})
        engine, out = Engine(model, block_size=16, max_tokens=2048, max_requests=2, kv_dtype=kv), []
        for r, cut in enumerate(cuts):
            engine.add_request(r)
            at = 0
            for n in cut:
                got = engine.step([StepEntry(r, ids[at:at + n], [n - 1])])
                at += n
            out.append(torch.cat([got.clone()] + [engine.step([StepEntry(r, [5 + i], [0])]).clone() for i in range(5)]).float().cpu())
            engine.finish_request(r)
        return out
    real = K.backend()
    try:
        K.set_backend(EmuKv8())
        plain, emu = (run(kv, torch.float32, "cpu", [[300]])[0] for kv in ("auto", "int8"))
    finally:
        K.set_backend(real)
    own = float((run("auto", DT[dtype], DEV, [[300]])[0] - plain).abs().max())
    far = float((emu - plain).abs().max())
    assert far > 0
    for got in run("int8", DT[dtype], DEV, [[300], [200, 90, 10], [3, 40, 257]]):
        assert torch.isfinite(got).all()
        assert float((got - emu).abs().max()) <= (0.25 * far + 1e-4 if dtype == "float32" else far + 2 * own)
    K.check_device_errors()


@pytest.mark.parametrize("d", [64, 128])
def test_two_streams_and_a_graph_at_once(d):
    """Calls that run beside each other, each with scratch of its own: two streams' eager launches and a graph's replays, of tiles that many
    CTAs share."""
    K, H = native(), 8
    s = step([1, 100, 1, 1], [9000, 4000, 30, 5000], 16, 2, d, seed=d)
    cache = pack(s.k, s.ks, s.v, s.vs)
    plan = {n: torch.from_numpy(a).to(DEV) for n, a in K.kv8_step_arrays(s.q_lens, H // 2).items()}
    assert len(plan) == 6
    qs = [torch.randn(s.T, H * d, generator=s.g, device=DEV).bfloat16() for _ in range(3)]
    right = [attend(s, q, cache, H, plan=plan) for q in qs]
    check(s, qs[0], cache, right[0], H)
    bufs, outs, streams = [context() for _ in qs], [torch.zeros_like(q) for q in qs], [torch.cuda.Stream() for _ in qs]
    attend(s, qs[2], cache, H, plan=plan, buf=bufs[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(s, qs[2], cache, H, plan=plan, buf=bufs[2], out=outs[2])
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o.zero_()
        for i, stream in enumerate(streams):
            stream.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            for i, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    graph.replay() if i == 2 else attend(s, qs[i], cache, H, plan=plan, buf=bufs[i], out=outs[i])
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        assert all(torch.equal(a, b) for a, b in zip(outs, right))
    K.check_device_errors()
