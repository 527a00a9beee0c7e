"""The cache in 8 bits without a GPU: its layout and numbers, tile lists, refusals, and the engine's host side on a stand-in backend."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import hfcpu_b200
from conftest import TINY
from hfcpu_b200 import kernels
from hfcpu_b200.config import config_from_dict
from hfcpu_b200.config.base import UnsupportedError
from hfcpu_b200.engine import Engine, StepEntry
from hfcpu_b200.models import random_model
from kv8_util import EmuKv8, pack, quantised, unpack, values


@pytest.fixture
def emu():
    old = kernels._backend
    kernels.set_backend(EmuKv8())
    yield
    kernels.set_backend(old)


@pytest.mark.parametrize("bs", [1, 5, 8, 16, 64])
@pytest.mark.parametrize("d", [16, 64, 80, 128, 192, 256])
def test_records_hold_what_was_packed(bs, d):
    g = torch.Generator().manual_seed(bs * d)
    x = torch.randn(3, bs, 2, d, generator=g)
    k, ks = quantised(x)
    v, vs = quantised(x.flip(-1) * 3)
    c = pack(k, ks, v, vs)
    assert c.shape[2] == kernels.kv8_record_bytes(bs, d) and c.shape[2] % 16 == 0
    assert all(torch.equal(a, b) for a, b in zip(unpack(c, bs, 2, d), (k, ks, v, vs)))
    # off by half a step at most: half the scale, which is the row's largest / 127 (rounded to float32)
    kk, _ = values(c, bs, 2, d)
    assert ((kk - x.double()).abs() <= ks.double()[..., None] * 0.5 * (1 + 2.0 ** -22)).all()


def test_rows_of_zeros_and_of_no_numbers():
    x = torch.zeros(4, 16)
    x[1, 3], x[2, 0], x[3, 5] = float("inf"), float("nan"), 1e-45
    codes, scale = quantised(x)
    assert scale[0] == 2.0 ** -126 and (codes[0] == 0).all()
    assert torch.isnan(scale[1:3]).all()
    assert scale[3] == 2.0 ** -126 and (codes[3] == 0).all()


@pytest.mark.parametrize("r", [1, 3, 7, 16, 17, 20, 32, 64])
@pytest.mark.parametrize("q_lens", [[1], [1, 1, 1], [5, 1, 33, 2], [200], [1, 700, 3]])
def test_tile_lists_cover_every_token_once(q_lens, r):
    a = kernels.kv8_step_arrays(q_lens, r)
    assert all(x.dtype == np.int32 for x in a.values())
    first = np.concatenate([[0], np.cumsum(q_lens)])
    seen = np.zeros(sum(q_lens), dtype=int)
    for h in {n.split(".")[0] for n in a}:
        share = kernels.kv8_head_groups(r)
        for s, t0, nt in zip(a[h + ".seq"], a[h + ".t0"], a[h + ".nt"]):
            assert nt >= 1 and first[s] <= t0 and t0 + nt <= first[s + 1]
            if h == "few":
                assert nt * (r // share) <= 16 and (nt == 1 or share == 1)
            else:
                assert h == "many" and nt <= 2 * (128 // r)
            seen[t0:t0 + nt] += 1
        assert len(set(len(x) for n, x in a.items() if n.startswith(h))) == 1
    assert (seen == 1).all()


def _args(T=4, H=4, G=2, d=32, bs=8, dtype=torch.bfloat16):
    return dict(qkv=torch.zeros(T, (H + 2 * G) * d, dtype=dtype), cos_sin=torch.zeros(9, d // 2, 2), n_rot=d, positions=torch.zeros(T, dtype=torch.int32),
                slots=torch.zeros(T, dtype=torch.int32), q_out=torch.zeros(T, H * d, dtype=dtype), cache=kernels.kv8_cache(3, bs, G, d, "cpu"), H=H, G=G, d=d,
                block_size=bs)


@pytest.mark.parametrize("change", [dict(qkv=torch.zeros(4, 255, dtype=torch.bfloat16)), dict(qkv=torch.zeros(4, 256, dtype=torch.float16)),
                                    dict(q_out=torch.zeros(4, 128)), dict(n_rot=33), dict(n_rot=34), dict(cos_sin=None), dict(cos_sin=torch.zeros(9, 8, 2)),
                                    dict(positions=torch.zeros(3, dtype=torch.int32)), dict(slots=torch.zeros(4, dtype=torch.int64)),
                                    dict(cache=torch.zeros(3, 2, 100, dtype=torch.uint8)), dict(block_size=16), dict(pairing="pairs"), dict(G=4)])
def test_rope_kv8_write_refuses(emu, change):
    with pytest.raises(ValueError):
        kernels.rope_kv8_write(**{**_args(), **change})


def test_other_refusals(emu):
    c = kernels.kv8_cache(3, 8, 2, 32, "cpu")
    i4 = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        kernels.kv8_write(torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.bfloat16), i4, c, 2, 32, 8)
    with pytest.raises(ValueError):
        kernels.kv8_write(torch.zeros(4, 64), torch.zeros(4, 64), i4[:3], c, 2, 32, 8)
    out = torch.zeros(4, 8, 2, 32)
    for pages, rows, k, v in ((i4[:2], i4, out, out), (i4, i4.long(), out, out), (i4, i4, out, out.bfloat16()), (i4, i4, out.half(), out.half()),
                              (i4, i4, out[..., :16], out[..., :16])):
        with pytest.raises(ValueError):
            kernels.kv8_read(c, pages, rows, k, v)
    q = torch.zeros(4, 128)
    meta = SimpleNamespace(block_table=torch.zeros(1, 2, dtype=torch.int32), block_size=8, max_blocks=2)
    ctx = SimpleNamespace(positions=i4, token_seq=i4, max_q_len=4, max_kv_len=4)
    for bad in (dict(q=q.half()), dict(out=q.bfloat16()), dict(H=3), dict(G=3), dict(sinks=torch.zeros(3)), dict(slopes=torch.zeros(4).double()),
                dict(sinks=torch.zeros(4), zero_sink=True), dict(softcap=-1.0), dict(meta=SimpleNamespace(block_table=meta.block_table.long(), block_size=8, max_blocks=2)),
                dict(meta=SimpleNamespace(block_table=meta.block_table, block_size=16, max_blocks=2)), dict(ctx=SimpleNamespace(positions=i4[:3], token_seq=i4))):
        args = dict(q=q, cache=c, meta=meta, ctx=ctx, H=4, G=2, d=32, window=0, scale=1.0, out=torch.zeros_like(q))
        with pytest.raises(ValueError):
            kernels.paged_attention_kv8(**{**args, **bad})
    for bs, d in ((8, 24), (8, 272), (0, 64), (2000, 64)):
        with pytest.raises(UnsupportedError):
            kernels.kv8_cache(1, bs, 1, d, "cpu")


def _engine(name, kv_dtype, **more):
    model = random_model(config_from_dict(TINY[name]), seed=3, dtype=torch.float32, device="cpu", std=0.05)
    return Engine(model, block_size=8, max_tokens=512, max_requests=4, kv_dtype=kv_dtype, **more)


@pytest.mark.parametrize("name", ["A", "B"])
def test_engine_on_8_bits_follows_the_plain_cache(emu, name):
    """Logits near those of the float32 cache, the same however the prompt is cut, and again on recycled pages."""
    prompt = [int(x) for x in torch.randint(0, 500, (75,), generator=torch.Generator().manual_seed(1))]
    got = {}
    for kv in ("auto", "int8"):
        for cut in ([75], [16, 1, 58], [40, 35]):
            eng = _engine(name, kv)
            for again in range(2):
                eng.add_request("r")
                at = 0
                for n in cut:
                    out = eng.step([StepEntry("r", prompt[at:at + n], [n - 1])])
                    at += n
                out = eng.step([StepEntry("r", [7], [0])])
                got[kv, tuple(cut), again] = out.clone()
                eng.finish_request("r")
            eng.cache.check()
    ref = got["auto", (75,), 0]
    for (kv, cut, again), x in got.items():
        if kv == "int8":
            assert torch.allclose(x, got["int8", (75,), 0], atol=1e-4), (cut, again)
            # (rows are off by 1/254 of their largest value at most)
            assert float((x - ref).abs().max() / ref.abs().max()) < 0.05
            assert not torch.equal(x, ref)


def test_read_cache_and_forks(emu):
    eng8, eng = _engine("B", "int8"), _engine("B", "auto")
    prompt = [int(x) for x in torch.randint(0, 500, (90,), generator=torch.Generator().manual_seed(2))]
    for e in (eng8, eng):
        e.add_request("a")
        e.step([StepEntry("a", prompt, [89])])
        e.add_request("b")
        assert e.fork_request("a", "b", 90) > 0
        e.step([StepEntry("b", prompt[e.length("b"):] + [3], [0])])
        e.step([StepEntry("a", [3], [0])])
    for entry in range(3):
        for r in ("a", "b"):
            (f8, k8, v8), (f, k, v) = eng8.read_cache(r, entry), eng.read_cache(r, entry)
            assert f8 == f and k8.shape == k.shape and v8.shape == v.shape and k8.shape[0] + f == 91
            if entry == 0:
                # the first layer's rows are those of the plain cache, off by half a step at most
                for a, b in ((k8, k), (v8, v)):
                    step = b.abs().amax(-1, keepdim=True) / 127
                    assert ((a - b).abs() <= 0.51 * step + 1e-6).all()
    group = eng8.cache.groups[0]
    assert group.page_bytes * 3 < eng.cache.groups[0].page_bytes * 1.1       # (float32: 4 bytes against 1 and the scales)


def test_kv_dtype_refusals_and_options(emu):
    with pytest.raises(ValueError):
        _engine("A", "int4")
    from hfcpu_b200.cli import opts
    assert opts.defaults()["kv_dtype"] == "auto"
    assert opts.apply(opts.defaults(), ["--kv-dtype", "int8"])["kv_dtype"] == "int8"
    with pytest.raises(opts.OptionError):
        opts.apply(opts.defaults(), ["--kv-dtype", "int4"])
    model = random_model(config_from_dict(TINY["A"]), seed=3, dtype=torch.float32, device="cpu", std=0.05)
    wide = hfcpu_b200.Session(model, kv_mem=1 << 18, max_seqs=64, ctx_max=256)
    small = hfcpu_b200.Session(model, kv_mem=1 << 18, max_seqs=64, ctx_max=256, kv_dtype="int8")
    assert small.engine.num_pages > 2 * wide.engine.num_pages
    a, b = (s.generate([1, 2, 3], temp=0.0, max_tokens=6, eos_ids=[])[0].tokens for s in (wide, small))
    assert len(a) == len(b) == 6


def test_mixers_that_cannot_are_refused(emu):
    class Other(type(_engine("A", "auto").model.layers[0].mixer)):
        caches_eight_bits = False
    model = random_model(config_from_dict(TINY["A"]), seed=3, dtype=torch.float32, device="cpu", std=0.05)
    model.layers[1].mixer.__class__ = Other
    with pytest.raises(UnsupportedError):
        Engine(model, block_size=8, max_tokens=64, kv_dtype="int8")
    cfg = dict(TINY["A"], head_dim=24, num_attention_heads=4)
    with pytest.raises((UnsupportedError, ValueError)):
        Engine(random_model(config_from_dict(cfg), seed=3, dtype=torch.float32, device="cpu"), block_size=8, max_tokens=64, kv_dtype="int8")


def test_argument_types_are_the_headers():
    """The binding's argument types of the 8-bit cache's functions, against the C header."""
    import os
    import re
    from hfcpu_b200.kernels import build
    from hfcpu_b200.kernels.native import NativeBackend
    header = open(os.path.join(build.CSRC, "hfb200.h")).read()
    for name, signature in NativeBackend._KV8_SIGNATURES.items():
        args = re.search(r"int %s\((.*?)\);" % name, header, re.S).group(1).split(",")
        assert signature == "".join("p" if "*" in a or "hfb_stream" in a else "l" if "int64_t" in a else "z" if "size_t" in a else "f" if "float" in a else "i"
                                    for a in args), name


@pytest.mark.parametrize("arch", ["manapel", "tupalorn"])
def test_other_architectures_plain_layers(emu, arch):
    """Layers with head norms, a norm over the row, caches that other layers read: on 8 bits near the plain cache, and forks too."""
    import importlib
    cfg = config_from_dict(importlib.import_module(arch + "_util").WIDE)
    got = {}
    for kv in ("auto", "int8"):
        model = random_model(cfg, seed=3, dtype=torch.float32, device="cpu", std=0.05)
        eng = Engine(model, block_size=16, max_tokens=512, max_requests=2, ctx_max=256, kv_dtype=kv)
        ids = [int(x) for x in torch.randint(0, model.plan.vocab_size, (50,), generator=torch.Generator().manual_seed(1))]
        eng.add_request("r")
        eng.step([StepEntry("r", ids[:30], [29])])
        got[kv] = eng.step([StepEntry("r", ids[30:], [19])]).clone()
    assert not torch.equal(got["auto"], got["int8"])
    assert float((got["auto"] - got["int8"]).abs().max() / got["auto"].abs().max()) < 0.05


@pytest.mark.parametrize("arch", ["peludra", "mokisun", "silupel", "birizen"])
def test_latent_and_other_mixers_are_refused(emu, arch):
    import importlib
    model = random_model(config_from_dict(importlib.import_module(arch + "_util").WIDE), seed=3, dtype=torch.float32, device="cpu", std=0.05)
    with pytest.raises(UnsupportedError, match="8 bits"):
        Engine(model, block_size=16, max_tokens=512, max_requests=2, ctx_max=128, kv_dtype="int8")


def test_places_stay_where_captured_steps_point(emu):
    """A step with more tokens than any before asks for more places; graphs made earlier go on reading theirs."""
    import gc
    engine = Engine(random_model(config_from_dict(TINY["A"]), seed=3, dtype=torch.float32, device="cpu"), block_size=16, max_tokens=64, kv_dtype="int8")
    small = engine.places(8)
    address = small.data_ptr()
    storage = small.untyped_storage()._cdata
    large = engine.places(5000)
    del small
    gc.collect()
    assert torch.equal(large, torch.arange(5000, dtype=torch.int32))
    assert any(p.data_ptr() == address and p.untyped_storage()._cdata == storage for p in engine._places)
    assert torch.equal(engine.places(3), torch.arange(3, dtype=torch.int32))


def test_tile_lists_are_looked_at(emu):
    """Lists of another type, of different lengths or of another device are refused, and a kind of tile without one of its lists."""
    q, i4 = torch.zeros(4, 128), torch.zeros(4, dtype=torch.int32)
    meta = SimpleNamespace(block_table=torch.zeros(1, 2, dtype=torch.int32), block_size=8, max_blocks=2)
    ctx = SimpleNamespace(positions=i4, token_seq=i4, max_q_len=4, max_kv_len=4)
    args = dict(q=q, cache=kernels.kv8_cache(3, 8, 2, 32, "cpu"), meta=meta, ctx=ctx, H=4, G=2, d=32, window=0, scale=1.0, out=torch.zeros_like(q))
    for kind in ("few", "many"):
        good = {f"{kind}.{n}": torch.ones(2, dtype=torch.int32) for n in ("seq", "t0", "nt")}
        kernels.paged_attention_kv8(**args, tiles=good)
        for n in good:
            for bad in (good[n].long(), good[n].float(), good[n][:1], good[n][None], good[n].to("meta"), None):
                with pytest.raises(ValueError):
                    kernels.paged_attention_kv8(**args, tiles={**good, n: bad})
    kernels.paged_attention_kv8(**args, tiles={})


def test_captured_launches_share_counters_with_their_scratch():
    """However many steps are captured, none of their launches comes to counters of its own (zeroed by a node of the graph), and
    outgrown counters stay where captured launches point."""
    from hfcpu_b200.kernels import native
    b = native.NativeBackend.__new__(native.NativeBackend)
    b._kv8_counters = {}
    first = b._kv8_zeros("cpu", 1000, False, 256)
    assert first.numel() >= 256 and not first.any()
    at = first.data_ptr()
    assert all(b._kv8_zeros("cpu", 1000, capturing, 256).data_ptr() == at for capturing in (True, False) for _ in range(8192))
    # other scratch, which may be in use at the same time: other counters; and more counters than there were
    other, more = b._kv8_zeros("cpu", 2000, False, 256), b._kv8_zeros("cpu", 1000, False, 100000)
    assert len({at, other.data_ptr(), more.data_ptr()}) == 3 and more.numel() >= 100000 and not more.any()
    assert any(c is first for c in b._kv8_counters["cpu", 1000])
    assert b._kv8_zeros("cpu", 3000, True, 8).numel() == 8 and ("cpu", 3000) not in b._kv8_counters


def test_counters_are_cleared_behind_a_launch_that_gave_up(monkeypatch):
    """A nonzero error word clears whatever counters there are, not the other kernels' alone."""
    import ctypes
    from hfcpu_b200.kernels import native
    b = native.NativeBackend.__new__(native.NativeBackend)
    word = [0]

    class Lib:
        @staticmethod
        def hfb_error_word_take(at, stream):
            ctypes.cast(at, ctypes.POINTER(ctypes.c_int32))[0] = word[0]
            return 0
    b.lib, b._counters, b.launches = Lib, torch.ones(4, dtype=torch.int32), 0
    b._stream = lambda: None
    synced = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda d=None: synced.append(d))
    held = [torch.ones(n, dtype=torch.int32) for n in (8, 5, 3)]
    b._kv8_counters = {(0, 17): held[:2], (0, 18): held[2:]}
    assert b.error_word() == 0 and all(bool(x.all()) for x in held)
    word[0] = 8
    assert b.error_word() == 8 and not any(bool(x.any()) for x in held) and not b._counters.any()
    assert synced


@pytest.mark.parametrize("change,what", [(dict(d=24, dv=24), "heads of 24 and 24"), (dict(values_are_keys=True), "values inside its keys"), (dict(dv=48), "heads of 32 and 48"),
                                         (dict(caches_eight_bits=False), "does not run")])
def test_refusals_name_the_layer(emu, change, what):
    """A model with a layer that 8 bits do not serve, behind others that they do."""
    model = random_model(config_from_dict(TINY["A"]), seed=3, dtype=torch.float32, device="cpu", std=0.05)
    mixer = model.layers[1].mixer
    mixer.d, mixer.dv = 32, 32
    for name, value in change.items():
        setattr(mixer, name, value)
    with pytest.raises(UnsupportedError, match=rf"layer 1 \(PagedAttention\) .*{what}"):
        Engine(model, block_size=8, max_tokens=64, kv_dtype="int8")


def test_a_single_row_may_say_what_it_likes_of_the_next(emu):
    """One row's stride to the next one means nothing: any number is taken, as torch makes them."""
    row = torch.randn(1, 256)
    odd = torch.as_strided(row.clone(), (1, 256), (1, 1))
    assert odd.stride(0) == 1
    caches = []
    for x in (row, odd):
        a = _args(T=1, dtype=torch.float32)
        kernels.rope_kv8_write(**{**a, "qkv": x})
        kernels.kv8_write(x[:, 128:192], x[:, 192:], a["slots"] + 9, a["cache"], 2, 32, 8)
        caches.append(a["cache"])
    assert torch.equal(*caches) and caches[0].any()
    with pytest.raises(ValueError):
        kernels.rope_kv8_write(**{**_args(T=2, dtype=torch.float32), "qkv": torch.as_strided(torch.zeros(512), (2, 256), (1, 1))})
