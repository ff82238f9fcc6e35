"""What the batched entries refuse before anything is launched (no GPU)."""
import ctypes

import pytest

import mlb

P = ctypes.c_void_p(64)       # aligned, never followed
ODD = ctypes.c_void_p(68)
BIG = 1 << 30


def packed(q=P, k=P, v=P, out=P, qo=P, ko=P, n=2, rows=4, keys=4, nh=8, kvh=2, hd=64, scratch=P,
           floats=BIG):
    return mlb.load().mlb_attention_packed_f32(q, k, v, out, qo, ko, n, rows, keys, nh, kvh, hd,
                                               scratch, floats, None, None)


def write(kc=P, vc=P, ks=P, vs=P, blocks=4, block=32, table=P, cols=2, n=2, k=P, v=P, o=P, p=P,
          rows=4, kvh=2, hd=64):
    return mlb.load().mlb_kv8_write_f32(kc, vc, ks, vs, blocks, block, table, cols, n, k, v, o, p,
                                        rows, kvh, hd, None, None)


def read(kc=P, vc=P, ks=P, vs=P, blocks=4, block=32, table=P, cols=2, n=2, k=P, v=P, o=P, p=P,
         rows=4, kvh=2, hd=64):
    return mlb.load().mlb_kv8_read_f32(kc, vc, ks, vs, blocks, block, table, cols, n, k, v, o, p,
                                       rows, kvh, hd, None, None)


def decode(q=P, kc=P, vc=P, ks=P, vs=P, blocks=4, block=32, table=P, cols=2, lengths=P, n=2, nh=8,
           kvh=2, hd=64, out=P, mass_in=None, mass_out=None, scratch=P, floats=BIG):
    return mlb.load().mlb_attention_kv8_f32(q, kc, vc, ks, vs, blocks, block, table, cols, lengths,
                                            n, nh, kvh, hd, out, mass_in, mass_out, scratch,
                                            floats, None, None)


def evict(table=P, cols=8, lengths=P, mass=P, n=2, block=32, keep=4, sink=1, recent=1, to=P, lo=P,
          mo=P, freed=None):
    return mlb.load().mlb_kv8_evict(table, cols, lengths, mass, n, block, keep, sink, recent, to,
                                    lo, mo, freed, None, None)


NULLS = [
    (packed, ["q", "k", "v", "out", "qo", "ko"]),
    (write, ["kc", "vc", "ks", "vs", "table", "k", "v", "o", "p"]),
    (read, ["kc", "vc", "ks", "vs", "table", "o", "p"]),
    (decode, ["q", "kc", "vc", "ks", "vs", "table", "lengths", "out", "scratch"]),
    (evict, ["table", "lengths", "mass", "to", "lo", "mo"]),
]


@pytest.mark.parametrize("call,name", [(c, n) for c, names in NULLS for n in names])
def test_null_pointers(call, name):
    assert call(**{name: None}) == 1
    assert b"mlb_" in mlb.load().mlb_last_error()


@pytest.mark.parametrize("call,name", [
    (packed, n) for n in ("q", "k", "v", "out", "scratch")] + [
    (write, n) for n in ("kc", "vc", "k", "v")] + [
    (read, n) for n in ("kc", "vc", "k", "v")] + [
    (decode, n) for n in ("q", "kc", "vc", "out", "scratch")])
def test_misaligned_pointers(call, name):
    assert call(**{name: ODD}) == 1


@pytest.mark.parametrize("call,bad", [
    (packed, dict(nh=7)), (packed, dict(nh=18)), (packed, dict(hd=66)), (packed, dict(hd=260)),
    (packed, dict(hd=0)), (packed, dict(kvh=0)), (packed, dict(rows=-1)), (packed, dict(keys=-1)),
    (packed, dict(n=-1)), (packed, dict(rows=1 << 30)), (packed, dict(n=1 << 30)),
    (write, dict(block=16)), (write, dict(block=48)), (write, dict(hd=40)), (write, dict(hd=288)),
    (write, dict(rows=-1)), (write, dict(n=-1)), (write, dict(cols=-1)), (write, dict(blocks=-1)),
    (write, dict(kvh=0)), (write, dict(cols=1 << 30)), (write, dict(rows=1 << 40)),
    (read, dict(block=0)), (read, dict(hd=-32)), (read, dict(k=None, v=None)),
    (decode, dict(block=33)), (decode, dict(hd=48)), (decode, dict(nh=9)), (decode, dict(nh=18)),
    (decode, dict(n=-1)), (decode, dict(cols=-1)), (decode, dict(blocks=-1)),
    (decode, dict(blocks=1 << 40)), (decode, dict(mass_in=P)), (decode, dict(floats=0)),
    (evict, dict(block=1)), (evict, dict(keep=1)), (evict, dict(recent=0)), (evict, dict(sink=-1)),
    (evict, dict(sink=3, recent=2)), (evict, dict(cols=-1)), (evict, dict(n=-1)),
    (evict, dict(sink=1 << 62, recent=1 << 62, keep=1 << 62)),
])
def test_bad_sizes(call, bad):
    assert call(**bad) == 1
    assert mlb.load().mlb_last_error()


def test_nothing_to_do():
    """Empty calls launch nothing and need no pointers."""
    assert packed(rows=0, q=None, out=None) == 0
    assert packed(n=0, qo=None, ko=None) == 0
    assert write(rows=0, k=None, v=None) == 0 and write(n=0) == 0
    assert read(rows=0, k=None, v=None) == 0 and read(n=0) == 0
    assert decode(n=0, q=None, out=None) == 0
    assert evict(n=0, table=None) == 0


def test_scratch_sizes():
    lib = mlb.load()
    assert lib.mlb_attention_packed_scratch_floats(10, 10, 2, 8, 2, 64) >= 0
    assert lib.mlb_attention_packed_scratch_floats(10, 10, 2, 8, 3, 64) == -1
    plain = lib.mlb_attention_kv8_scratch_floats(4, 16, 32, 8, 2, 64, 0)
    mass = lib.mlb_attention_kv8_scratch_floats(4, 16, 32, 8, 2, 64, 1)
    assert mass >= plain >= 0
    assert lib.mlb_attention_kv8_scratch_floats(4, 16, 16, 8, 2, 64, 0) == -1
    need = lib.mlb_attention_kv8_scratch_floats(2, 2, 32, 8, 2, 64, 1)
    assert decode(mass_out=P, floats=need - 1) == 1


def test_binding_refusals():
    """The Python binding's own checks (CPU tensors are enough)."""
    import torch
    f, i = torch.zeros(4, 8, 64), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        mlb.attention_packed(f, f, f, i)
    with pytest.raises(ValueError):
        mlb.kv8_cache(4, 2, 48, 64, "cpu")
    cache = mlb.kv8_cache(4, 2, 32, 64, "cpu")
    assert cache.k_codes.shape == (4, 2, 32, 64) and cache.v_codes.shape == (4, 2, 64, 32)
    table = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        mlb.kv8_write(cache, table, torch.zeros(4, 2, 64), torch.zeros(4, 2, 64), i, i[:2])
    with pytest.raises(ValueError):
        mlb.kv8_read(cache, table, i, i[:2], 4)
    with pytest.raises(ValueError):
        mlb.attention_kv8(torch.zeros(2, 8, 64), cache, table, i[:2])
    with pytest.raises(ValueError):
        mlb.kv8_evict(table, i[:2], torch.zeros(2, 2), 32, 4)
