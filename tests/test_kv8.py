"""The 8-bit KV cache on the host: the C ABI's refusals (before any launch), the fake kernels, the oracle."""
from __future__ import annotations

from fractions import Fraction

import pytest
import torch

from oracle import kv8 as ok


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg._abi.lib()


# Fake, never-dereferenced addresses: validation fails before any launch.
BASE = dict(k=16, vt=16, s=16, kt=16, vtt=16, dt=0, B=2, T=3, H=4, KVH=2, D=128, L=128, NB=2, pos=16, ps=1, qkv=16, ldq=1024,
            bias=16, cos=16, sin=16, ldc=64, q=16, out=16, window=0, sinks=0, scale=0.1, ws=16, wsb=1 << 40, length=16, ls=1,
            first=0, n=128)


def call(lib, name, **kw):
    a = dict(BASE, **kw)
    c = [a[x] for x in ("k", "vt", "s", "kt", "vtt", "dt")]
    rope = [a[x] for x in ("qkv", "ldq", "bias", "cos", "sin", "ldc")]
    if name == "write":
        return lib.w4a8_rope_kv8(*rope, a["pos"], a["ps"], a["q"], *c, a["B"], a["T"], a["H"], a["KVH"], a["D"], a["L"], a["NB"], None)
    if name == "read":
        return lib.w4a8_kv8_read(*c, a["length"], a["ls"], a["out"], a["out"], a["first"], a["n"], a["B"], a["KVH"], a["D"], a["NB"], None)
    end = [a[x] for x in ("L", "NB", "window", "sinks", "scale", "ws", "wsb")]
    if name == "attend":
        return lib.w4a8_attention_kv8(a["q"], *c, a["out"], a["pos"], a["ps"], a["B"], a["T"], a["H"], a["KVH"], a["D"], *end, None)
    return lib.w4a8_attention_kv8_rope(*rope, *c, a["out"], a["pos"], a["ps"], a["B"], a["H"], a["KVH"], a["D"], *end, None)


ALL = ("write", "read", "attend", "step")


@pytest.mark.parametrize("names,kw,code,msg", [
    (ALL, dict(dt=2), 3, "code_dtype"),
    (ALL, dict(D=96), 5, "head_dim"),
    (ALL, dict(NB=0), 2, "cache"),
    (ALL, dict(KVH=0), 2, "cache"),
    (ALL, dict(B=-1), 2, "cache"),
    (ALL, dict(NB=1 << 18), 2, "2^31"),
    (ALL, dict(NB=1 << 40), 2, "2^31"),
    (ALL, dict(B=1 << 30), 2, "B*KVH"),
    (ALL, dict(k=None), 1, "NULL"),
    (ALL, dict(vt=24), 4, "16-byte"),
    (ALL, dict(s=20), 4, "8-byte"),
    (ALL, dict(kt=8), 4, "16-byte"),
    (("write", "attend", "step"), dict(H=5), 2, "multiple of KVH"),
    (("write", "attend", "step"), dict(L=129), 2, "64 * NB"),
    (("write", "attend", "step"), dict(L=0), 2, "64 * NB"),
    (("write", "attend", "step"), dict(pos=None), 1, "NULL"),
    (("write", "attend", "step"), dict(ps=-1), 2, "pos_stride"),
    (("write", "attend"), dict(T=-1), 2, "bad shape"),
    (("write", "attend"), dict(T=1 << 31), 2, "bad shape"),
    (("write", "attend"), dict(T=1 << 30), 2, "B*T|bad shape"),
    (("write", "attend"), dict(H=1 << 18, KVH=1, B=1, T=1 << 14, ldq=1 << 30), 2, "bad heads"),
    (("write", "step"), dict(qkv=None), 1, "NULL"),
    (("write", "step"), dict(ldq=1016), 2, "ldq"),
    (("write", "step"), dict(ldq=1025), 2, "multiple of 8"),
    (("write", "step"), dict(ldc=63), 2, "ldc"),
    (("write", "step"), dict(bias=8), 4, "16-byte"),
    (("write", "step"), dict(cos=2), 4, "4-byte"),
    (("write", "attend"), dict(q=8), 4, "16-byte"),
    (("read",), dict(first=-1), 2, "inside"),
    (("read",), dict(first=129, n=0), 2, "inside"),
    (("read",), dict(first=1, n=128), 2, "inside"),
    (("read",), dict(n=1 << 62), 2, "inside"),
    (("read",), dict(length=None), 1, "NULL"),
    (("read",), dict(ls=-8), 2, "length_stride"),
    (("attend", "step"), dict(window=-1), 2, "window"),
    (("attend", "step"), dict(sinks=-1), 2, "sinks"),
    (("attend", "step"), dict(scale=float("inf")), 2, "finite"),
    (("attend", "step"), dict(out=None), 1, "NULL"),
    (("attend", "step"), dict(ws=8), 4, "16-byte"),
    (("attend", "step"), dict(B=1, NB=100, ws=None), 6, "workspace"),
    (("attend", "step"), dict(B=1, NB=100, wsb=16), 6, "workspace"),
])
def test_refusals(lib, names, kw, code, msg):
    for name in names:
        assert call(lib, name, **kw) == code, name
        assert any(m in lib.w4a8_last_error().decode() for m in msg.split("|")), (name, lib.w4a8_last_error())


def test_nothing_to_do(lib):
    for name in ALL:
        assert call(lib, name, B=0, k=None, vt=None, s=None, kt=None, vtt=None, qkv=None, q=None, out=None, pos=None, length=None) == 0
    for name in ("write", "attend"):
        assert call(lib, name, T=0, qkv=None, q=None, out=None, pos=None) == 0
    assert call(lib, "read", n=0, out=None, length=None) == 0


def test_workspace_bytes(lib):
    f = lambda *a: lib.w4a8_attention_kv8_workspace_bytes(*a, *((0, 0) if len(a) == 6 else ()))  # noqa: E731
    assert f(0, 1, 40, 8, 128, 20) == 0 and f(1, 0, 40, 8, 128, 20) == 0
    assert f(4096, 1, 40, 8, 128, 20) == 0                       # row tiles enough for every CU
    assert f(1, 1, 40, 8, 128, 512) % (40 * (128 + 4) * 4) == 0 and f(1, 1, 40, 8, 128, 512) > 0
    for bad in [(-1, 1, 40, 8, 128, 20), (1, -1, 40, 8, 128, 20), (1, 1, 40, 7, 128, 20), (1, 1, 40, 8, 96, 20),
                (1, 1, 40, 8, 128, 0), (1, 1, 40, 8, 128, 20, -1, 0), (1, 1, 40, 8, 128, 20, 0, -1)]:
        assert f(*bad) == -1


def test_workspace_bytes_extremes(lib):
    f = lib.w4a8_attention_kv8_workspace_bytes
    assert f(1, 1, 40, 8, 128, 512, 70, 2 ** 63 - 1) == f(1, 1, 40, 8, 128, 512, 70, 64 * 512)
    assert f(1, 1, 40, 8, 128, 512, 2 ** 63 - 1, 2 ** 63 - 1) == f(1, 1, 40, 8, 128, 512, 0, 0) > 0
    for bad in [(1, 1, 40, 8, 128, 2 ** 58, 0, 0), (2 ** 40, 1, 40, 8, 128, 20, 0, 0), (1, 2 ** 40, 40, 8, 128, 20, 0, 0),
                (1, 1, 2 ** 40, 8, 128, 20, 0, 0), (2 ** 20, 2 ** 20, 40, 8, 128, 20, 0, 0)]:
        assert f(*bad) == -1


def test_fakes(pkg):
    with torch.device("meta"):
        c = pkg.kv8.KV8Cache(2, 2, 100, 64, "fp8", device="meta")
        tab, pos = torch.empty((100, 32)), torch.empty((1,), dtype=torch.long)
        q = c.append(torch.empty((2, 7, 12 * 64), dtype=torch.bfloat16), tab, tab, pos, 8)
        assert q.shape == (2, 7, 8, 64) and q.dtype == torch.bfloat16
        assert c.attend(q, pos, 10, 2).shape == q.shape
        assert c.step(torch.empty((2, 12 * 64), dtype=torch.bfloat16), tab, tab, pos, 8).shape == (2, 1, 8, 64)
        k, v = c.read(pos)
        assert k.shape == v.shape == (2, 2, 100, 64) and k.dtype == torch.bfloat16


def test_cache_object(pkg):
    c = pkg.kv8.KV8Cache(3, 2, 65, 128, "int8", device="cpu")
    assert c.k_codes.shape == (3, 2, 2, 64, 128) and c.vt_codes.shape == (3, 2, 2, 128, 64) and c.k_codes.dtype == torch.int8
    # codes a byte an element, 8 bytes of scales a block, a bf16 block each of K and V
    assert c.nbytes == 3 * 2 * (2 * 2 * 64 * 128 + 2 * 8 + 2 * 64 * 128 * 2)
    for bad in [dict(dtype="int4"), dict(dtype=torch.bfloat16), dict(head_dim=96), dict(batch=0), dict(max_len=0)]:
        with pytest.raises(ValueError):
            pkg.kv8.KV8Cache(**{**dict(batch=1, kv_heads=1, max_len=64, head_dim=64, device="cpu"), **bad})


def test_cpu_tensors_raise(pkg):
    c = pkg.kv8.KV8Cache(1, 1, 64, 64, "int8", device="cpu")
    with pytest.raises(NotImplementedError):
        c.read(torch.zeros((1,), dtype=torch.long))


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_oracle_quantiser(dtype):
    """Against exact rational rounding, ties among the values, and torch's own e4m3 conversion."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn((4, 64, 64), generator=g).to(torch.bfloat16)
    x[1] *= 2.0 ** -126
    x[2, :, ::2] = (torch.arange(64 * 32) % 255).view(64, 32).to(torch.bfloat16)   # amax 254: x / 2, many ties
    x[2, :, 1::2] = 0
    x[3] = 0
    codes, scale = ok.quantise(x, dtype)
    top = ok.TOP[dtype]
    for b in range(4):
        amax = Fraction(float(x[b].abs().max()))
        assert float(scale[b]) == max(float(torch.tensor(float(amax)) / top), 2.0 ** -126)
        for v, c in list(zip(x[b].flatten().tolist(), codes[b].flatten().tolist()))[::7]:
            y = Fraction(v) * top / amax if amax else Fraction(0)
            if dtype == torch.int8:
                assert c == round(y)
            else:
                step = Fraction(1, 512)
                while abs(y) >= 16 * step:
                    step *= 2
                assert c == float(round(y / step) * step)
    if dtype != torch.int8:
        vals = torch.arange(256, dtype=torch.uint8).view(dtype).double()
        vals = vals[~torch.isnan(vals)]
        assert torch.equal(ok.round_e4m3(vals), vals)
        r = torch.randn((4096,), generator=g) * 100
        assert torch.equal(ok.round_e4m3(r.double()), r.to(dtype).double())


def test_oracle_attention():
    """attend against a plain loop with a window and sinks, a row that sees nothing, values of few positions."""
    g = torch.Generator().manual_seed(1)
    T, H, KVH, D, n = 5, 4, 2, 64, 9
    q = torch.randn((T, H, D), generator=g).to(torch.bfloat16)
    k, v = torch.randn((2, KVH, n, D), generator=g, dtype=torch.float64)
    p = torch.tensor([-1, 0, 3, 7, 8])
    for window, sinks in [(0, 0), (2, 0), (2, 3), (1, 20)]:
        out, bound = ok.attend(q, p, k, v, 0.3, window, sinks)
        for t in range(T):
            see = [i for i in range(n) if i <= p[t] and (not window or i > p[t] - window or i < sinks)]
            for h in range(H):
                if not see:
                    assert (out[t, h] == 0).all()
                    continue
                w = torch.softmax(torch.stack([(q[t, h].double() * k[h // 2, i]).sum() * 0.3 for i in see]), 0)
                assert torch.allclose(out[t, h], sum(w[j] * v[h // 2, i] for j, i in enumerate(see)), atol=1e-12)
        assert (bound >= 0).all()


@pytest.mark.parametrize("kw", [dict(kv_cache="int4"), dict(kv_cache="int8", attention="sdpa"), dict(window=5), dict(sinks=1),
                                dict(kv_cache="fp8", window=-1), dict(kv_cache="fp8", sinks=-1)], ids=str)
def test_decoder_refusals(pkg, kw):
    cfg = pkg.decoder.DecoderConfig(layers=1, hidden=64, heads=1, kv_heads=1, head_dim=64, ffn=64, vocab=10, group=64)
    with pytest.raises(ValueError):
        pkg.decoder.W4A8Decoder(cfg, batch=1, max_len=8, device="cpu", **kw)


@pytest.mark.parametrize("names,kw", [
    (("write",), dict(B=1 << 14, T=1 << 14, KVH=2, H=2, NB=1, L=64)),        # 2^26 waves of the queries
    (("write",), dict(B=1 << 20, T=1, KVH=8, H=8, NB=1, L=64, ldq=24 * 128)),  # 2^24 blocks of K and V
    (("read",), dict(B=1 << 16, KVH=2, NB=64, n=4096)),
    (("attend", "step"), dict(B=1 << 24, T=1, KVH=1, H=1, NB=1, L=64)),
    (("attend",), dict(B=1 << 23, T=20, KVH=1, H=1, NB=1, L=64)),              # two row tiles a sequence
])
def test_launch_limits(lib, names, kw):
    """Calls of 2^32 threads or more are refused by the library, before any launch."""
    for name in names:
        assert call(lib, name, **kw) == 5, (name, lib.w4a8_last_error())
        assert "too many workgroups" in lib.w4a8_last_error().decode()
