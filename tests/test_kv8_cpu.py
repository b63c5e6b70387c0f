"""The 8-bit cache's entry points without a GPU: the C ABI's refusals and sizes,
the Python entry points' checks, the definition's own rounding."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

import kv8_reference as ref

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
D = C.c_void_p(16)  # never dereferenced: every call below is refused first
ODD = C.c_void_p(24)


@pytest.fixture(scope="module")
def lib(tq4):
    return tq4.kv8._lib()


def test_every_declared_symbol_is_exported(lib):
    text = open(os.path.join(REPO, "include", "tq4_kv8.h")).read()
    names = set(re.findall(r"\b(tq4_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert len(names) == 7
    for n in names:
        assert hasattr(lib, n), n
    assert lib.tq4_status_string(-14) != b"unknown status"


def test_plan_refusals(lib):
    def call(B=4, M=8, S=16, P=32, T=64, ws=D, n=None, ptr=D):
        n = lib.tq4_paged_plan_workspace_bytes(B) if n is None else n
        return lib.tq4_paged_plan(None, D, D, None, D, D, D, D, None, ptr, D, D, D, ws, n, B, M, S,
                                  P, T)
    assert call(B=0) == call(M=0) == call(P=0) == call(S=0) == call(S=24) == -3
    assert call(P=2 ** 28) == call(B=2 ** 16, M=2 ** 15) == call(T=2 ** 31) == -10
    assert call(ptr=None) == -1
    assert call(ws=None) == call(n=100) == call(ws=ODD) == -6


def test_writer_refusals(lib):
    def call(el=1, code=0, key=D, ks=256, vs=256, T=4, H=2, d=128, S=16, P=8, kc=D):
        return lib.tq4_kv8_reshape_and_cache(None, el, code, key, D, kc, D, D, D, ks, vs, T, H, d,
                                             S, P)
    assert call(d=96) == -2
    assert call(el=2) == call(code=2) == call(H=0) == call(P=0) == call(S=24) == call(S=1040) == -3
    assert call(ks=128) == call(vs=248) == -3
    assert call(P=2 ** 28) == call(T=2 ** 27, H=1) == call(H=8193) == -10
    assert call(key=None) == -1
    assert call(key=ODD) == call(kc=ODD) == call(ks=260) == -14
    assert call(T=0) == 0


def test_attention_refusals_and_sizes(lib):
    def dec(el=0, code=1, q=D, ws=None, n=0, qs=1024, B=2, Hq=8, H=2, d=128, S=16, P=64, M=64, K=1,
            out=D):
        return lib.tq4_kv8_paged_decode(None, el, code, q, D, D, D, D, D, ws, n, out, qs, B, Hq, H,
                                        d, S, P, M, K, 0.1)

    def pre(cu=D, T=9, B=2, Hq=8, H=2, M=64, longest=4, ws=None, n=0, S=16):
        return lib.tq4_kv8_paged_prefill(None, 1, 0, D, D, D, D, D, D, cu, ws, n, D, 1024, T, B,
                                         Hq, H, 128, S, 64, M, longest, 1, 0.1)
    assert dec(d=32) == -2
    assert dec(Hq=9) == dec(Hq=34) == dec(Hq=0) == dec(M=0) == dec(el=3) == dec(qs=512) == -3
    assert dec(K=257) == -5
    assert dec(M=2 ** 28) == dec(P=2 ** 28) == -10
    # the join's rows: workgroups of 1024 behind more than 32 parts
    many = dict(B=2 ** 18 - 1, Hq=17, H=17, qs=17 * 128, M=8)
    assert dec(K=33, **many) == -10 and dec(K=32, **many) == -6
    assert dec(q=None) == dec(out=None) == pre(cu=None) == -1
    assert dec(q=ODD) == dec(qs=1028) == -14
    need = lib.tq4_kv8_decode_workspace_bytes(2, 8, 2, 128, 16, 64, 4)
    assert need >= 2 * 8 * 4 * (128 + 2) * 4
    assert dec(K=4) == dec(K=4, ws=D, n=need - 1) == dec(K=4, ws=ODD, n=need) == -6
    assert lib.tq4_kv8_decode_workspace_bytes(2, 8, 2, 128, 16, 64, 1) == 0
    assert dec(B=0) == pre(B=0) == pre(T=0) == pre(longest=0) == 0
    # a longest of more rows than there are is the rows
    assert (lib.tq4_kv8_prefill_workspace_bytes(9, 2, 8, 2, 128, 16, 64, 4000) ==
            lib.tq4_kv8_prefill_workspace_bytes(9, 2, 8, 2, 128, 16, 64, 9))
    # the sizes of many geometries do not wrap
    for n in (1, 1000, 2 ** 31 - 1):
        assert lib.tq4_kv8_decode_workspace_bytes(n, 2 ** 31, 8, 256, 16, 2 ** 27, 256) >= n


def operands(**over):
    P, H, S, d, B, Hq, M = 6, 2, 16, 64, 3, 4, 2
    a = dict(q=torch.zeros(B, Hq, d, dtype=torch.bfloat16),
             key_cache=torch.zeros(P, H, S, d, dtype=torch.int8),
             value_cache=torch.zeros(P, H, S // 16, d, 16, dtype=torch.int8),
             scale_cache=torch.zeros(2, P, H), tables=torch.zeros(B, M, dtype=torch.int32),
             lens=torch.zeros(B, dtype=torch.int32), out=None)
    a.update(over)
    return a


def decode(tq4, **over):
    a = operands(**over)
    return tq4.kv8_paged_decode(a["q"], a["key_cache"], a["value_cache"], a["scale_cache"],
                                a["tables"], a["lens"], out=a["out"])


@pytest.mark.parametrize("over,match", [
    (dict(q=torch.zeros(3, 4, 64)), "q must be float16 or bfloat16"),
    (dict(q=torch.zeros(3, 256, dtype=torch.bfloat16)), "q must have 3 dimensions"),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), "head size"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), "2 rows of q for 3"),
    (dict(q=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), "rows of q"),
    (dict(q=torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(3, 4, 64)), "rows of q"),
    (dict(key_cache=torch.zeros(6, 2, 16, 64)), "key_cache must be"),
    (dict(key_cache=torch.zeros(6, 2, 1024, dtype=torch.int8)), "key_cache must have 4"),
    (dict(value_cache=torch.zeros(6, 2, 1, 64, 16).to(torch.float8_e4m3fn)), "value_cache must be"),
    (dict(value_cache=torch.zeros(100, dtype=torch.int8)), "value_cache must hold"),
    (dict(scale_cache=torch.zeros(6, 2)), "scale_cache must hold"),
    (dict(tables=torch.zeros(3, 2, dtype=torch.int64)), "block_tables must be"),
    (dict(lens=torch.zeros(4, dtype=torch.int32)), "context_lens must hold"),
    (dict(out=torch.zeros(3, 4, 64)), "out must be"),
    (dict(), "must be a device tensor"),
])
def test_decode_operands(tq4, over, match):
    with pytest.raises(ValueError, match=match):
        decode(tq4, **over)


def test_prefill_operands(tq4):
    a = operands()
    args = (a["q"], a["key_cache"], a["value_cache"], a["scale_cache"], a["tables"], a["lens"])
    with pytest.raises(ValueError, match="must be a device tensor"):
        tq4.kv8_paged_prefill(*args, torch.zeros(4, dtype=torch.int32), 2)


def test_writer_operands(tq4):
    a = operands()
    k = torch.zeros(5, 2, 64, dtype=torch.float16)
    s = torch.zeros(5, dtype=torch.int32)

    def call(k=k, v=k, s=s, kc=a["key_cache"]):
        tq4.kv8_reshape_and_cache(k, v, kc, a["value_cache"], a["scale_cache"], s)
    with pytest.raises(ValueError, match="value must be float16"):
        call(v=k.bfloat16())
    with pytest.raises(ValueError, match="key's shape"):
        call(v=k[:4])
    with pytest.raises(ValueError, match="key has rows"):
        call(k=k[:, :1].contiguous(), v=k[:, :1].contiguous())
    with pytest.raises(ValueError, match="slot_mapping must hold at least 5"):
        call(s=s[:4])
    with pytest.raises(ValueError, match="must be a device tensor"):
        call()


def test_plan_operands(tq4):
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731

    def call(ctx=i(3), tables=i(3, 4), ring=i(9), state=i(2), cu=i(4), slots=i(5), pos=None):
        tq4.paged_plan(ctx, i(3), tables, ring, state, slots, cu, i(3), 16, positions=pos)
    for over, match in ((dict(ctx=i(4)), "context_lens must hold 3"),
                        (dict(tables=i(12)), "block_tables must have 2"),
                        (dict(state=i(3)), "free_state must hold 2"),
                        (dict(cu=i(3)), "cu_seqlens must hold 4"),
                        (dict(pos=i(6)), "positions must hold 5"),
                        (dict(slots=i(5).long()), "slot_mapping must be int32"),
                        (dict(), "must be a device tensor")):
        with pytest.raises(ValueError, match=match):
            call(**over)


def test_cache_shapes(tq4):
    k, v, s = tq4.kv8_cache(5, 2, 48, 64, device="cpu")
    assert k.shape == (5, 2, 48, 64) and v.shape == (5, 2, 3, 64, 16) and s.shape == (2, 5, 2)
    assert k.dtype == v.dtype == torch.float8_e4m3fn
    for kw in (dict(dtype=torch.float16), dict(block_size=24)):
        with pytest.raises(ValueError):
            tq4.kv8_cache(5, 2, kw.get("block_size", 16), 64, kw.get("dtype", torch.int8), "cpu")


def test_definition_rounds_as_torch():
    """The tests' e4m3 rounding against torch's conversion."""
    x = torch.cat([torch.randn(5000) * 100, torch.randn(5000) * 0.01,
                   torch.tensor([0.0, -0.0, 448.0, 464.0, 1e9, -1e9])]).clamp(-448, 448)
    assert np.array_equal(ref.to_codes(x.numpy(), "fp8"),
                          x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_torch_ops_schemas_and_fakes(tq4):
    ops = torch.ops.tq4
    m = lambda *s, dtype=torch.int32: torch.empty(s, dtype=dtype, device="meta")  # noqa: E731
    assert str(ops.paged_plan.default._schema).count("!") == 8
    w = str(ops.kv8_reshape_and_cache.default._schema)
    assert "Tensor(a2!) key_cache" in w and "Tensor(a4!) scale_cache" in w and w.endswith("-> ()")
    c = (m(9, 2, 16, 64, dtype=torch.int8), m(9, 2, 1, 64, 16, dtype=torch.int8),
         m(2, 9, 2, dtype=torch.float32))
    q = m(7, 8, 64, dtype=torch.float16)
    for out in (ops.kv8_paged_decode(q, *c, m(7, 3), m(7), 0, 0.0),
                ops.kv8_paged_prefill(q, *c, m(2, 3), m(2), m(3), 4, True, 0.0)):
        assert out.shape == q.shape and out.dtype == q.dtype and out.device.type == "meta"
    with pytest.raises(NotImplementedError):
        ops.kv8_paged_decode(*[torch.zeros(x.shape, dtype=x.dtype) for x in (q, *c, m(7, 3), m(7))],
                             0, 0.0)
