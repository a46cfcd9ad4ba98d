"""Refusals of the 16-bit operators, decided on the host before any CUDA call (no GPU needed)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

P16, P2, ODD = 0x10000, 0x10002, 0x10001   # addresses that no refused call follows
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 6


def _v(p):
    return C.c_void_p(p)


def _grouped(x=P16, w=P16, type=1, offs=P16, rows=P16, n=4, P=4, inn=64, out=32, E=2, y=P16, yt=1, ws=0, nb=0):
    from glmserve_b200._lib import lib
    return lib().gsb_grouped_gemm(_v(x), _v(w), type, _v(offs), _v(rows), n, P, inn, out, E, _v(y), yt, _v(ws), C.c_size_t(nb), None)


@pytest.mark.parametrize("kw,st", [
    (dict(P=0), OK), (dict(n=0, x=0), OK), (dict(type=0), INVALID), (dict(type=3), INVALID), (dict(yt=2), INVALID),
    (dict(yt=7), INVALID), (dict(n=-1), INVALID), (dict(P=-1), INVALID), (dict(inn=0), INVALID), (dict(out=0), INVALID),
    (dict(E=0), INVALID), (dict(rows=0, P=5), INVALID), (dict(x=0), INVALID), (dict(w=0), INVALID),
    (dict(offs=0), INVALID), (dict(y=0), INVALID), (dict(x=P2), INVALID), (dict(w=P2), INVALID), (dict(y=ODD), INVALID),
    (dict(y=P2, yt=0), INVALID), (dict(offs=P2), INVALID), (dict(rows=P2), INVALID),
    (dict(inn=60), UNSUPPORTED), (dict(E=1025), UNSUPPORTED), (dict(P=(1 << 30) + 1), UNSUPPORTED),
    (dict(inn=(1 << 30) + 8), UNSUPPORTED), (dict(out=(1 << 30) + 1), UNSUPPORTED),
    (dict(P=2000), INVALID), (dict(P=2000, ws=P16 + 16, nb=1 << 30), INVALID), (dict(P=2000, ws=P16, nb=64), WORKSPACE)])
def test_grouped_gemm_refusals(kw, st):
    assert _grouped(**kw) == st


def _ffn(x=P16, ids=P16, wt=P16, g=P16, u=P16, d=P16, type=2, n=4, topk=2, H=64, I=32, E=4, out=P16, ot=2, ws=P16, nb=1 << 30):
    from glmserve_b200._lib import lib
    return lib().gsb_moe_expert_ffn_w16(_v(x), _v(ids), _v(wt), _v(g), _v(u), _v(d), type, n, topk, H, I, E, _v(out), ot,
                                        _v(ws), C.c_size_t(nb), None)


@pytest.mark.parametrize("kw,st", [
    (dict(n=0), OK), (dict(type=0), INVALID), (dict(ot=1), INVALID), (dict(n=-1), INVALID), (dict(topk=0), INVALID),
    (dict(H=0), INVALID), (dict(I=0), INVALID), (dict(E=0), INVALID), (dict(x=0), INVALID), (dict(ids=0), INVALID),
    (dict(wt=0), INVALID), (dict(g=0), INVALID), (dict(u=0), INVALID), (dict(d=0), INVALID), (dict(out=0), INVALID),
    (dict(ws=0), INVALID), (dict(ws=P16 + 16), INVALID), (dict(g=P2), INVALID), (dict(out=P2), INVALID),
    (dict(H=60), UNSUPPORTED), (dict(I=36), UNSUPPORTED), (dict(E=1025), UNSUPPORTED),
    (dict(n=1 << 30, topk=2), UNSUPPORTED), (dict(H=(1 << 30) + 8), UNSUPPORTED), (dict(I=(1 << 30) + 8), UNSUPPORTED), (dict(nb=64), WORKSPACE)])
def test_ffn_refusals(kw, st):
    assert _ffn(**kw) == st


def _lora(x=P16, A=P16, B=P16, type=1, offs=P16, rows=P16, ranks=0, scales=0, n=4, P=4, inn=64, out=32, nA=2, R=8,
          y=2 * P16, yt=0, sc=P16, nb=1 << 30):
    from glmserve_b200._lib import lib
    return lib().gsb_lora_add(_v(x), _v(A), _v(B), type, _v(offs), _v(rows), _v(ranks), _v(scales), n, P, inn, out, nA, R,
                              _v(y), yt, _v(sc), C.c_size_t(nb), None)


@pytest.mark.parametrize("kw,st", [
    (dict(P=0), OK), (dict(type=0), INVALID), (dict(yt=2), INVALID), (dict(n=-1, P=-1), INVALID), (dict(P=5), INVALID),
    (dict(inn=0), INVALID), (dict(out=0), INVALID), (dict(nA=0), INVALID), (dict(R=0), INVALID), (dict(x=0), INVALID),
    (dict(A=0), INVALID), (dict(B=0), INVALID), (dict(offs=0), INVALID), (dict(rows=0), INVALID), (dict(y=0), INVALID), (dict(y=P16), INVALID),
    (dict(x=P2), INVALID), (dict(A=P2), INVALID), (dict(B=ODD), INVALID), (dict(y=P2), INVALID), (dict(ranks=P2), INVALID),
    (dict(scales=P2), INVALID), (dict(n=9999, P=9999, sc=0), INVALID), (dict(n=9999, P=9999, sc=P16 + 16), INVALID),
    (dict(inn=60), UNSUPPORTED), (dict(R=257), UNSUPPORTED), (dict(nA=1025), UNSUPPORTED), (dict(inn=(1 << 30) + 8), UNSUPPORTED),
    (dict(out=(1 << 30) + 1), UNSUPPORTED), (dict(n=(1 << 30) + 1, P=(1 << 30) + 1), UNSUPPORTED), (dict(n=9999, P=9999, nb=64), WORKSPACE)])
def test_lora_refusals(kw, st):
    assert _lora(**kw) == st


def test_sizes():
    from glmserve_b200._lib import lib
    L = lib()
    assert L.gsb_moe_expert_ffn_w16_workspace_bytes(0, 8, 64, 64, 4) == 0
    small, large = (L.gsb_moe_expert_ffn_w16_workspace_bytes(n, 8, 6144, 2048, 32) for n in (64, 8192))
    assert 64 * 8 * (2 * 2048 + 4 * 6144) <= small < large and large >= 8192 * 8 * (2 * 2048 + 4 * 6144)
    assert L.gsb_grouped_gemm_workspace_bytes(8, 6144, 32) == 0 and L.gsb_grouped_gemm_workspace_bytes(8192, 6144, 8) == 8192 * 6144 * 2
    assert L.gsb_lora_scratch_bytes(0, 16, 4) == 0 and L.gsb_lora_scratch_bytes(8192, 64, 8) >= 8192 * 64 * 4


def test_python_refuses_wrong_tensors():
    from glmserve_b200 import ops
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ops.grouped_gemm(x, x, i), lambda: ops.moe_expert_ffn_w16(x, i, x, x, x, x),
                 lambda: ops.lora_add(x, x, x, x, i, i)):
        with pytest.raises(ValueError, match="expected"):
            call()


def test_ffn_refuses_what_its_last_launch_could_not_cover():
    """256 tokens or more of over 65535 * 4096 features: before anything is launched (fewer tokens: no such limit)."""
    assert _ffn(n=256, H=65535 * 4096 + 8, nb=1 << 62) == 7
    assert _ffn(n=255, H=65535 * 4096 + 8) == WORKSPACE and _ffn(n=256, H=65535 * 4096) == WORKSPACE


FAR = 1 << 40       # the other buffers, away from the pair that shares memory


@pytest.mark.parametrize("kw", [
    dict(x=P16), dict(x=P16 + 48), dict(x=P16 - 512 + 16), dict(w=P16 - 2 * 32 * 64 * 2 + 16), dict(w=P16 + 192, rows=0),
    dict(offs=P16 + 4), dict(rows=P16 + 252), dict(y=P16 + 2, x=P16 - 496), dict(yt=0, x=P16 + 496),
    dict(x=8 * FAR - (1 << 30) * 8 * 2 + 16, n=1 << 30, inn=8, y=8 * FAR), dict(w=P16 + 16, inn=1 << 30, out=1 << 30, E=1024)])
def test_grouped_gemm_refuses_a_result_over_its_inputs(kw):
    """y: four rows of 32, 256 bytes from P16 (512 in fp32)."""
    far = dict(x=FAR, w=2 * FAR, offs=3 * FAR, rows=4 * FAR, y=P16)
    assert _grouped(**{**far, **kw}) == INVALID


@pytest.mark.parametrize("kw", [dict(ids=P16 + 508), dict(wt=P16), dict(wt=P16 - 28), dict(ot=0, wt=P16 + 1020)])
def test_ffn_refuses_a_result_over_its_ids_or_weights(kw):
    far = dict(x=FAR, ids=2 * FAR, wt=3 * FAR, g=4 * FAR, u=5 * FAR, d=6 * FAR, ws=7 * FAR, out=P16)
    assert _ffn(**{**far, **kw}) == INVALID


@pytest.mark.parametrize("kw", [
    dict(x=P16), dict(x=P16 + 496), dict(x=P16 - 496), dict(A=P16 + 16), dict(A=P16 - 2 * 8 * 64 * 2 + 16), dict(B=P16 + 510),
    dict(offs=P16), dict(rows=P16 + 508), dict(ranks=P16 + 4), dict(scales=P16 - 4), dict(yt=1, B=P16 + 254)])
def test_lora_refuses_a_result_over_its_inputs(kw):
    """y: four rows of 32 in fp32, 512 bytes from P16 (256 in 16 bits)."""
    far = dict(x=FAR, A=2 * FAR, B=3 * FAR, offs=4 * FAR, rows=5 * FAR, sc=6 * FAR, y=P16)
    assert _lora(**{**far, **kw}) == INVALID
