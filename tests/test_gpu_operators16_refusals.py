"""Every check of arguments that the Python entry points of the 16-bit operators make: one wrong property a call, on CUDA
tensors (the library behind them takes addresses and sizes and cannot see what a tensor is)."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF, HF, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _z(dev, shape, dtype, **kw):
    return torch.zeros(shape, dtype=dtype, device=dev, **kw)


def _gaps(t):
    """The same shape and type, not contiguous."""
    return torch.stack([t, t], dim=-1)[..., 0]


def _refused(call, good, change):
    from glmserve_b200._lib import GsbError
    call(**good)                                    # the call is right without the change
    with pytest.raises((ValueError, GsbError)):
        call(**{**good, **change(good)})


n, K, N, E, P, H, I, T = 12, 64, 40, 3, 20, 64, 24, 2


def _grouped(dev):
    return dict(x=_z(dev, (n, K), BF), w=_z(dev, (E, N, K), BF), expert_offsets=_z(dev, (E + 1,), I32), rows=_z(dev, (P,), I32),
                out=_z(dev, (P, N), BF))


GROUPED = {
    "x fp32": lambda a: dict(x=a["x"].float(), w=a["w"].float()),
    "x of another type than w": lambda a: dict(x=a["x"].half()),
    "x on the CPU": lambda a: dict(x=a["x"].cpu()),
    "x with gaps": lambda a: dict(x=_gaps(a["x"])),
    "x of one dimension": lambda a: dict(x=a["x"][0]),
    "x of another K": lambda a: dict(x=a["x"][:, :56].contiguous()),
    "K not a multiple of 8": lambda a: dict(x=a["x"][:, :60].contiguous(), w=a["w"][..., :60].contiguous()),
    "w on the CPU": lambda a: dict(w=a["w"].cpu()),
    "w with gaps": lambda a: dict(w=_gaps(a["w"])),
    "w transposed": lambda a: dict(w=a["w"].transpose(1, 2)),
    "w of two dimensions": lambda a: dict(w=a["w"][0]),
    "w of more experts": lambda a: dict(w=torch.cat([a["w"], a["w"]])),
    "offsets int64": lambda a: dict(expert_offsets=a["expert_offsets"].long()),
    "offsets on the CPU": lambda a: dict(expert_offsets=a["expert_offsets"].cpu()),
    "offsets short": lambda a: dict(expert_offsets=a["expert_offsets"][:-1]),
    "offsets with gaps": lambda a: dict(expert_offsets=_gaps(a["expert_offsets"])),
    "offsets of two dimensions": lambda a: dict(expert_offsets=a["expert_offsets"][None]),
    "rows int64": lambda a: dict(rows=a["rows"].long()),
    "rows on the CPU": lambda a: dict(rows=a["rows"].cpu()),
    "rows with gaps": lambda a: dict(rows=_gaps(a["rows"])),
    "rows of two dimensions": lambda a: dict(rows=a["rows"][:, None]),
    "out of fewer rows": lambda a: dict(out=a["out"][:-1]),
    "out of other columns": lambda a: dict(out=a["out"][:, :-1].contiguous()),
    "out of the other 16-bit type": lambda a: dict(out=a["out"].half()),
    "out fp64": lambda a: dict(out=a["out"].double()),
    "out on the CPU": lambda a: dict(out=a["out"].cpu()),
    "out with gaps": lambda a: dict(out=_gaps(a["out"])),
    "out and another out_dtype": lambda a: dict(out_dtype=F32),
    "out_dtype of the other 16-bit type": lambda a: dict(out=None, out_dtype=HF),
    "out_dtype fp64": lambda a: dict(out=None, out_dtype=torch.float64),
    "x off the 16-byte border": lambda a: dict(x=_z(a["x"].device, (n * K + 1,), BF)[1:].view(n, K)),
    "w off the 16-byte border": lambda a: dict(w=_z(a["x"].device, (E * N * K + 1,), BF)[1:].view(E, N, K)),
}


@pytest.mark.parametrize("name", GROUPED)
def test_grouped_gemm_refuses(dev, name):
    from glmserve_b200 import ops
    _refused(ops.grouped_gemm, _grouped(dev), GROUPED[name])


def _ffn(dev):
    return dict(x=_z(dev, (n, H), HF), topk_ids=_z(dev, (n, T), I32), topk_w=_z(dev, (n, T), F32), gate_w=_z(dev, (E, I, H), HF),
                up_w=_z(dev, (E, I, H), HF), down_w=_z(dev, (E, H, I), HF), out=_z(dev, (n, H), HF))


FFN = {
    "all fp32": lambda a: {k: a[k].float() for k in ("x", "gate_w", "up_w", "down_w", "out")},
    "x of another type": lambda a: dict(x=a["x"].bfloat16()),
    "x on the CPU": lambda a: dict(x=a["x"].cpu()),
    "x with gaps": lambda a: dict(x=_gaps(a["x"])),
    "x of another width": lambda a: dict(x=a["x"][:, :56].contiguous()),
    "ids int64": lambda a: dict(topk_ids=a["topk_ids"].long()),
    "ids of one dimension": lambda a: dict(topk_ids=a["topk_ids"][:, 0].contiguous()),
    "ids of fewer tokens": lambda a: dict(topk_ids=a["topk_ids"][:-1]),
    "ids with gaps": lambda a: dict(topk_ids=_gaps(a["topk_ids"])),
    "ids on the CPU": lambda a: dict(topk_ids=a["topk_ids"].cpu()),
    "weights of the activations' type": lambda a: dict(topk_w=a["topk_w"].half()),
    "weights of fewer slots": lambda a: dict(topk_w=a["topk_w"][:, :1].contiguous()),
    "weights with gaps": lambda a: dict(topk_w=_gaps(a["topk_w"])),
    "no slot": lambda a: dict(topk_ids=a["topk_ids"][:, :0], topk_w=a["topk_w"][:, :0]),
    "gate of another type": lambda a: dict(gate_w=a["gate_w"].bfloat16()),
    "gate with gaps": lambda a: dict(gate_w=_gaps(a["gate_w"])),
    "gate of fewer experts": lambda a: dict(gate_w=a["gate_w"][:-1]),
    "up of fewer features": lambda a: dict(up_w=a["up_w"][:, :16].contiguous()),
    "up on the CPU": lambda a: dict(up_w=a["up_w"].cpu()),
    "down not transposed": lambda a: dict(down_w=a["gate_w"]),
    "down transposed in place": lambda a: dict(down_w=a["gate_w"].transpose(1, 2)),
    "down of more experts": lambda a: dict(down_w=torch.cat([a["down_w"], a["down_w"]])),
    "out of fewer tokens": lambda a: dict(out=a["out"][:-1]),
    "out of the other 16-bit type": lambda a: dict(out=a["out"].bfloat16()),
    "out with gaps": lambda a: dict(out=_gaps(a["out"])),
    "out_dtype of the other 16-bit type": lambda a: dict(out=None, out_dtype=BF),
    "gate off the 16-byte border": lambda a: dict(gate_w=_z(a["x"].device, (E * I * H + 1,), HF)[1:].view(E, I, H)),
    "out off the 16-byte border": lambda a: dict(out=_z(a["x"].device, (n * H + 1,), HF)[1:].view(n, H)),
}


@pytest.mark.parametrize("name", FFN)
def test_expert_ffn_refuses(dev, name):
    from glmserve_b200 import ops
    _refused(ops.moe_expert_ffn_w16, _ffn(dev), FFN[name])


R = 8


def _lora(dev):
    return dict(y=_z(dev, (n, N), F32), x=_z(dev, (n, K), BF), A=_z(dev, (E, R, K), BF), B=_z(dev, (E, N, R), BF),
                adapter_offsets=_z(dev, (E + 1,), I32), rows=_z(dev, (n,), I32), ranks=_z(dev, (E,), I32), scales=_z(dev, (E,), F32))


LORA = {
    "no y": lambda a: dict(y=None),
    "y of fewer rows": lambda a: dict(y=a["y"][:-1]),
    "y of other columns": lambda a: dict(y=a["y"][:, :-1].contiguous()),
    "y with gaps": lambda a: dict(y=_gaps(a["y"])),
    "y on the CPU": lambda a: dict(y=a["y"].cpu()),
    "y of the other 16-bit type": lambda a: dict(y=a["y"].half()),
    "x fp32": lambda a: dict(x=a["x"].float()),
    "x of another type than A": lambda a: dict(x=a["x"].half()),
    "x of another K": lambda a: dict(x=a["x"][:, :56].contiguous()),
    "x with gaps": lambda a: dict(x=_gaps(a["x"])),
    "A of another type": lambda a: dict(A=a["A"].half()),
    "A transposed": lambda a: dict(A=a["A"].transpose(1, 2)),
    "A of fewer adapters": lambda a: dict(A=a["A"][:-1]),
    "A of another rank": lambda a: dict(A=a["A"][:, :4].contiguous()),
    "B of another type": lambda a: dict(B=a["B"].half()),
    "B of fewer adapters": lambda a: dict(B=a["B"][:-1]),
    "B of other columns": lambda a: dict(B=a["B"][:, :-1].contiguous()),
    "B with gaps": lambda a: dict(B=_gaps(a["B"])),
    "B on the CPU": lambda a: dict(B=a["B"].cpu()),
    "rank 257": lambda a: dict(A=_z(a["x"].device, (E, 257, K), BF), B=_z(a["x"].device, (E, N, 257), BF)),
    "offsets short": lambda a: dict(adapter_offsets=a["adapter_offsets"][:-1]),
    "offsets int64": lambda a: dict(adapter_offsets=a["adapter_offsets"].long()),
    "rows int64": lambda a: dict(rows=a["rows"].long()),
    "rows of two dimensions": lambda a: dict(rows=a["rows"][:, None]),
    "more rows than x has": lambda a: dict(rows=torch.cat([a["rows"], a["rows"]])),
    "rows on the CPU": lambda a: dict(rows=a["rows"].cpu()),
    "ranks short": lambda a: dict(ranks=a["ranks"][:-1]),
    "ranks int64": lambda a: dict(ranks=a["ranks"].long()),
    "ranks on the CPU": lambda a: dict(ranks=a["ranks"].cpu()),
    "scales short": lambda a: dict(scales=a["scales"][:-1]),
    "scales of the activations' type": lambda a: dict(scales=a["scales"].bfloat16()),
    "scales of two dimensions": lambda a: dict(scales=a["scales"][:, None]),
}


@pytest.mark.parametrize("name", LORA)
def test_lora_refuses(dev, name):
    from glmserve_b200 import ops
    _refused(ops.lora_add, _lora(dev), LORA[name])
