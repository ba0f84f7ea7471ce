"""qk_norm_rope: a head's output depends on that head alone, not on the heads that share its warp nor on
what was left where the heads of a step that do not exist would be."""
import pytest
import torch

import tqkv

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _rand(shape, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _call(q, k, interleaved=False):
    T, D = q.shape[2], q.shape[3]
    pos = torch.arange(T, dtype=torch.int32, device="cuda").expand(q.shape[0], T).contiguous()
    return tqkv.qk_norm_rope(q, k, pos, tqkv.rope_table(T, D), interleaved=interleaved)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (2, 1), (3, 2), (14, 2), (5, 3)])
def test_calls_repeat_whatever_ran_before(Hq, Hkv, D, dtype):
    """Between the calls, others of full steps leave rows of zeros, ordinary rows, rows whose squares
    overflow and NaN in every warp's buffer."""
    T = 1500
    q, k = _rand((1, Hq, T, D), 1, dtype), _rand((1, Hkv, T, D), 2, dtype)
    fills = [torch.full((1, 512 // D, 9000, D), v, dtype=dtype, device="cuda")
             for v in (1.0, 0.0, float("inf"), float("nan"))]
    got = []
    for f in fills:
        _call(f, f)
        got.append(_call(q, k))
    for other in got[1:]:
        assert torch.equal(other[0], got[0][0]) and torch.equal(other[1], got[0][1])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("beside", [0.0, 1e-19, 3e4, float("nan")])
def test_a_head_beside_others_is_the_head_alone(D, dtype, interleaved, beside):
    """Neighbours without elements, with squares outside fp32's range or with NaN."""
    T, H = 1500, 8
    x = _rand((1, H, T, D), 3, dtype)
    alone = [_call(x[:, h:h + 1].contiguous(), x[:, h:h + 1].contiguous(), interleaved)[0] for h in range(H)]
    odd = (1, 4, 6)
    x[:, list(odd)] = beside
    q, k = _call(x, x, interleaved)
    assert torch.equal(q, k) or beside != beside
    for h in range(H):
        if h not in odd:
            assert torch.equal(q[:, h], alone[h][:, 0]) and torch.equal(k[:, h], alone[h][:, 0]), h
