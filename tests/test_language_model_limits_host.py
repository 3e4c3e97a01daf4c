"""Host side of the language model operators: what they refuse besides wrong extents and types."""
import ctypes as C

import pytest

from flashlight_b200 import _lib as L


@pytest.mark.parametrize("off", [1, 8, 16, 24])
def test_linear_cce_gradient_refuses_a_workspace_off_32_bytes(off):
    """It stores the scores' gradient 32 bytes at a time at multiples of 256 from the workspace's start."""
    d = L.LinearCceDesc(rows=4, features=8, classes=16, reduction=L.REDUCE_MEAN, ignore_index=-1, dtype=L.BF16)
    assert L.lib.flb200_linear_cce_backward(C.byref(d), 16, 16, None, 16, 16, 16, 16, 16, 16, L.BF16, None, 4096 + off,
                                            1 << 40, None) == L.WORKSPACE_TOO_SMALL
    assert b"32-byte aligned" in L.lib.flb200_last_error()


# ---------------------------------------------------------------------- tensors of several devices
@pytest.fixture
def fake(monkeypatch):
    """Tensors of any device without memory; a call that looks further than their devices finds no GPU here."""
    import torch
    import torch._subclasses.fake_tensor as ft
    monkeypatch.setattr(ft, "init_gpu_context", lambda device: None)
    mode = ft.FakeTensorMode()

    def make(*shape, dtype=torch.bfloat16, device="cuda:0"):
        with mode:
            return torch.empty(shape, dtype=dtype, device=device)

    return make


def test_attention_refuses_tensors_of_several_devices(fake):
    import torch
    from flashlight_b200 import functions as F
    mask = F.AttentionMask(1, 16, 16, True, None, None)
    table = int(L.lib.flb200_attention_mask_bytes(1, 16, 16))
    there = lambda t: fake(*t.shape, dtype=t.dtype, device="cuda:1")  # noqa: E731
    x, lse = fake(1, 16, 4, 64), fake(1, 4, 16, dtype=torch.float32)
    slopes = fake(4, dtype=torch.float32)
    for i in range(3):
        q = [x, x, x]
        q[i] = there(x)
        with pytest.raises(ValueError, match="one device"):
            F.masked_attention(*q, mask, 1.0)
    for other in (F.AttentionMask(1, 16, 16, True, fake(1, dtype=torch.int32, device="cuda:1"), None),
                  F.AttentionMask(1, 16, 16, True, None, fake(table, dtype=torch.uint8, device="cuda:1"))):
        with pytest.raises(ValueError, match="one device"):
            F.masked_attention(x, x, x, other, 1.0)
    with pytest.raises(ValueError, match="one device"):
        F.masked_attention(x, x, x, mask, 1.0, 0.0, there(slopes))
    ids = fake(1, 16, dtype=torch.int32)
    with pytest.raises(ValueError, match="one device"):
        F.attention_mask(1, 16, documents=ids, prefix=fake(1, dtype=torch.int32, device="cuda:1"))
    good = [x, x, x, lse, None, None, None]  # out, rest, the output's gradient, lse, and the gradients
    for i, t in enumerate([x, x, x, lse, x, x, x]):
        bad = list(good)
        bad[i] = there(t)
        with pytest.raises(ValueError, match="one device"):
            F.masked_attention_backward(x, x, x, bad[0], bad[1], bad[2], bad[3], mask, 1.0, grads=bad[4:])


def test_loss_refuses_tensors_of_several_devices(fake):
    import torch
    from flashlight_b200 import functions as F
    x, w, b = fake(8, 64), fake(64, 512), fake(512, dtype=torch.float32)
    t, lse, gl = fake(8, dtype=torch.int32), fake(8, dtype=torch.float32), fake(1, dtype=torch.float32)
    meta = fake(2, dtype=torch.int32)
    there = lambda t: fake(*t.shape, dtype=t.dtype, device="cuda:1")  # noqa: E731
    for i in range(1, 4):
        bad = [x, w, b, t]
        bad[i] = there(bad[i])
        with pytest.raises(ValueError, match="one device"):
            F.linear_cross_entropy(*bad)
    for i in range(1, 7):
        bad = [x, w, b, lse, gl, t, meta]
        bad[i] = there(bad[i])
        with pytest.raises(ValueError, match="one device"):
            F.linear_cross_entropy_backward(*bad[:5], F.CrossEntropyState(bad[5], bad[6], L.REDUCE_MEAN, -1))


@pytest.mark.parametrize("off", [1, 2, 3])
def test_attention_gradient_refuses_a_workspace_off_4_bytes(off):
    d = L.AttentionDesc(batch=1, q_len=4, k_len=4, heads=4, kv_heads=2, head_dim=64, scale=1.0, softcap=0.0, dtype=L.F16)
    t = C.byref(L.HeadTensor(16, 1024, 256, 64))
    assert L.lib.flb200_masked_attention_backward(C.byref(d), t, t, t, t, None, t, 16, None, None, t, t, t, 4096 + off,
                                                  1 << 40, None) == L.WORKSPACE_TOO_SMALL
    assert b"4-byte aligned" in L.lib.flb200_last_error()
