"""The gradient of masked attention through the C entry point, with workspaces on every alignment that it accepts: the
same bits, and nothing written in front of or behind the bytes that it asks for."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H", [(1, 1), (33, 3), (129, 5), (3001, 2)])
def test_any_alignment(dtype, T, H):
    from flashlight_b200 import _lib as L
    from flashlight_b200 import functions as F
    D = 64
    g = torch.Generator("cuda").manual_seed(T)
    q, k, v, go = ((torch.randn(1, T, H, D, generator=g, device="cuda") * 0.01).to(dtype) for _ in range(4))
    mask = F.attention_mask(1, T)
    out, lse, rest = F.masked_attention(q, k, v, mask, 0.125)
    want = F.masked_attention_backward(q, k, v, out, rest, go, lse, mask, 0.125)
    d = L.AttentionDesc(batch=1, q_len=T, k_len=T, heads=H, kv_heads=H, head_dim=D, scale=0.125, softcap=0.0, causal=1,
                        dtype=L.BF16 if dtype == torch.bfloat16 else L.F16)
    head = lambda t: C.byref(L.HeadTensor(t.data_ptr(), T * H * D, H * D, D))  # noqa: E731
    need = L.lib.flb200_masked_attention_backward_workspace_bytes(C.byref(d))
    for off in (0, 4, 8, 12):
        ws = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
        grads = [torch.empty_like(t) for t in (q, k, v)]
        assert L.lib.flb200_masked_attention_backward(
            C.byref(d), head(q), head(k), head(v), head(out), rest.data_ptr(), head(go), lse.data_ptr(), None, None,
            *(head(t) for t in grads), ws.data_ptr() + 256 + off, need, torch.cuda.current_stream().cuda_stream) == L.OK
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
        assert bool((ws[:256 + off] == 77).all()) and bool((ws[256 + off + need:] == 77).all())
