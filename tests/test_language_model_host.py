"""Host side of the language model operators: refusals of the C entry points before any launch, and the packed batches."""
import ctypes as C

import pytest
import torch

from flashlight_b200 import _lib as L


def adamw(tensor=None, count=1, **more):
    d = L.AdamwDesc(lr=1e-3, beta1=0.9, beta2=0.99, epsilon=1e-8, weight_decay=0.0, grad_scale=1.0, step=1,
                    param_dtype=L.F32, grad_dtype=L.F32, state_bits=32)
    for k, v in more.items():
        setattr(d, k, v)
    t = tensor if tensor is not None else L.AdamwTensor(16, 32, 48, 64, 80, 96, 4)
    return L.lib.flb200_adamw_step(C.byref(d), C.byref(t), count, None)


@pytest.mark.parametrize("more,status", [
    (dict(step=0), L.INVALID_ARG), (dict(beta1=1.0), L.INVALID_ARG), (dict(beta2=-0.1), L.INVALID_ARG),
    (dict(epsilon=-1.0), L.INVALID_ARG), (dict(state_bits=16), L.INVALID_ARG), (dict(param_dtype=9), L.INVALID_ARG),
    (dict(grad_dtype=9), L.INVALID_ARG), (dict(param_dtype=L.F16), L.UNSUPPORTED),
    (dict(param_dtype=L.BF16, grad_dtype=L.F16), L.UNSUPPORTED), (dict(count=-1), L.INVALID_ARG),
    (dict(tensor=L.AdamwTensor(0, 32, 48, 64, 80, 96, 4)), L.INVALID_ARG),      # no parameter
    (dict(tensor=L.AdamwTensor(16, 32, 48, 64, 0, 96, 4), state_bits=8), L.INVALID_ARG),  # no scale
    (dict(tensor=L.AdamwTensor(18, 32, 48, 64, 80, 96, 4)), L.INVALID_ARG),     # not on an element's boundary
    (dict(tensor=L.AdamwTensor(16, 32, 48, 64, 80, 96, -4)), L.INVALID_ARG),
    (dict(tensor=L.AdamwTensor(0, 0, 0, 0, 0, 0, 0)), L.OK),                    # nothing to do
    (dict(count=0), L.OK)])
def test_adamw_refuses_before_it_launches(more, status):
    assert adamw(**more) == status
    assert L.lib.flb200_adamw_step(None, None, 0, None) == L.INVALID_ARG


def test_linear_cce_refuses_before_it_launches():
    ok = dict(rows=4, features=8, classes=16, reduction=L.REDUCE_MEAN, ignore_index=-1, dtype=L.BF16)
    for more in (dict(reduction=7), dict(rows=0), dict(features=0), dict(classes=-1)):
        d = L.LinearCceDesc(**{**ok, **more})
        assert L.lib.flb200_linear_cce_forward(C.byref(d), 16, 16, None, 16, 16, 16, None, None, None, 0, None) == \
            L.INVALID_ARG
        assert L.lib.flb200_linear_cce_backward(C.byref(d), 16, 16, None, 16, 16, 16, 16, 16, 16, L.BF16, None, None, 0,
                                                None) == L.INVALID_ARG
        if "reduction" not in more:
            assert L.lib.flb200_linear_cce_workspace_bytes(C.byref(d), 16, 16, 1) == 0
    d = L.LinearCceDesc(**{**ok, "dtype": L.F32})
    assert L.lib.flb200_linear_cce_supported(C.byref(d)) == 0
    assert L.lib.flb200_linear_cce_forward(C.byref(d), 16, 16, None, 16, 16, 16, None, None, None, 0, None) == \
        L.UNSUPPORTED


def test_attention_refuses_before_it_launches():
    assert L.lib.flb200_attention_mask_bytes(0, 4, 4) == 0
    assert L.lib.flb200_attention_mask_bytes(2, 300, 400) == 2 * 3 * 16 + 2 * 4 * 8 + 2 * 300 * 8
    for extents in ((0, 4, 4), (1, 0, 4), (1, 5, 4), (1, 4, 1 << 24)):
        assert L.lib.flb200_attention_mask(*extents, 1, 16, None, 16, None) == L.INVALID_ARG
    assert L.lib.flb200_attention_mask(1, 4, 4, 1, 16, None, None, None) == L.INVALID_ARG
    assert L.lib.flb200_attention_mask(1, 4, 4, 1, None, None, 16, None) == L.INVALID_ARG  # a table is for documents
    assert L.lib.flb200_attention_mask(1, 4, 4, 0, 16, 16, 16, None) == L.INVALID_ARG  # a prefix without causal
    ok = dict(batch=1, q_len=4, k_len=4, heads=4, kv_heads=2, head_dim=64, scale=1.0, softcap=0.0, dtype=L.BF16)
    t = L.HeadTensor(16, 1024, 256, 64)
    for more in (dict(kv_heads=3), dict(q_len=5), dict(heads=0), dict(scale=0.0), dict(scale=float("nan")),
                 dict(softcap=-1.0), dict(softcap=1e-35), dict(prefix=16)):
        d = L.AttentionDesc(**{**ok, **more})
        args = [C.byref(d)] + [C.byref(t)] * 3
        assert L.lib.flb200_masked_attention_forward(*args, None, 16, C.byref(t), None, None, None, 0,
                                                     None) == L.INVALID_ARG
    for more in (dict(head_dim=65), dict(head_dim=136), dict(dtype=L.F32)):
        d = L.AttentionDesc(**{**ok, **more})
        assert L.lib.flb200_masked_attention_supported(C.byref(d)) == 0
        assert L.lib.flb200_masked_attention_forward(C.byref(d), C.byref(t), C.byref(t), C.byref(t), None, 16, C.byref(t),
                                                     None, None, None, 0, None) == L.UNSUPPORTED


def test_packed_batches():
    from flashlight_b200.packed_lm import packed_batch
    ids, targets, documents = packed_batch(3, 257, 50, 20, torch.Generator().manual_seed(4))
    targets = targets.view(3, 257)
    assert ids.shape == documents.shape == (3, 257) and int(ids.min()) >= 0 and int(ids.max()) < 50
    for row in range(3):
        for at in range(257):
            last = at == 256 or documents[row, at + 1] != documents[row, at]
            if documents[row, at] < 0 or last:  # padding and a document's last token predict nothing
                assert targets[row, at] == -1
            else:
                assert targets[row, at] == ids[row, at + 1]
    assert int(documents.max()) >= 5
