"""What moves or casts a whole model leaves codes and scales as they are, whatever torch does with its other tensors."""
import copy

import pytest
import torch
from torch import nn

import slimkernels_b200.torch as sk


def _modules():
    g = torch.Generator().manual_seed(1)
    codes = lambda *shape: torch.randint(0, 126, shape, generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn)      # noqa: E731
    exps = lambda *shape: torch.randint(100, 255, shape, generator=g, dtype=torch.uint8).view(torch.float8_e8m0fnu)    # noqa: E731
    f32 = lambda *shape: torch.rand(*shape, generator=g) + 1e30                                                         # noqa: E731
    return [sk.FP8Linear(codes(32, 256), exps(1, 2), 250, torch.ones(32)), sk.FP8Linear(codes(32, 256), f32(1, 2), 250),
            sk.FP8Experts(codes(3, 2, 48, 64), exps(3, 2, 1, 1), codes(3, 64, 48), exps(3, 1, 1), 64, 48),
            sk.FP8Experts(codes(3, 2, 48, 64), f32(3, 2, 1, 1), codes(3, 64, 48), f32(3, 1, 1), 64, 48)]


@pytest.mark.parametrize("move", [lambda m: m.type(torch.float16), lambda m: m.type(torch.float64), lambda m: m.type(torch.int8),
                                  lambda m: m.type("torch.BFloat16Tensor"), lambda m: m.to(memory_format=torch.channels_last),
                                  lambda m: m.to(torch.float16, memory_format=torch.channels_last), lambda m: m.share_memory(), lambda m: m.bfloat16(),
                                  lambda m: m.cpu()],
                         ids=["type half", "type double", "type int8", "type by name", "channels last", "half, channels last", "share", "bfloat16", "cpu"])
@pytest.mark.parametrize("which", range(4))
def test_codes_and_scales_keep_type_shape_order_and_bits(which, move):
    m = _modules()[which]
    before = {n: getattr(m, n) for n in m._as_they_are}
    model = move(nn.Sequential(copy.deepcopy(m)))
    for n, t in before.items():
        u = getattr(model[0], n)
        assert u.dtype == t.dtype and u.shape == t.shape and u.stride() == t.stride()
        assert torch.equal(u.contiguous().view(torch.uint8), t.view(torch.uint8))


@pytest.mark.parametrize("which", range(4))
def test_empty_copies_keep_type_shape_and_order(which):
    m = _modules()[which]
    for e in (copy.deepcopy(m).to("meta"), copy.deepcopy(m).to_empty(device="meta")):
        for n in m._as_they_are:
            t, u = getattr(m, n), getattr(e, n)
            assert u.is_meta and u.dtype == t.dtype and u.shape == t.shape and u.stride() == t.stride()


def test_shared_memory_is_shared():
    m = _modules()[0]
    m.share_memory()
    assert m.w_q.untyped_storage().is_shared() and m.w_scale.untyped_storage().is_shared()


def test_a_weight_that_is_no_buffer_any_more_may_be_moved():
    m = _modules()[0]
    codes = m.w_q.clone()
    m.w_q = nn.Parameter(codes, requires_grad=False)
    assert m.to("cpu").w_q.dtype == codes.dtype and m.to("meta").w_q.is_meta
    m = _modules()[0]
    m.register_buffer("bias", None)
    del m.w_scale
    m.w_scale = torch.ones(1, 2)                            # (a plain attribute from now on)
    assert m.half().w_q.dtype == codes.dtype
