"""The FP8 part of the C ABI: every symbol of include/sk_fp8.h is exported and bound, and bad arguments are refused before a device
is touched.  Also the plain forms that the GPU tests compare with, against torch's own e4m3 conversion."""
import ctypes
import os
import re

import pytest
import torch

import fp8_util as F
from conftest import ROOT

FAKE = 4096  # never dereferenced: validation fails first


def test_library_exports_every_declared_symbol(built_libs):
    from slimkernels_b200 import capi
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "sk_fp8.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(sk_[a-z0-9_]+)\s*\(", header))
    lib = capi.load()
    for name in sorted(declared):
        assert hasattr(lib, name), f"{name} declared in sk_fp8.h but not exported"
    assert declared == set(capi.FP8_SIGNATURES), "ctypes binding and header disagree"


def _rows(capi, q=FAKE, ld=128, scale=FAKE, row=1, block=8):
    return ctypes.byref(capi.Fp8Rows(q, ld, scale, row, block))


def _weight(capi, q=FAKE, ld=128, scale=FAKE, experts=1, N=128, K=128):
    return ctypes.byref(capi.Fp8Weight(q, ld, scale, experts, N, K))


def test_products_refuse_bad_arguments(built_libs):
    from slimkernels_b200 import capi
    lib = capi.load()
    r, w = lambda **k: _rows(capi, **k), lambda **k: _weight(capi, **k)

    def gemm(M=8, x=None, weight=None, st=0, out=FAKE, ld_out=128, ot=0):
        return lib.sk_fp8_gemm(M, x or r(), weight or w(), st, out, ld_out, ot, None)

    assert gemm(out=None) == capi.SK_ERR_NULL_POINTER
    assert gemm(weight=w(q=None)) == capi.SK_ERR_NULL_POINTER
    assert gemm(weight=w(scale=None)) == capi.SK_ERR_NULL_POINTER
    assert gemm(x=r(q=None)) == capi.SK_ERR_NULL_POINTER
    assert gemm(x=r(scale=None)) == capi.SK_ERR_NULL_POINTER
    assert gemm(st=2) == capi.SK_ERR_BAD_ARGUMENT
    assert gemm(ot=2) == capi.SK_ERR_BAD_ARGUMENT
    assert gemm(M=-1) == capi.SK_ERR_BAD_SHAPE
    assert gemm(ld_out=127) == capi.SK_ERR_BAD_SHAPE
    assert gemm(weight=w(N=0)) == capi.SK_ERR_BAD_SHAPE
    assert gemm(weight=w(K=0)) == capi.SK_ERR_BAD_SHAPE
    assert gemm(weight=w(K=130)) == capi.SK_ERR_BAD_SHAPE          # rows longer than their pitch
    assert gemm(weight=w(experts=2)) == capi.SK_ERR_BAD_SHAPE      # a product of one matrix
    assert gemm(weight=w(K=120, ld=120), x=r(ld=128)) == capi.SK_ERR_BAD_ALIGNMENT
    assert gemm(weight=w(q=FAKE + 8)) == capi.SK_ERR_BAD_ALIGNMENT
    assert gemm(x=r(ld=136)) == capi.SK_ERR_BAD_ALIGNMENT
    assert gemm(x=r(ld=112)) == capi.SK_ERR_BAD_SHAPE
    assert gemm(x=r(scale=FAKE + 2)) == capi.SK_ERR_BAD_ALIGNMENT
    assert gemm(out=FAKE + 1) == capi.SK_ERR_BAD_ALIGNMENT
    assert gemm(M=0) == capi.SK_OK                                   # nothing to do

    def grouped(M=8, x=None, weight=None, offsets=FAKE):
        return lib.sk_fp8_grouped_gemm(M, x or r(), weight or w(experts=4), 0, offsets, FAKE, 128, 0, None)

    assert grouped(offsets=None) == capi.SK_ERR_NULL_POINTER
    assert grouped(offsets=FAKE + 2) == capi.SK_ERR_BAD_ALIGNMENT
    assert grouped(weight=w(experts=1025)) == capi.SK_ERR_BAD_SHAPE
    assert grouped(M=0) == capi.SK_OK

    need = lib.sk_fp8_linear_workspace_bytes(8, 128, 0)
    assert need >= 8 * 128 + 8 * 4

    def linear(M=8, x=FAKE, xt=0, ld=128, weight=None, ws=FAKE, bytes_=need):
        return lib.sk_fp8_linear(M, x, xt, ld, weight or w(), 0, FAKE, 128, 0, ws, bytes_, None)

    assert linear(x=None) == capi.SK_ERR_NULL_POINTER
    assert linear(ws=None) == capi.SK_ERR_NULL_POINTER
    assert linear(xt=3) == capi.SK_ERR_BAD_ARGUMENT
    assert linear(bytes_=need - 1) == capi.SK_ERR_BAD_ARGUMENT
    assert linear(ld=127) == capi.SK_ERR_BAD_SHAPE
    assert linear(ws=FAKE + 16) == capi.SK_ERR_BAD_ALIGNMENT
    assert linear(M=0) == capi.SK_OK


def test_quantisers_refuse_bad_arguments(built_libs):
    from slimkernels_b200 import capi
    lib = capi.load()

    def quantize(x=FAKE, t=0, ld=128, M=4, K=128, out=None, st=0):
        return lib.sk_fp8_quantize(x, t, ld, M, K, out or _rows(capi), st, None)

    assert quantize(x=None) == capi.SK_ERR_NULL_POINTER
    assert quantize(t=5) == capi.SK_ERR_BAD_ARGUMENT
    assert quantize(st=2) == capi.SK_ERR_BAD_ARGUMENT
    assert quantize(K=0) == capi.SK_ERR_BAD_SHAPE
    assert quantize(ld=100) == capi.SK_ERR_BAD_SHAPE
    assert quantize(out=_rows(capi, ld=120), K=120) == capi.SK_ERR_BAD_ALIGNMENT
    assert quantize(x=FAKE + 1) == capi.SK_ERR_BAD_ALIGNMENT
    assert quantize(M=0) == capi.SK_OK

    def prepare(w=FAKE, t=0, ld=128, count=1, N=128, K=128, ld_q=128, matrix=128 * 128, st=0):
        return lib.sk_fp8_prepare_weight(w, t, ld, N * ld, count, N, K, FAKE, ld_q, matrix, FAKE, st, None)

    assert prepare(w=None) == capi.SK_ERR_NULL_POINTER
    assert prepare(t=3) == capi.SK_ERR_BAD_ARGUMENT
    assert prepare(count=0) == capi.SK_ERR_BAD_SHAPE
    assert prepare(count=65536) == capi.SK_ERR_BAD_SHAPE
    assert prepare(ld=64) == capi.SK_ERR_BAD_SHAPE
    assert prepare(K=120, ld_q=120) == capi.SK_ERR_BAD_ALIGNMENT


def test_router_and_experts_refuse_bad_arguments(built_libs):
    from slimkernels_b200 import capi
    lib = capi.load()

    def route(T=4, E=8, k=2, ld=8, t=0, logits=FAKE, ids=FAKE):
        return lib.sk_route_tokens(logits, t, ld, T, E, k, 1, ids, FAKE, FAKE, FAKE, FAKE, 1 << 20, None)

    assert route(logits=None) == capi.SK_ERR_NULL_POINTER
    assert route(ids=None) == capi.SK_ERR_NULL_POINTER
    assert route(t=3) == capi.SK_ERR_BAD_ARGUMENT
    assert route(k=9) == capi.SK_ERR_BAD_SHAPE
    assert route(k=0) == capi.SK_ERR_BAD_SHAPE
    assert route(E=1025, ld=1025) == capi.SK_ERR_BAD_SHAPE
    assert route(E=64, ld=64, k=33) == capi.SK_ERR_BAD_SHAPE
    assert route(T=-1) == capi.SK_ERR_BAD_SHAPE
    assert route(ld=7) == capi.SK_ERR_BAD_SHAPE
    assert lib.sk_group_by_expert(None, 4, 2, 8, FAKE, FAKE, FAKE, 1 << 20, None) == capi.SK_ERR_NULL_POINTER
    assert lib.sk_group_by_expert(FAKE, 4, 2, 0, FAKE, FAKE, FAKE, 1 << 20, None) == capi.SK_ERR_BAD_SHAPE

    assert lib.sk_group_by_expert(FAKE, 1 << 24, 1024, 8, FAKE, FAKE, FAKE, 1 << 40, None) == capi.SK_ERR_BAD_SHAPE      # places past 31 bits

    need = lib.sk_fp8_experts_workspace_bytes(4, 2, 128, 256, 0)

    def experts(T=4, k=2, x=FAKE, gate_up=None, down=None, ws=need, out=FAKE):
        return lib.sk_fp8_experts(T, k, x, 0, 128, FAKE, FAKE, FAKE, gate_up or _weight(capi, experts=16, N=256, K=128),
                                  down or _weight(capi, experts=8, N=128, K=256, ld=256), 0, out, 128, 0, FAKE, ws, None)

    assert experts(x=None) == capi.SK_ERR_NULL_POINTER
    assert experts(out=None) == capi.SK_ERR_NULL_POINTER
    assert experts(ws=need - 1) == capi.SK_ERR_BAD_ARGUMENT
    assert experts(k=0) == capi.SK_ERR_BAD_SHAPE
    assert experts(gate_up=_weight(capi, experts=8, N=256, K=128)) == capi.SK_ERR_BAD_SHAPE      # two matrices per expert are wanted
    assert experts(gate_up=_weight(capi, experts=16, N=128, K=128)) == capi.SK_ERR_BAD_SHAPE
    assert experts(T=0) == capi.SK_OK


def test_options_are_checked(built_libs):
    from slimkernels_b200 import capi
    lib = capi.load()
    for key, value in [(1, 48), (1, -1), (2, 3), (3, 10), (3, 999_999), (0, 0), (99, 0), (5, 4), (1, 64)]:
        assert lib.sk_fp8_set_option(key, value) == capi.SK_ERR_BAD_ARGUMENT, (key, value)
    for key in (1, 2, 3, 4, 5):
        assert lib.sk_fp8_set_option(key, 0) == capi.SK_OK


def test_module_casts_leave_codes_and_scales_alone():
    import slimkernels_b200.torch as sk
    codes = torch.arange(126, dtype=torch.uint8).repeat(64)[:4096].view(32, 128).view(torch.float8_e4m3fn)
    scale = torch.tensor([[254]], dtype=torch.uint8).view(torch.float8_e8m0fnu)             # (beyond fp16's range)
    m = sk.FP8Linear(codes, scale, 120, torch.ones(32), torch.float16)
    for cast in (m.half, m.double, lambda: m.to(torch.bfloat16), lambda: m.to("cpu", torch.float16)):
        assert cast() is m
        assert m.w_q.dtype == codes.dtype and torch.equal(m.w_q.view(torch.uint8), codes.view(torch.uint8))
        assert m.w_scale.dtype == scale.dtype and torch.equal(m.w_scale.view(torch.uint8), scale.view(torch.uint8))
    assert m.bias.dtype == torch.float16
    assert m.to("meta").w_q.is_meta and m.w_q.dtype == codes.dtype
    assert list(m.state_dict()) == ["w_q", "w_scale", "bias"]


def test_torch_ops_refuse_host_tensors(built_libs):
    import slimkernels_b200.torch as sk
    x = torch.zeros(4, 128)
    q = x.to(torch.float8_e4m3fn)
    s = torch.ones(4, 1)
    for call in (lambda: sk.quantize_fp8(x), lambda: sk.prepare_weight_fp8(x), lambda: sk.fp8_gemm(q, s, q, s[:1]),
                 lambda: sk.fp8_linear(x, q, s[:1]), lambda: sk.route_tokens(x, 2), lambda: sk.group_by_expert(torch.zeros(4, 2, dtype=torch.int32), 8)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("scale", [1.0, 1e-3, 300.0])
def test_plain_rounding_is_torchs(scale):
    t = (torch.randn(4096, generator=torch.Generator().manual_seed(1)) * scale).clamp(-448, 448)
    assert torch.equal(F.round_e4m3(t.double()).float(), t.to(torch.float8_e4m3fn).float())


def test_plain_exponents():
    a = torch.tensor([0.0, 448.0, 448.0001, 224.0, 1.75, 1.7500001, 2.0 ** -130], dtype=torch.float64)
    assert F.block_exponent(a).tolist() == [0, 0, 1, -1, -8, -7, -126]
