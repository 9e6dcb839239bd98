"""Pointers that lie between elements are refused before a device is touched."""
import ctypes

import pytest

FAKE = 4096  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def capi(built_libs):
    from slimkernels_b200 import capi
    capi.load()
    return capi


def test_quantisers_refuse_float_scales_between_elements(capi):
    lib = capi.load()

    def quantize(scale, st, M=4):
        return lib.sk_fp8_quantize(FAKE, 0, 128, M, 128, ctypes.byref(capi.Fp8Rows(FAKE, 128, scale, 1, 4)), st, None)

    for off in (1, 2, 3):
        assert quantize(FAKE + off, capi.SK_SCALE_F32) == capi.SK_ERR_BAD_ALIGNMENT
        assert quantize(FAKE + off, capi.SK_SCALE_E8M0, M=0) == capi.SK_OK                # (bytes may lie anywhere)
        assert lib.sk_fp8_prepare_weight(FAKE, 0, 128, 128 * 128, 1, 128, 128, FAKE, 128, 128 * 128, FAKE + off, capi.SK_SCALE_F32,
                                         None) == capi.SK_ERR_BAD_ALIGNMENT


@pytest.mark.parametrize("name", ["logits", "ids", "weights", "rows", "offsets"])
@pytest.mark.parametrize("type_,size", [(0, 2), (1, 2), (2, 4)])
def test_router_refuses_pointers_between_elements(capi, name, type_, size):
    for off in (1, 2, 3):
        p = dict(logits=FAKE, ids=FAKE, weights=FAKE, rows=FAKE, offsets=FAKE)
        p[name] += off
        if off % (size if name == "logits" else 4) == 0:
            continue                                        # (nothing wrong with that one: it would be launched)
        rc = capi.load().sk_route_tokens(p["logits"], type_, 8, 4, 8, 2, 1, p["ids"], p["weights"], p["rows"], p["offsets"], FAKE, 1 << 20, None)
        assert rc == capi.SK_ERR_BAD_ALIGNMENT


@pytest.mark.parametrize("name", ["ids", "rows", "offsets"])
def test_order_by_expert_refuses_pointers_between_elements(capi, name):
    for off in (1, 2, 3):
        p = dict(ids=FAKE, rows=FAKE, offsets=FAKE)
        p[name] += off
        assert capi.load().sk_group_by_expert(p["ids"], 4, 2, 8, p["rows"], p["offsets"], FAKE, 1 << 20, None) == capi.SK_ERR_BAD_ALIGNMENT


@pytest.mark.parametrize("name", ["rows", "weights", "offsets"])
def test_expert_layers_refuse_pointers_between_elements(capi, name):
    lib = capi.load()
    gate_up, down = capi.Fp8Weight(FAKE, 128, FAKE, 16, 256, 128), capi.Fp8Weight(FAKE, 256, FAKE, 8, 128, 256)
    need = lib.sk_fp8_experts_workspace_bytes(4, 2, 128, 256, 0)
    for off in (1, 2, 3):
        p = dict(rows=FAKE, weights=FAKE, offsets=FAKE)
        p[name] += off
        rc = lib.sk_fp8_experts(4, 2, FAKE, 0, 128, p["rows"], p["weights"], p["offsets"], ctypes.byref(gate_up), ctypes.byref(down), 0, FAKE, 128, 0,
                                FAKE, need, None)
        assert rc == capi.SK_ERR_BAD_ALIGNMENT
