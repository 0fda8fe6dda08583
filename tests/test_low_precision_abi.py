"""The entry points on microscaled 4-bit floating point, of the norm with codes and of the choice of experts without a
GPU: calls without a context or a handle are refused, not followed, and header and binding agree."""
import ctypes
import re
from pathlib import Path

import pytest

from decisive_amd import rocm

ROOT = Path(__file__).resolve().parent.parent
INVALID_REQUEST = 1


def test_calls_without_a_context_are_refused():
    lib = rocm.load()
    out = ctypes.c_void_p()
    rule = rocm.MoeSelection(experts=1, top_k=1, sigmoid=0, groups=1, top_groups=1, group_best=1, renormalize=0, scale=1)
    assert lib.dz_mx4_weight_create(None, None, None, 1, 1, ctypes.byref(out)) == INVALID_REQUEST
    assert lib.dz_mx4_weight_quantize(None, None, 0, 1, 1, ctypes.byref(out)) == INVALID_REQUEST
    assert lib.dz_mx4_weight_free(None, None) == INVALID_REQUEST
    assert lib.dz_mx4_weight_info(None, None, None, None) == INVALID_REQUEST
    assert lib.dz_mx4_dequant(None, None, None) == INVALID_REQUEST
    assert lib.dz_mx4_quantize(None, None, 0, 1, 1, None, None) == INVALID_REQUEST
    assert lib.dz_mx4_linear(None, None, None, 0, 1, None, 0) == INVALID_REQUEST
    assert lib.dz_mx4_linear_q4(None, None, None, None, 1, None, 0) == INVALID_REQUEST
    for name in ("dz_add_rmsnorm_fp8", "dz_add_rmsnorm_mx4"):
        assert getattr(lib, name)(None, None, None, 0, 1, 1, None, 0.0, 0, None, None, None, None) == INVALID_REQUEST
    assert lib.dz_moe_logits(None, None, None, 0, 1, None) == INVALID_REQUEST
    assert lib.dz_moe_select(None, ctypes.byref(rule), None, 0, 1, None, None, None) == INVALID_REQUEST
    assert lib.dz_moe_forward_selected(None, None, None, 0, 1, None, None, None) == INVALID_REQUEST
    assert out.value is None


@pytest.mark.parametrize("m,k", [(0, 1), (1, 1), (16, 128), (17, 129), (64, 4096), (65, 4097), (1 << 24, 1 << 20)])
def test_bytes_of_codes_and_scales(m, k):
    g = -(-k // 128)
    assert rocm.mx4_bytes(m, k) == (-(-m // 16) * g * 1024, -(-m // 64) * g * 256)


@pytest.mark.parametrize("m,k", [(1, 0), (1, (1 << 20) + 1), ((1 << 24) + 1, 1)])
def test_bytes_of_shapes_that_no_call_takes(m, k):
    with pytest.raises(rocm.DzError) as e:
        rocm.mx4_bytes(m, k)
    assert e.value.code == "INVALID_PARAMETERS"


def test_bytes_may_be_asked_for_one_at_a_time():
    codes, scales = ctypes.c_size_t(), ctypes.c_size_t()
    assert rocm.load().dz_mx4_bytes(20, 300, ctypes.byref(codes), None) == 0
    assert rocm.load().dz_mx4_bytes(20, 300, None, ctypes.byref(scales)) == 0
    assert (codes.value, scales.value) == rocm.mx4_bytes(20, 300)


def test_the_rule_s_fields_are_the_header_s():
    header = (ROOT / "include" / "decisive_rocm.h").read_text()
    fields = re.search(r"typedef struct dz_moe_selection \{(.*?)\}", header, re.S).group(1)
    named = re.findall(r"(int32_t|float) (\w+);", fields)
    kinds = {"int32_t": ctypes.c_int32, "float": ctypes.c_float}
    assert [(name, kinds[kind]) for kind, name in named] == list(rocm.MoeSelection._fields_)


def test_the_header_lists_every_variant():
    header = (ROOT / "include" / "decisive_rocm.h").read_text()
    source = (ROOT / "decisive_amd" / "csrc" / "products.hip").read_text()
    names = re.findall(r'"([^"]+)"', re.search(r"kMx4Names\[\] = \{(.*?)\};", source, re.S).group(1))
    listed = re.search(r'\n \*   "mx4" (.*?)\*/', header, re.S).group(1)
    assert names and not set(names) - set(re.findall(r"[\w-]+", listed))


def test_barriers_between_stages_wait_for_loads_and_reads():
    """Stages filled by DMA: before a barrier after which one is loaded again, this wave's loads and its reads are waited
    for in the same statement, since the compiler's own waits see neither."""
    source = (ROOT / "decisive_amd" / "csrc" / "mx4.hip").read_text()
    found = [a for a in re.findall(r"asm volatile\(\s*((?:\"[^\"]*\"\s*)+)", source) if "s_barrier" in a]
    assert len(found) >= 2
    for text in found:
        wait = text.split("s_barrier")[0]
        assert re.search(r"vmcnt\((%0|0)\)", wait) and "lgkmcnt(0)" in wait, text
