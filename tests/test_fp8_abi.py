"""The 8-bit floating point entry points without a GPU: calls without a context or a handle are refused, not
followed, and the header lists every variant of the product."""
import ctypes
import re
from pathlib import Path

from decisive_amd import rocm

ROOT = Path(__file__).resolve().parent.parent
INVALID_REQUEST = 1


def test_calls_without_a_context_are_refused():
    lib = rocm.load()
    out = ctypes.c_void_p()
    cfg = rocm.MoeConfig(experts=1, top_k=1, hidden=1, ff=1, renormalize=0)
    assert lib.dz_fp8_weight_create(None, None, None, 1, 1, ctypes.byref(out)) == INVALID_REQUEST
    assert lib.dz_fp8_weight_quantize(None, None, 0, 1, 1, ctypes.byref(out)) == INVALID_REQUEST
    assert lib.dz_fp8_weight_free(None, None) == INVALID_REQUEST
    assert lib.dz_fp8_dequant(None, None, None) == INVALID_REQUEST
    assert lib.dz_fp8_quantize(None, None, 0, 1, 1, None, None) == INVALID_REQUEST
    assert lib.dz_fp8_linear(None, None, None, 0, 1, None, 0) == INVALID_REQUEST
    assert lib.dz_fp8_linear_q8(None, None, None, None, 1, None, 0) == INVALID_REQUEST
    assert lib.dz_moe_create(None, ctypes.byref(cfg), None, 0, *[None] * 6, ctypes.byref(out)) == INVALID_REQUEST
    assert lib.dz_moe_free(None, None) == INVALID_REQUEST
    assert lib.dz_moe_route(None, None, None, 0, 1, None, None) == INVALID_REQUEST
    assert lib.dz_moe_forward(None, None, None, 0, 1, None) == INVALID_REQUEST
    assert out.value is None


def test_info_of_no_handle_is_refused():
    lib = rocm.load()
    assert lib.dz_fp8_weight_info(None, None, None, None) == INVALID_REQUEST
    assert lib.dz_moe_info(None, None, None) == INVALID_REQUEST


def test_header_and_binding_agree():
    header = (ROOT / "include" / "decisive_rocm.h").read_text()
    source = (ROOT / "decisive_amd" / "csrc" / "products.hip").read_text()
    names = re.findall(r'"([^"]+)"', re.search(r"kFp8Names\[\] = \{(.*?)\};", source, re.S).group(1))
    listed = re.search(r'\n \*   "fp8" (.*?)\*/', header, re.S).group(1)
    assert names and not set(names) - set(re.findall(r"[\w-]+", listed))
    assert int(re.search(r"#define DZ_MOE_MAX_TOKENS (\d+)", header).group(1)) == rocm.MOE_MAX_TOKENS
    fields = re.search(r"typedef struct dz_moe_config \{(.*?)\}", header, re.S).group(1)
    assert re.findall(r"int32_t (\w+);", fields) == [name for name, _ in rocm.MoeConfig._fields_]
