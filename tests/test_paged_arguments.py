"""More of what the paged operators refuse, or have to take, by their arguments alone (CPU).  Calls of
no tokens: what is not refused returns 0 without touching a device."""

import ctypes
from ctypes import c_void_p

import pytest

import cudaforge_amd as cf

DUMMY = ctypes.create_string_buffer(256)
DP = ctypes.addressof(DUMMY)
STORES = ["kv_page_store_f16_cuda", "kv_page_store_f32_cuda"]


def store(native, op, ins, outs, **kw):
    p = cf.KvPageStoreParams(**dict(dict(num_tokens=0, num_heads=8, num_kv_heads=2, head_dim=64, page_size=16, num_pages=8,
                                         rope_base=0.0), **kw))
    a, b = (c_void_p * len(ins))(*ins), (c_void_p * len(outs))(*outs)
    return native.operator_find(op.encode()).contents.func(a, b, ctypes.cast(ctypes.pointer(p), c_void_p), None)


@pytest.mark.parametrize("op", STORES)
@pytest.mark.parametrize("H_kv,d,rc", [
    (65535, 65535, -1), (32768, 32768, -1), (32768, 16384 + 1, -1), (32768, 16384, 0), (65535, 64, 0), (1, 65535, 0),
])
def test_store_refuses_rows_that_pass_its_counters(native, op, H_kv, d, rc):
    """A row of K is counted in 32 bits, K and V together: 2^29 elements at most."""
    assert store(native, op, [DP] * 3, [DP] * 2, num_kv_heads=H_kv, head_dim=d) == rc


@pytest.mark.parametrize("op", STORES)
@pytest.mark.parametrize("same,strides,rc", [
    (True, (0, 0), 0), (True, (512, 0), 0), (True, (0, 512), 0), (True, (768, 768), 0), (True, (768, 0), -1),
    (True, (0, 768), -1), (True, (768, 512), -1), (False, (768, 0), 0), (False, (0, 768), 0),
])
def test_store_in_place_takes_one_stride(native, op, same, strides, rc):
    """Q turned where it lies: its rows have to be those of the result (8 heads of 64: 512 is the
    stride that 0 stands for), as another row's place may be written before it is read."""
    q, q_out = DP + 64, DP + (64 if same else 128)
    assert store(native, op, [DP] * 4 + [q], [DP, DP, q_out], rope_base=10000.0, q_stride=strides[0],
                 q_out_stride=strides[1]) == rc
