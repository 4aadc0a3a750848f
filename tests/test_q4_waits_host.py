"""The limit of waits inside the 4-bit cache's attention, as checked on the host."""
import ctypes as ct

from astc_kv_cuda import _lib as L
from test_q4_host import _attention


def test_a_limit_below_zero_is_refused():
    d = _attention()
    assert d.wait_tries == 0 and L.lib().akv_q4_attention_workspace(ct.byref(d)) > 0
    d.wait_tries = 1
    assert L.lib().akv_q4_attention_workspace(ct.byref(d)) > 0
    d.wait_tries = -1
    assert L.lib().akv_q4_attention_workspace(ct.byref(d)) == 0
    assert L.lib().akv_q4_attention(ct.byref(d), None) == 1
