"""nsa_kv8_adopt's argument checks, which come before any CUDA call."""
import ctypes
import importlib

KV8 = importlib.import_module("numerics-and-sparse-attn_b200.kv8")
LIB = importlib.import_module("numerics-and-sparse-attn_b200._lib")


def _desc(batch=2):
    d = KV8.Kv8CacheDesc(batch, 2, 128, 8, 4, 1, 0)
    for n in ("k_codes", "v_codes", "scales", "page_table", "k_ring", "v_ring", "lens", "ring_floor", "unclean", "tickets"):
        setattr(d, n, 4096)
    return ctypes.byref(d)


def test_arguments_are_checked():
    lib = LIB.load()
    assert lib.nsa_kv8_adopt(None, 4096, None) == 1
    assert lib.nsa_kv8_adopt(_desc(), None, None) == 1 and b"lens" in lib.nsa_last_error_message()
    assert lib.nsa_kv8_adopt(_desc(batch=-1), 4096, None) == 1
    assert lib.nsa_kv8_adopt(_desc(batch=0), None, None) == 0
