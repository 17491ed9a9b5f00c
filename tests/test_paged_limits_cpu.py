"""CPU: sizes of paged attention that the kernels' 32-bit counts cannot go over are refused before a GPU is asked for."""
import ctypes

from test_paged_cpu import at, attention_of, cache_of, made_up


@made_up
def test_requests_of_attention(pkg):
    lib = pkg.load_library()
    where = [at(1024 * i) for i in range(11)]      # (16 GiB apart: tables of 2^31 rows)

    def call(requests):
        desc = attention_of(pkg, requests=requests, columns=1, table_stride=1)
        return lib.ixk_fmha_paged_fwd(ctypes.byref(desc), ctypes.byref(cache_of(pkg)), *where, 1 << 30, None)

    assert call(0x7fffffff) == pkg.IXK_UNIMPLEMENTED and call(0x7fffffff - 65535) == pkg.IXK_UNIMPLEMENTED
    assert call(0x7fffffff - 65536) == pkg.IXK_NO_DEVICE and call(3) == pkg.IXK_NO_DEVICE
    desc = attention_of(pkg, requests=0x7fffffff)
    assert lib.ixk_fmha_paged_fwd_workspace_bytes(ctypes.byref(desc), ctypes.byref(cache_of(pkg))) == 0
