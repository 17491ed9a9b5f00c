"""CPU: the calls on a paged cache: their descriptors' layout, the workspace queries, and what the C entries refuse before they ask for a
GPU.  Addresses are made up: nothing reads them, and where there is a GPU that could, the tests are skipped."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

made_up = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where no kernel can run")


def at(i):
    """Addresses 16 MiB apart."""
    return 0x10000000 + i * (1 << 24)


def test_descriptors_are_laid_out_as_in_the_header(pkg):
    pairs = {"ixk_page_pool": pkg._PagePool, "ixk_paged_cache": pkg._PagedCache, "ixk_qk_desc": pkg._QkDesc, "ixk_fmha_paged_desc": pkg._FmhaPagedDesc}
    lines = [f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in s._fields_) for c, s in pairs.items()]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        with open(src, "w") as f:
            f.write("#include <stdio.h>\n#include <stddef.h>\n#include \"ixk.h\"\nint main(void) {" + "\n".join(lines) + "return 0; }\n")
        subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = [v for s in pairs.values() for v in [ctypes.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]]
    assert got == want


def pool_of(pkg, **change):
    d = dict(page_size=16, pages=40, requests=3, columns=8, table_stride=8)
    d.update(change)
    return pkg._PagePool(**d)


def cache_of(pkg, **change):
    d = dict(dtype=pkg.IXK_BF16, page_size=16, pages=40, heads=2, head_size=64, layers=1)
    strides = dict(k_strides=(0, 2048, 128, 64), v_strides=(0, 2048, 128, 64))
    for k, v in change.items():
        (strides if k in strides else d)[k] = v
    c = pkg._PagedCache(**d)
    for k, v in strides.items():
        getattr(c, k)[:] = v
    return c


@made_up
def test_extend_refuses(pkg):
    lib = pkg.load_library()
    names = ("lengths", "new_tokens", "page_table", "free_pages", "free_count", "free_count_out", "granted", "row_start", "rows", "request",
             "position", "slot")

    def call(pool=None, **change):
        a = dict(zip(names, (at(i) for i in range(len(names)))), rows=20)
        a.update(change)
        return lib.ixk_paged_extend(ctypes.byref(pool_of(pkg) if pool is None else pool), *(a[n] for n in names), None)

    bad, un = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_UNIMPLEMENTED
    for name in names:
        if name != "rows":
            assert call(**{name: None}) == bad, name
    assert call(rows=-1) == bad and call(rows=0x7fffffff) == un
    for change, status in ((dict(page_size=0), bad), (dict(pages=0), bad), (dict(requests=-1), bad), (dict(columns=0), bad), (dict(table_stride=7), bad),
                           (dict(page_size=1 << 27), un), (dict(pages=1 << 28), un), (dict(requests=16385), un)):
        assert call(pool_of(pkg, **change)) == status, change
    # an output in an input's or another output's place, whole or in part
    assert call(granted=at(0) + 8) == bad and call(row_start=at(1) - 12) == bad and call(request=at(2) + 4 * 23) == bad
    assert call(position=at(3) + 4 * 39) == bad and call(slot=at(9) + 4 * 19) == bad and call(free_count_out=at(0)) == bad
    assert call(page_table=at(3) - 4 * 23) == bad
    # the same table as a slice of a wider one may have other things between its rows' ends and starts, but not in its span
    assert call(pool_of(pkg, table_stride=100), granted=at(2) + 4 * 207) == bad


@made_up
def test_keep_refuses(pkg):
    lib = pkg.load_library()
    names = ("lengths", "granted", "kept", "path", "path_columns", "path_stride", "page_table", "free_pages", "free_count", "free_count_out",
             "lengths_out", "cache", "k", "v")

    def call(pool=None, cache=None, **change):
        a = dict(zip(names, (at(i) for i in range(len(names)))), path_columns=5, path_stride=5)
        a["cache"] = ctypes.byref(cache_of(pkg) if cache is None else cache)
        a.update(change)
        return lib.ixk_paged_keep(ctypes.byref(pool_of(pkg) if pool is None else pool), *(a[n] for n in names), None)

    bad, un = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_UNIMPLEMENTED
    for name in names:
        if name not in ("path_columns", "path_stride", "cache"):
            assert call(**{name: None}) == bad, name
    assert call(path_columns=0) == bad and call(path_stride=4) == bad and call(path_columns=1025, path_stride=1025) == un
    for change, status in ((dict(page_size=8), bad), (dict(pages=39), bad), (dict(dtype=pkg.IXK_F32), un), (dict(head_size=60), un), (dict(head_size=264), un),
                           (dict(heads=0), bad), (dict(layers=0), bad), (dict(k_strides=(0, 2048, 128, 32)), bad), (dict(v_strides=(0, 2048, 132, 64)), un),
                           (dict(layers=2), bad)):
        assert call(cache=cache_of(pkg, **change)) == status, change
    assert call(k=at(12) + 8) == bad and call(k=at(13)) == bad
    assert call(lengths_out=at(0) + 4) == bad and call(lengths_out=at(1)) == bad and call(lengths_out=at(3) + 4 * 14) == bad
    assert call(lengths_out=at(6) - 8) == bad and call(free_count_out=at(2)) == bad and call(free_pages=at(6) + 4 * 20) == bad


def qk_of(pkg, **change):
    d = dict(dtype=pkg.IXK_BF16, param_dtype=pkg.IXK_F32, heads=4, kv_heads=2, head_size=64, rotary_dim=32, interleaved=0, position_bytes=4, eps=1e-6,
             gain_offset=0.0, tokens=10, places=100)
    strides = dict(q_strides=(256, 64), k_strides=(128, 64), v_strides=(128, 64), q_out_strides=(256, 64), k_out_strides=(128, 64), gq_strides=(256, 64),
                   gk_strides=(128, 64))
    for k, v in change.items():
        (strides if k in strides else d)[k] = v
    c = pkg._QkDesc(**d)
    for k, v in strides.items():
        getattr(c, k)[:] = v
    return c


FAULTS = [dict(dtype=99), dict(param_dtype=1), dict(heads=0), dict(kv_heads=-1), dict(head_size=60), dict(head_size=264), dict(rotary_dim=0),
          dict(rotary_dim=72), dict(rotary_dim=24), dict(interleaved=1, rotary_dim=12), dict(position_bytes=2), dict(eps=-1.0), dict(eps=float("nan")),
          dict(gain_offset=float("nan")), dict(tokens=-1), dict(places=0), dict(tokens=1 << 31), dict(heads=1 << 17), dict(q_strides=(260, 64)),
          dict(k_strides=(-128, 64)), dict(q_out_strides=(256, 32)), dict(k_out_strides=(56, 64))]


@made_up
@pytest.mark.parametrize("paged", [False, True])
def test_qk_forward_refuses(pkg, paged):
    lib = pkg.load_library()
    names = ("q", "k", "v", "q_gain", "k_gain", "cos", "sin", "positions", "q_out", "k_out", "cache", "slots", "k_pages", "v_pages")

    def call(desc=None, cache=None, **change):
        a = dict(zip(names, (at(i) for i in range(len(names)))))
        if paged:
            a.update(k_out=None, cache=ctypes.byref(cache_of(pkg) if cache is None else cache))
        else:
            a.update(v=None, cache=None, slots=None, k_pages=None, v_pages=None)
        a.update(change)
        return lib.ixk_qk_norm_rotary_fwd(ctypes.byref(qk_of(pkg) if desc is None else desc), *(a[n] for n in names), None)

    refused = (pkg.IXK_INVALID_ARGUMENT, pkg.IXK_UNIMPLEMENTED)
    for name in ("q", "k", "cos", "sin", "q_out") + (("v", "slots", "k_pages", "v_pages") if paged else ("k_out",)):
        assert call(**{name: None}) in refused, name
    for change in FAULTS:
        if not (paged and "k_out_strides" in change):
            assert call(qk_of(pkg, **change)) in refused, change
    for name in ("q", "k", "q_gain", "k_gain", "cos", "sin", "q_out"):
        assert call(**{name: at(40) + 8}) in refused, name
    assert call(q_out=at(1)) in refused and call(q_out=at(5)) in refused
    assert call(qk_of(pkg, q_out_strides=(512, 64)), q_out=at(0)) in refused       # in place, but laid out in another way
    if paged:
        for change in (dict(heads=1), dict(head_size=128), dict(dtype=pkg.IXK_F16), dict(page_size=0)):
            assert call(cache=cache_of(pkg, **change)) in refused, change
        assert call(v_pages=at(12)) in refused and call(q_out=at(12)) in refused
    else:
        assert call(k_out=at(0)) in refused and call(q_out=at(9)) in refused


@made_up
def test_qk_backward_refuses(pkg):
    lib = pkg.load_library()
    names = ("grad_q", "grad_k", "q", "k", "q_gain", "k_gain", "cos", "sin", "positions", "dq", "dk", "dq_gain", "dk_gain", "workspace", "bytes")

    def call(desc=None, **change):
        a = dict(zip(names, (at(i) for i in range(len(names)))), bytes=1 << 24)
        a.update(change)
        return lib.ixk_qk_norm_rotary_bwd(ctypes.byref(qk_of(pkg) if desc is None else desc), *(a[n] for n in names), None)

    refused = (pkg.IXK_INVALID_ARGUMENT, pkg.IXK_UNIMPLEMENTED)
    for name in ("grad_q", "grad_k", "q", "k", "cos", "sin", "dq", "dk"):
        assert call(**{name: None}) in refused, name
    for change in FAULTS + [dict(gq_strides=(8, -8)), dict(gk_strides=(130, 64))]:
        assert call(qk_of(pkg, **change)) in refused, change
    need = lib.ixk_qk_norm_rotary_bwd_workspace_bytes(ctypes.byref(qk_of(pkg)))
    assert need > 0 and call(bytes=need - 1) == pkg.IXK_WORKSPACE_TOO_SMALL and call(workspace=None) == pkg.IXK_WORKSPACE_TOO_SMALL
    assert call(dq=at(1)) in refused and call(dk=at(2)) in refused and call(dk=at(9)) in refused and call(dq=at(13)) in refused
    assert call(qk_of(pkg, gq_strides=(0, 64)), dq=at(0)) in refused
    assert lib.ixk_qk_norm_rotary_bwd_workspace_bytes(ctypes.byref(qk_of(pkg, heads=0))) == 0


def attention_of(pkg, **change):
    d = dict(heads=4, requests=3, columns=8, mask_words=1, head_scale=0.1, reserved=0, rows=12, table_stride=8, mask_stride=1)
    strides = dict(q_strides=(256, 64), o_strides=(256, 64))
    for k, v in change.items():
        (strides if k in strides else d)[k] = v
    c = pkg._FmhaPagedDesc(**d)
    for k, v in strides.items():
        getattr(c, k)[:] = v
    return c


@made_up
def test_attention_refuses(pkg):
    lib = pkg.load_library()
    names = ("q", "k", "v", "table", "lengths", "row_start", "granted", "mask", "out", "lse", "workspace", "bytes")

    def call(desc=None, cache=None, **change):
        a = dict(zip(names, (at(i) for i in range(len(names)))), bytes=1 << 30)
        a.update(change)
        return lib.ixk_fmha_paged_fwd(ctypes.byref(attention_of(pkg) if desc is None else desc), ctypes.byref(cache_of(pkg) if cache is None else cache),
                                      *(a[n] for n in names), None)

    refused = (pkg.IXK_INVALID_ARGUMENT, pkg.IXK_UNIMPLEMENTED)
    for name in ("q", "k", "v", "table", "lengths", "row_start", "granted", "out"):
        assert call(**{name: None}) in refused, name
    for change in (dict(heads=0), dict(heads=3), dict(heads=258), dict(requests=-1), dict(columns=0), dict(mask_words=0), dict(mask_words=2), dict(head_scale=float("inf")),
                   dict(head_scale=float("nan")), dict(reserved=1), dict(rows=-1), dict(rows=1 << 31), dict(table_stride=7), dict(columns=1 << 27, table_stride=1 << 27),
                   dict(q_strides=(256, 60)), dict(q_strides=(32, 64)), dict(o_strides=(0, 64)), dict(o_strides=(256, -64))):
        assert call(attention_of(pkg, **change)) in refused, change
    for change in (dict(page_size=12), dict(page_size=4), dict(page_size=512), dict(head_size=60), dict(head_size=0), dict(head_size=264), dict(heads=0), dict(heads=3),
                   dict(dtype=pkg.IXK_F32), dict(pages=0), dict(pages=1 << 28), dict(k_strides=(0, 2048, 100, 64)), dict(v_strides=(0, 32, 128, 64))):
        assert call(cache=cache_of(pkg, **change)) in refused, change
    for name in ("q", "k", "v", "out", "workspace"):
        assert call(**{name: at(40) + 8}) in refused, name
    assert call(out=at(1)) in refused and call(out=at(2)) in refused
    assert call(attention_of(pkg, o_strides=(512, 64)), out=at(0)) in refused
    need = lib.ixk_fmha_paged_fwd_workspace_bytes
    small = need(ctypes.byref(attention_of(pkg)), ctypes.byref(cache_of(pkg)))
    large = need(ctypes.byref(attention_of(pkg, rows=1000)), ctypes.byref(cache_of(pkg, head_size=256)))
    assert 0 < small < large < 1 << 27
    assert need(ctypes.byref(attention_of(pkg, heads=3)), ctypes.byref(cache_of(pkg))) == 0


def test_tensors_off_the_gpu(pkg):
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    x, pages, table = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 16, 4, 64, dtype=torch.bfloat16), ints(2, 3)
    cos = torch.zeros(5, 16)
    for call in (lambda: pkg.paged_extend(table, ints(2), ints(2), ints(3), ints(1), rows=2, page_size=16),
                 lambda: pkg.paged_keep(table, ints(2), ints(2), ints(2), ints(3), ints(1), page_size=16),
                 lambda: pkg.qk_norm_rotary_forward(x, x, cos=cos, sin=cos),
                 lambda: pkg.qk_norm_rotary_backward(x, x, x, x, cos=cos, sin=cos),
                 lambda: pkg.fmha_paged_forward(x, pages, pages, table, ints(2), ints(3), ints(2), scale=1.0)):
        with pytest.raises(pkg.IxkError) as e:
            call()
        assert e.value.status == pkg.IXK_NO_DEVICE
