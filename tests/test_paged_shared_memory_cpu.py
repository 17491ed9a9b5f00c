"""CPU: what the calls on a paged cache write may share memory with no other operand, in whole or in part, and not with itself; slices
of one projection, of one buffer of keys and values, and results in the place of their inputs are as good as tensors of their own.
The C entries say so before they ask for a GPU: what they accept ends with IXK_NO_DEVICE here."""
import ctypes
import os
import random
import subprocess
import tempfile

import pytest

from test_paged_cpu import ROOT, at, attention_of, cache_of, made_up, pool_of, qk_of

# heads of 64 elements: 10 tokens of 4 + 2 + 2 heads in one projection
QKV = dict(q_strides=(512, 64), k_strides=(512, 64), v_strides=(512, 64))
H = 128        # bytes of a head


def forward(pkg, paged=False, desc=None, cache=None, **change):
    names = ("q", "k", "v", "q_gain", "k_gain", "cos", "sin", "positions", "q_out", "k_out", "cache", "slots", "k_pages", "v_pages")
    a = dict(zip(names, (at(i) for i in range(len(names)))))
    a.update(dict(k_out=None, cache=ctypes.byref(cache or cache_of(pkg))) if paged else dict(v=None, cache=None, slots=None, k_pages=None, v_pages=None))
    a.update(change)
    return pkg.load_library().ixk_qk_norm_rotary_fwd(ctypes.byref(qk_of(pkg, **(desc or {}))), *(a[n] for n in names), None)


@made_up
def test_norm_and_rotation(pkg):
    bad, fine = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_NO_DEVICE
    one = dict(q=at(0), k=at(0) + 4 * H)                                    # slices of one projection
    assert forward(pkg) == fine and forward(pkg, desc=QKV, **one) == fine
    # in place, and into another projection's places
    in_place = dict(QKV, q_out_strides=(512, 64), k_out_strides=(512, 64))
    assert forward(pkg, desc=in_place, **one, q_out=one["q"], k_out=one["k"]) == fine
    assert forward(pkg, desc=in_place, **one, q_out=at(20), k_out=at(20) + 4 * H) == fine
    assert forward(pkg, desc=in_place, **one, q_out=at(20), k_out=at(20) + 3 * H) == bad
    # where the values are: free for a forward pass without a cache
    assert forward(pkg, desc=in_place, **one, q_out=one["q"], k_out=at(0) + 6 * H) == fine
    assert forward(pkg, desc=in_place, **one, q_out=one["q"], k_out=at(0) + 7 * H) == bad        # its second head is the next token's first
    # one head, one token, or less, beside the input
    for shift in (H, 16, -16, -H, 512 * 2, -512 * 2 + 16):
        assert forward(pkg, desc=in_place, **one, q_out=one["q"] + shift, k_out=at(20)) == bad, shift
    assert forward(pkg, desc=in_place, **one, q_out=one["q"] + 10 * 1024, k_out=at(20)) == fine
    assert forward(pkg, desc=in_place, **one, q_out=one["q"] + 9 * 1024 + 6 * H - 16, k_out=at(20)) == bad       # (the last token's keys)
    assert forward(pkg, desc=in_place, **one, q_out=one["q"] + 9 * 1024 + 6 * H, k_out=at(20)) == fine
    assert forward(pkg, desc=dict(QKV, q_out_strides=(256, 64)), **one, q_out=one["q"]) == bad   # in place, laid out in another way
    # dense results over parts of other operands
    for name, size in (("cos", 100 * 64), ("sin", 100 * 64), ("positions", 40), ("q_gain", 256), ("k_gain", 256)):
        where = at(20)
        assert forward(pkg, **{name: where + 16, "q_out": where}) == bad, name
        assert forward(pkg, **{name: where, "k_out": where + (size - 1) // 16 * 16}) == bad, name
        assert forward(pkg, **{name: where, "k_out": where + (size + 15) // 16 * 16}) == fine, name
    # results that fold into themselves
    assert forward(pkg, desc=dict(q_out_strides=(64, 64))) == bad and forward(pkg, desc=dict(k_out_strides=(64, 128))) == bad
    assert forward(pkg, desc=dict(q_out_strides=(64, 640))) == fine and forward(pkg, desc=dict(q_out_strides=(64, 632))) == bad


@made_up
def test_into_the_pages(pkg):
    bad, fine = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_NO_DEVICE
    assert forward(pkg, True) == fine
    # keys and values of a page, of a token and of a head side by side
    for strides, apart in (((0, 4096, 128, 64), 4096), ((0, 4096, 256, 64), 256), ((0, 4096, 256, 128), 128)):
        cache = cache_of(pkg, k_strides=strides, v_strides=strides)
        assert forward(pkg, True, cache=cache, k_pages=at(12), v_pages=at(12) + apart) == fine, strides
        assert forward(pkg, True, cache=cache, k_pages=at(12) + apart, v_pages=at(12)) == fine, strides
        assert forward(pkg, True, cache=cache, k_pages=at(12), v_pages=at(12) + apart - 16) == bad, strides
        assert forward(pkg, True, cache=cache, k_pages=at(12), v_pages=at(12) + apart + 16) == bad, strides
    assert forward(pkg, True, k_pages=at(12), v_pages=at(12)) == bad and forward(pkg, True, v_pages=at(12) + 39 * 4096) == bad
    assert forward(pkg, True, v_pages=at(12) + 40 * 4096) == fine
    for name in ("q", "k", "v", "q_out", "cos", "positions", "slots", "k_gain"):
        assert forward(pkg, True, **{name: at(13) + 40 * 4096 - 16}) == bad, name
        assert forward(pkg, True, **{name: at(13) + 40 * 4096}) == fine, name
    assert forward(pkg, True, cache=cache_of(pkg, k_strides=(0, 2048, 64, 64))) == bad
    # in the place of the queries of one projection, the values beside them
    assert forward(pkg, True, desc=dict(QKV, q_out_strides=(512, 64)), q=at(0), k=at(0) + 4 * H, v=at(0) + 6 * H, q_out=at(0)) == fine
    assert forward(pkg, True, desc=dict(QKV, q_out_strides=(512, 64)), q=at(0), k=at(0) + 4 * H, v=at(0) + 6 * H, q_out=at(0) + H) == bad
    assert forward(pkg, True, desc=dict(QKV, q_out_strides=(512, 64)), q=at(20), k=at(0), v=at(0) + 6 * H, q_out=at(0) + 2 * H) == fine
    assert forward(pkg, True, desc=dict(QKV, q_out_strides=(512, 64)), q=at(20), k=at(0), v=at(0) + 5 * H, q_out=at(0) + 2 * H) == bad


@made_up
def test_the_gradients(pkg):
    lib = pkg.load_library()
    names = ("grad_q", "grad_k", "q", "k", "q_gain", "k_gain", "cos", "sin", "positions", "dq", "dk", "dq_gain", "dk_gain", "workspace", "bytes")
    need = lib.ixk_qk_norm_rotary_bwd_workspace_bytes(ctypes.byref(qk_of(pkg)))

    def call(desc=None, **change):
        a = dict(zip(names, (at(i) for i in range(len(names)))), bytes=need)
        a.update(change)
        return lib.ixk_qk_norm_rotary_bwd(ctypes.byref(qk_of(pkg, **(desc or {}))), *(a[n] for n in names), None)

    bad, fine = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_NO_DEVICE
    assert call() == fine and call(dq=at(2), dk=at(3)) == fine and call(dq=at(0), dk=at(1)) == fine
    for name, other in (("dq", "q"), ("dq", "grad_q"), ("dk", "k"), ("dk", "grad_k")):
        assert call(**{name: at(names.index(other)) + H}) == bad and call(**{name: at(names.index(other)) - 16}) == bad, (name, other)
    wide = dict(q_strides=(512, 64), k_strides=(512, 64), q_out_strides=(512, 64), k_out_strides=(512, 64))
    assert call(desc=wide, q=at(2), k=at(2) + 4 * H, dq=at(2), dk=at(2) + 4 * H) == fine
    assert call(desc=wide, q=at(2), k=at(2) + 4 * H, dq=at(9), dk=at(9) + 3 * H) == bad
    # the gains' gradients: with each other, the results, the scratch, other inputs; in the gains' places they are written last
    for where in (at(9) + 16, at(10), at(12) + 240, at(13) + need - 16, at(2), at(0) + 64, at(6), at(8) + 32, at(5)):
        assert call(dq_gain=where) == bad, hex(where)
    assert call(dq_gain=at(4), dk_gain=at(5)) == fine and call(dq_gain=at(4) + 16) == bad and call(dk_gain=at(4)) == bad
    for where in (at(9) - need + 16, at(10) + 64, at(2) + 16, at(3), at(4), at(7)):
        assert call(workspace=where) == bad, hex(where)
    assert call(workspace=at(9) - need) == fine
    # without gains the scratch is not used
    assert call(workspace=at(9), dq_gain=None, dk_gain=None) == fine


@made_up
def test_attention(pkg):
    lib = pkg.load_library()
    names = ("q", "k", "v", "table", "lengths", "row_start", "granted", "mask", "out", "lse", "workspace", "bytes")
    need = lib.ixk_fmha_paged_fwd_workspace_bytes(ctypes.byref(attention_of(pkg)), ctypes.byref(cache_of(pkg)))

    def call(desc=None, cache=None, **change):
        a = dict(zip(names, (at(8 * i) for i in range(len(names)))), bytes=need)
        a.update(change)
        return lib.ixk_fmha_paged_fwd(ctypes.byref(attention_of(pkg, **(desc or {}))), ctypes.byref(cache or cache_of(pkg)), *(a[n] for n in names), None)

    bad, fine = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_NO_DEVICE
    assert call() == fine and call(out=at(0)) == fine and call(v=at(8)) == fine           # (keys and values are only read)
    size = dict(q=12 * 512, k=40 * 4096, v=40 * 4096, table=96, lengths=12, row_start=16, granted=12, mask=48)
    for name, n in size.items():
        i = names.index(name)
        for out, bytes_of in (("out", 12 * 512), ("lse", 12 * 16), ("workspace", need)):
            assert call(**{out: at(8 * i) + (n - 1) // 16 * 16}) == bad, (out, name)
            assert call(**{out: at(8 * i) - bytes_of + 16}) == bad, (out, name)
            assert call(**{out: at(8 * i) + (n + 15) // 16 * 16}) == fine and call(**{out: at(8 * i) - bytes_of}) == fine, (out, name)
    assert call(lse=at(64) + 16) == bad and call(workspace=at(64) + 12 * 512 - 16) == bad and call(workspace=at(72)) == bad
    # slices of one projection
    assert call(desc=dict(q_strides=(512, 64), o_strides=(512, 64)), out=at(0)) == fine
    assert call(desc=dict(q_strides=(512, 64), o_strides=(512, 64)), out=at(0) + 4 * H) == fine
    assert call(desc=dict(q_strides=(512, 64), o_strides=(512, 64)), out=at(0) + 3 * H) == bad
    assert call(desc=dict(o_strides=(64, 64))) == bad and call(desc=dict(o_strides=(64, 768))) == fine
    # a scratch that is too small is not charged with what lies behind it (that it is too small is said where there is a GPU)
    assert call(workspace=at(64) - 64, bytes=64) == fine


@made_up
def test_keep(pkg):
    lib = pkg.load_library()
    names = ("lengths", "granted", "kept", "path", "path_columns", "path_stride", "page_table", "free_pages", "free_count", "free_count_out",
             "lengths_out", "cache", "k", "v")

    def call(cache=None, **change):
        a = dict(zip(names, (at(i) for i in range(len(names)))), path_columns=5, path_stride=5)
        a["cache"] = ctypes.byref(cache or cache_of(pkg))
        a.update(change)
        return lib.ixk_paged_keep(ctypes.byref(pool_of(pkg)), *(a[n] for n in names), None)

    bad, fine = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_NO_DEVICE
    assert call() == fine and call(lengths_out=at(0), free_count_out=at(8)) == fine
    assert call(v=at(12) + 16) == bad and call(v=at(12) + 40 * 4096 - 16) == bad and call(v=at(12) + 40 * 4096) == fine
    # keys and values of a layer behind one another, or layers side by side in a page
    by_layer = cache_of(pkg, layers=3, k_strides=(2 * 40 * 2048, 2048, 128, 64), v_strides=(2 * 40 * 2048, 2048, 128, 64))
    assert call(by_layer, v=at(12) + 40 * 4096) == fine and call(by_layer, v=at(12) + 39 * 4096) == bad
    in_page = cache_of(pkg, layers=3, k_strides=(4096, 3 * 4096, 128, 64), v_strides=(4096, 3 * 4096, 128, 64))
    assert call(in_page, v=at(12) + 4096) == fine and call(in_page, v=at(12) + 8192) == bad
    assert call(cache_of(pkg, layers=3, k_strides=(2048, 2048, 128, 64))) == bad
    for name, size in (("lengths", 12), ("granted", 12), ("kept", 12), ("path", 60), ("page_table", 96), ("free_pages", 160), ("free_count", 4), ("lengths_out", 12)):
        assert call(**{name: at(13) + 40 * 4096 - 4}) == bad and call(**{name: at(12) - size + 4}) == bad and call(**{name: at(12) - size}) == fine, name


def test_any_layouts(pkg):
    """The two questions, of random operands of a few bytes, against their bytes written down."""
    source = r'''
#include <cstdio>
#include "paged.h"
namespace ixk { int fail(int code, const std::string&) { return code; } }
int main() {
  using ixk::paged::Operand;
  long long p[2], run[2], e[6], s[6];
  while (scanf("%lld %lld %lld %lld", &p[0], &run[0], &p[1], &run[1]) == 4) {
    for (int i = 0; i < 6; ++i) if (scanf("%lld %lld", &e[i], &s[i]) != 2) return 1;
    const int64_t a[3] = {s[0], s[1], s[2]}, b[3] = {s[3], s[4], s[5]};
    const Operand x(reinterpret_cast<void*>(p[0]), run[0], {e[0], e[1], e[2]}, a, 1), y(reinterpret_cast<void*>(p[1]), run[1], {e[3], e[4], e[5]}, b, 1);
    printf("%d%d%d ", ixk::paged::meet(x, y), ixk::paged::folds(x), ixk::paged::folds(y));
  }
}
'''
    rng = random.Random(5)
    cases, want = [], []
    for _ in range(3000):
        p, run = [rng.randint(1, 200) for _ in range(2)], [rng.randint(1, 5) for _ in range(2)]
        e, s = [rng.randint(0 if rng.random() < 0.05 else 1, 4) for _ in range(6)], [rng.choice((0, 1, 3, 5, 8, 15, 16, 40, 64)) for _ in range(6)]
        cases.append(f"{p[0]} {run[0]} {p[1]} {run[1]} " + " ".join(f"{a} {b}" for a, b in zip(e, s)))
        places = [[p[t] + x * s[3 * t] + y * s[3 * t + 1] + z * s[3 * t + 2] + i for x in range(e[3 * t]) for y in range(e[3 * t + 1])
                   for z in range(e[3 * t + 2]) for i in range(run[t])] for t in range(2)]
        want.append(f"{int(bool(set(places[0]) & set(places[1])))}{int(len(set(places[0])) < len(places[0]))}{int(len(set(places[1])) < len(places[1]))}")
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "probe.cc"), os.path.join(d, "probe")
        with open(src, "w") as f:
            f.write(source)
        cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
        if not os.path.exists(os.path.join(cuda, "include", "cuda.h")):
            pytest.skip("no CUDA headers")
        csrc = os.path.join(os.path.dirname(pkg.__file__), "csrc")
        subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), "-I", csrc, "-I", os.path.join(cuda, "include"), src, "-o", exe], check=True)
        got = subprocess.run([exe], input="\n".join(cases), check=True, capture_output=True, text=True).stdout.split()
    assert got == want and len({w[0] for w in want}) == 2
