"""CPU: what the host decides for the losses at the vocabulary head: the pieces of the vocabulary, scratch, the workspace query."""
import ctypes
import importlib
import math
import os
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "intel-extension-for-openxla_b200", "csrc")

PIECES = r'''
#include <stdio.h>
#include "head_pieces.h"
using namespace ixk::head;
int main() {
  long long rows, vocab;
  while (scanf("%lld %lld", &rows, &vocab) == 2) {
    const Pieces p = pieces_for(rows, vocab);
    long long n = 0, most = 0, end = 0, short_piece = 0;
    for (int64_t first = 0; first < vocab; first += p.columns, ++n) {
      const long long columns = p.columns_of(first);
      most = most > p.bias_parts * columns ? most : p.bias_parts * columns;
      if (columns <= 0) short_piece = 1;
      end = first + columns;
    }
    printf("%lld %lld %lld %lld %lld %lld %lld %lld\n", (long long)p.columns, (long long)p.count, (long long)p.bias_parts,
           (long long)p.bias_partials(), n, most, end, short_piece);
  }
}
'''


def test_every_piece_of_the_vocabulary_fits_its_scratch():
    """Pieces cover the vocabulary, start on multiples of 256 columns, and the bias's partial sums of every one of them, the
    shorter last one too, fit what is laid out for a whole piece."""
    rows = [1, 2, 100, 128, 129, 1000, 2048, 4095, 4096, 5274, 7000, 8192, 12000, 16384, 65536, 1 << 18, 1 << 24]
    vocab = [1, 7, 8, 255, 256, 257, 1000, 17000, 32000, 32003, 37914, 50257, 50304, 50400, 51200, 128256, 151936, 250880, 256000, 600000]
    sizes = [(r, v) for r in rows for v in vocab] + [(r, v) for r in range(4096, 16384, 617) for v in range(20000, 256000, 3557)]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "probe.cc"), os.path.join(d, "probe")
        with open(src, "w") as f:
            f.write(PIECES)
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, src, "-o", exe], check=True)
        out = subprocess.run([exe], input="\n".join(f"{r} {v}" for r, v in sizes), check=True, capture_output=True, text=True).stdout
    several = 0
    for (r, v), line in zip(sizes, out.splitlines(), strict=True):
        columns, count, parts, partials, n, most, end, short_piece = (int(t) for t in line.split())
        assert n == count and end == v and not short_piece, (r, v)
        assert parts >= 1 and most <= partials, (r, v, most, partials)
        assert count == 1 or columns % 256 == 0, (r, v)
        assert 2 * ((r + 255) // 256 * 256) * columns <= (256 << 20) or columns <= 256, (r, v)
        several += count > 1
    assert several > 500


@pytest.mark.parametrize("rows", [1, 128, 129, 5000])
@pytest.mark.parametrize("entries", [0, 9])
def test_the_workspace_query_knows_the_weights_layout(pkg, rows, entries):
    """What Python tells is what the call with this weight will ask for."""
    lib = pkg.load_library()
    x, row_major, column_major = torch.empty(rows, 512), torch.empty(4000, 512), torch.empty(512, 4000).t()
    for backward in (False, True):
        for w, order in ((row_major, pkg.ROW_MAJOR), (column_major, pkg.COL_MAJOR)):
            d = pkg._LinearLossDesc()
            d.rows, d.hidden, d.vocab, d.entries, d.w_order = rows, 512, 4000, entries, order
            want = lib.ixk_linear_loss_workspace_bytes(ctypes.byref(d), int(backward))
            assert pkg.linear_loss_workspace_bytes(x, w, entries, backward) == want > 0


def test_plain_form_with_teacher_logits_at_the_ends_of_the_type(pkg):
    """Entries masked by the type's lowest number are there: alone they weigh alike, beside others nothing."""
    layers = importlib.import_module(pkg.__name__ + ".layers")
    low = torch.finfo(torch.float32).min
    logits = torch.tensor([[low, low, low, low], [1.0, 2.0, low, low], [-low, 0.0, -low, low], [1.0, -math.inf, 3.0, 2.0]])
    index = torch.tensor([[1, 2, 3, 4]] * 4)
    _, q, rows = layers._head_targets(None, torch.empty(10, 8), (index, logits), 0.25)
    e = [math.exp(-4.0), math.exp(-8.0)]
    want = torch.tensor([[0.25] * 4, [e[0] / (1 + e[0]), 1 / (1 + e[0]), 0, 0], [0.5, 0, 0.5, 0],
                         [e[1] / (1 + e[0] + e[1]), 0, 1 / (1 + e[0] + e[1]), e[0] / (1 + e[0] + e[1])]])
    assert rows.all()
    assert (q - want).abs().max() < 1e-6
