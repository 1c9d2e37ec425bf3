"""The groups of rows that share a prefix, as la_groups.cuh reads them, compiled
for the CPU. The plan counts a row's own keys by the groups that hold it, the
warps that read them look its group up; both have to say the same for any
bounds, sound or not, and no row may be in two groups that share."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent

SOURCE = r"""
#include <algorithm>
using std::max;
using std::min;
template <typename T> T __ldcg(const T* p) { return *p; }
#include "la_groups.cuh"
using namespace la;

static PrefixGroups groups(const int* cu, const int* lens, int n, int batch, int bs, long long cap) {
  return PrefixGroups{cu, lens, n, batch, bs, (bs & (bs - 1)) == 0 ? __builtin_ctz(bs) : -1, cap};
}

// The table as the plan fills it; the groups that share, and for each row with
// ctx keys those that its group covers: by the groups one after another
// (planned), and looked up (read).
extern "C" void divide(const int* cu, const int* lens, int n, int batch, int bs, long long cap, const int* ctx,
                       int* out, int* planned, int* read) {
  const PrefixGroups G = groups(cu, lens, n, batch, bs, cap);
  static PrefixGroup tab[kMaxGroups];
  bool sound = true;
  for (int g = 0; g < n; ++g) {
    sound &= run_of_rows(G, cu[g], cu[g + 1]);
    if (n <= kMaxGroups) tab[g] = load_group(G, g);
  }
  if (!sound) std::fill(tab, tab + min(n, kMaxGroups), PrefixGroup{0, 0, 0});
  if (n > kMaxGroups) tab->rows = sound;
  std::fill(planned, planned + batch, 0);
  for (int g = 0; g < n; ++g) {
    const PrefixGroup r = prefix_group(G, tab, g);
    out[3 * g] = r.first, out[3 * g + 1] = r.rows, out[3 * g + 2] = r.keys;
    for (int b = r.first; b < r.first + r.rows; ++b)
      if (ctx[b] >= r.keys) planned[b] = r.keys;
  }
  for (int b = 0; b < batch; ++b) read[b] = prefix_keys(G, tab, b, ctx[b]);
}
"""


@pytest.fixture(scope="module")
def divide(tmp_path_factory):
    d = tmp_path_factory.mktemp("groups")
    (d / "groups.cpp").write_text(SOURCE)
    so = d / "groups.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-shared", "-fPIC", f"-I{REPO}/lean-infer_b200/csrc",
                    f"-I{REPO}/include", "-I/usr/local/cuda/include", "-o", str(so), str(d / "groups.cpp")], check=True)
    f = ctypes.CDLL(str(so)).divide

    def call(cu, lens, batch, bs, cap, ctx):
        n = len(lens)
        arr = lambda x: (ctypes.c_int * max(1, len(x)))(*x)  # noqa: E731
        out, planned, read = arr([0] * 3 * n), arr([0] * batch), arr([0] * batch)
        f(arr(cu), arr(lens), n, batch, bs, ctypes.c_longlong(cap), arr(ctx), out, planned, read)
        return [tuple(out[3 * g:3 * g + 3]) for g in range(n)], list(planned)[:batch], list(read)[:batch]

    return call


def _check(divide, cu, lens, batch, bs, cap, ctx):
    groups, planned, read = divide(cu, lens, batch, bs, cap, ctx)
    assert planned == read
    seen = set()
    for first, rows, keys in groups:
        if rows and keys:
            mine = set(range(first, first + rows))
            assert 0 <= first and first + rows <= batch and not mine & seen
            seen |= mine
    sound = all(0 <= a <= b <= batch for a, b in zip(cu, cu[1:]))
    want = [0] * batch
    for g, n in enumerate(lens if sound else []):
        keys = min(max(n, 0), cap) // bs * bs if cu[g + 1] - cu[g] >= 2 else 0
        for b in range(cu[g], cu[g + 1]):
            want[b] = keys if ctx[b] >= keys else 0
    assert read == want


# the second list of bounds that run backwards leaves two overlapping runs of rows
@pytest.mark.parametrize("cu", [[0, 2, 99], [0, 100, 50, 128], [0, 3, 2], [-1, 2, 4], [10, 60, 20, 70, 30, 128],
                                [0, 128, 0, 128], [5, 5, 4, 128], [0, 64, 128]])
@pytest.mark.parametrize("empty", [0, 30, 600])
def test_bounds_that_run_backwards(divide, cu, empty):
    cu = cu + [cu[-1]] * empty
    _check(divide, cu, [256] * (len(cu) - 1), 128, 16, 4096, [300] * 100 + [200] * 28)


@pytest.mark.parametrize("seed", range(200))
def test_random_bounds(divide, seed):
    r = random.Random(seed)
    batch, bs = r.choice((1, 7, 128, 300)), r.choice((16, 48, 256))
    n = r.choice((1, 2, 5, 32, 33, 512, 513, 700))
    cu = sorted(r.randint(0, batch) for _ in range(n + 1))
    for _ in range(r.choice((0, 0, 1, 3))):  # some bounds out of order, or out of the batch
        cu[r.randrange(n + 1)] = r.randint(-2, batch + 2)
    lens = [r.choice((0, bs, r.randint(-3, 3000), 10 ** 9)) for _ in range(n)]
    _check(divide, cu, lens, batch, bs, 2048 // bs * bs, [r.randint(0, 2048) for _ in range(batch)])


def test_all_lanes_entries_are_published_with_the_plan():
    """Every lane fills entries of the table, one lane arrives for all of them.
    Shuffles and votes between do not order memory: the other lanes' stores are
    published only if the warp synchronises before that lane arrives."""
    text = (REPO / "lean-infer_b200" / "csrc" / "la_prefix.cu").read_text()
    made = text.index("make_plan(p, tab, in, lane)")
    published = text.index("mbar_arrive(bars.planned())", made)
    assert text[made:published].count("__syncwarp();") == 1
    assert text.index("__syncwarp();", made) < text.index("if (lane == 0)", made) < published
