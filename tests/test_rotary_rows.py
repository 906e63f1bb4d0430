"""ringattn_rotary_apply without a GPU: outputs that have rows of the other tensor are refused before any HIP call, by the rule that the header's
ringattn::rotary::rows_meet is, which is held here against all rows one by one."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from ringattention_amd._lib import RingattnRotary, RingattnRows

E_SHAPE = 6
D, HEADS, TOKENS, BATCH = 64, 4, 5, 2


def test_an_output_on_rows_of_the_other_tensor_is_refused(ralib):
    memory = np.zeros(8 << 20, dtype=np.uint8)
    x = memory.ctypes.data + (-memory.ctypes.data % 16)
    far, mid = x + (6 << 20), x + (4 << 20)
    r = RingattnRotary(D, 0, 0, 1.0, x)

    def call(first, second, batch=1, tokens=TOKENS):
        """(in, out, heads, strides of both) of two tensors."""
        rows = (RingattnRows * 2)(*(RingattnRows(i, o, n, *s, *s) for i, o, n, s in (first, second)))
        return ralib.ringattn_rotary_apply(ctypes.byref(r), D, 0, rows, 2, batch, tokens, None, 0, None)

    # a fused product [batch, tokens, heads, D] of which K begins among Q's heads: in place, and of outputs alone
    w = (HEADS + 2) * D
    s = (TOKENS * w, D, w)
    for batch in (1, BATCH):
        for step in ((HEADS - 1) * D, 8, HEADS * D - 8, D):
            assert call((mid, mid, HEADS, s), (mid + 2 * step, mid + 2 * step, 2, s), batch) == E_SHAPE, step
            assert call((mid + 2 * step, mid + 2 * step, 2, s), (mid, mid, HEADS, s), batch) == E_SHAPE, step
            assert call((x, mid, HEADS, s), (far, mid + 2 * step, 2, s), batch) == E_SHAPE, step
            assert call((x, mid, HEADS, s), (mid + 2 * step, far, 2, s), batch) == E_SHAPE, step
    # K that begins a token, or a batch, too early or too late
    assert call((mid, mid, HEADS, s), (mid + 2 * w, mid + 2 * w, 2, s)) == E_SHAPE
    assert call((mid, mid, HEADS, s), (mid - 2 * w * (TOKENS - 1), mid - 2 * w * (TOKENS - 1), 2, s)) == E_SHAPE
    assert call((mid, mid, HEADS, s), (mid + 2 * s[0], mid + 2 * s[0], 2, s), BATCH) == E_SHAPE
    assert call((mid, mid, HEADS, s), (mid - 2 * s[0], mid - 2 * s[0], 2, s), BATCH) == E_SHAPE
    # head by head
    s = ((HEADS + 2) * TOKENS * D, TOKENS * D, D)
    for batch in (1, BATCH):
        assert call((mid, mid, HEADS, s), (mid + 2 * (HEADS - 1) * TOKENS * D, mid + 2 * (HEADS - 1) * TOKENS * D, 2, s), batch) == E_SHAPE


@pytest.mark.skipif(not shutil.which("g++"), reason="no host compiler")
def test_the_rule_against_all_rows(tmp_path):
    """Random strides, offsets and sizes: what is apart has no row on another, what meets has one, and equal strides always tell."""
    with open(os.path.join(ROOT, "ringattention_amd", "csrc", "ringattn_rotary.h")) as f:
        text = f.read()
    rule = text[text.index("struct RowsAt {"):text.index("struct Rows {")]
    source = "#include <cstdint>\n#include <cstdio>\n#include <cstdlib>\n#include <random>\n" + rule + r'''
int main() {
  std::mt19937 g(1);
  auto r = [&](int lo, int hi) { return lo + (int)(g() % (unsigned)(hi - lo + 1)); };
  long told[3] = {0, 0, 0};
  for (int it = 0; it < 400000; ++it) {
    const int dim = 8 * r(1, 2), tokens = r(1, 5), ha = r(1, 5), hb = r(1, 5);
    RowsAt a{(void*)(uintptr_t)100000, 8 * r(0, 24), 8 * r(0, 24), ha};
    if (r(0, 1)) { a.hs = dim * r(1, 3); a.ts = a.hs * ha + 8 * r(0, 12); }
    else if (r(0, 1)) { a.ts = dim * r(1, 3); a.hs = a.ts * tokens + 8 * r(0, 5); }
    const long heads_span = ha > 1 ? (ha - 1) * a.hs + dim : dim, tokens_span = (tokens - 1) * a.ts + dim;
    if ((tokens > 1 && a.ts < dim) || (ha > 1 && a.hs < dim) || (tokens > 1 && ha > 1 && a.ts < heads_span && a.hs < tokens_span)) continue;  // rows on each other
    RowsAt b{(void*)(uintptr_t)(100000 + 16 * r(-80, 80)), r(0, 2) ? a.ts : 8 * r(0, 24), r(0, 2) ? a.hs : 8 * r(0, 24), hb};
    bool meet = false;
    for (int i = 0; i < tokens; ++i)
      for (int h = 0; h < ha; ++h)
        for (int j = 0; j < tokens; ++j)
          for (int e = 0; e < hb; ++e)
            meet = meet || std::labs(50000 + i * a.ts + h * a.hs - ((long)(uintptr_t)b.at / 2 + j * b.ts + e * b.hs)) < dim;
    const Meet said = rows_meet(a, b, tokens, dim);
    ++told[(int)said];
    const bool alike = (tokens == 1 || a.ts == b.ts) && (ha == 1 || hb == 1 || a.hs == b.hs) && ha >= hb;
    if ((said == Meet::kApart && meet) || (said == Meet::kMeet && !meet) || (alike && said == Meet::kUnknown)) {
      std::printf("%d: a %ld %ld %d, b %ld %ld %d at %ld, %d tokens of %d\n", (int)said, (long)a.ts, (long)a.hs, ha, (long)b.ts, (long)b.hs, hb, ((long)(uintptr_t)b.at - 100000) / 2, tokens, dim);
      return 1;
    }
  }
  std::printf("%ld %ld %ld\n", told[0], told[1], told[2]);
  return !(told[0] > 10000 && told[1] > 10000);
}
'''
    at = tmp_path / "rule.cpp"
    at.write_text(source)
    subprocess.run(["g++", "-O2", "-o", str(tmp_path / "rule"), str(at)], check=True)
    res = subprocess.run([str(tmp_path / "rule")], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout
