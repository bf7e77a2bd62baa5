"""Host-side bounds of the decode operators, without a GPU: which notes on shared rows the
attention's second kernel follows, and the sizes that its workspace query takes."""

import subprocess

import pytest

from kernelpilot_b200 import build, ext

PROGRAM = r"""
#include <cstdio>
#include "kp_kv_cache.cuh"
int main() {
  int first, count, workers;
  while (std::scanf("%d %d %d", &first, &count, &workers) == 3)
    std::puts(kpb::note_is_sound(first, count, workers) ? "1" : "0");
}
"""


def test_no_note_leads_past_the_partials(tmp_path):
    # what the kernel reads for a note it follows: partials of workers first / 2 to
    # first / 2 + count - 1, in arithmetic without an end
    src, exe = tmp_path / "notes.cu", tmp_path / "notes"
    src.write_text(PROGRAM)
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr",
                    f"-I{build.INCLUDE}", f"-I{build.CSRC}", str(src), "-o", str(exe)], check=True)
    ends = [0, 1, 2, 3, 7, 8, 2367, 2368, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1]
    ends += [-e for e in ends] + [-2 ** 31]
    cases = [(f, c, w) for f in ends for c in ends for w in (0, 1, 4, 2368, 4736)]
    out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, c)) for c in cases),
                         capture_output=True, text=True, check=True).stdout.split()
    assert len(out) == len(cases)
    for (first, count, workers), got in zip(cases, out, strict=True):
        want = first >= 0 and count >= 0 and first // 2 < workers and first // 2 + count <= workers
        assert got == str(int(want)), (first, count, workers)


@pytest.mark.parametrize("B", [1, 4, 1 << 20])
def test_workspace_query_of_lengths_past_the_limit(B):
    # max_pages * page_size must be below 2^31; the query answers 0 for what the call refuses,
    # and never less for a longer table than for a shorter one
    query = ext.capi().kpb_paged_attention_workspace_bytes
    sizes = [query(1, B, 32, 8, 128, n) for n in (1, 16, 1000, 1 << 20, (1 << 31) - 1)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    for n in (1 << 31, 1 << 40, (1 << 63) - 1, -1):
        assert query(1, B, 32, 8, 128, n) == 0
