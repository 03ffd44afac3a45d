"""How the row kernels of the norms lay rows out, over all widths, without a GPU: the layout's own source compiled for
the host."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def run(tmp_path, body):
    """The lines that a C++ program with the row layout in scope prints."""
    source = tmp_path / "probe.cpp"
    source.write_text('#include <cstdio>\n#include "rows_layout.cuh"\nusing namespace p3d::rows;\nint main() {\n%s\n}\n' % body)
    exe = tmp_path / "probe"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(ROOT / "include"), "-I", str(ROOT / "pack3d_b200" / "csrc"),
                    str(source), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()


def test_every_cta_has_columns_of_its_row(tmp_path):
    """A CTA of a row's cluster without columns would read the gate of a sample past its end."""
    lines = run(tmp_path, """
  for (int dim = 1; dim <= 16384; ++dim)
    for (int dtype : {P3D_F32, P3D_F16, P3D_BF16})
      for (bool backward : {false, true}) {
        const Shape s = shape_of(dim, dtype, backward);
        const bool held = s.members * s.columns() >= dim, empty = (s.members - 1) * s.columns() >= dim;
        const bool fits = s.members >= 1 && s.members <= 8 && s.row_threads * s.groups <= 512 && s.groups >= 1 &&
                          s.groups <= kMaxGroups && (s.members == 1 || s.groups == 1);
        if (!held || empty || !fits) std::printf("%d %d %d\\n", dim, dtype, (int)backward);
      }
""")
    assert lines == []


@pytest.mark.parametrize("dim,members", [(8192, 4), (8200, 7), (8960, 7), (8968, 8), (12296, 7), (16384, 8)])
def test_ctas_of_wide_fp32_rows(tmp_path, dim, members):
    assert run(tmp_path, f'std::printf("%d", shape_of({dim}, P3D_F32, true).members);') == [str(members)]


def test_copied_pieces_stay_in_the_tensor(tmp_path):
    """Unaligned batches are copied in whole 16-byte pieces: for every row length, start of the tensor and batch, the
    pieces of a batch that is copied lie inside the tensor, and batches away from the ends are copied."""
    lines = run(tmp_path, """
  const int rows = 40;
  for (int bytes = 2; bytes <= 66; bytes += 2)
    for (int base = 0; base < 16; base += 2)
      for (int row = 0; row < rows; ++row)
        for (int n = 1; n <= 8 && row + n <= rows; ++n) {
          const int start = base + row * bytes, size = n * bytes, total = base + rows * bytes;
          const uint32_t shift = start & 15;
          const int from = start - (int)shift, to = from + (int)piece_bytes(shift, size);
          const bool kept = !in_place(row, n, rows, edge_rows(bytes));
          const bool inside = from >= base && to <= total, wide = from % 16 == 0 && to >= start + size;
          const bool middle = row >= 8 && row + n <= rows - 8;
          if ((kept && !(inside && wide)) || (middle && !kept)) std::printf("%d %d %d %d\\n", bytes, base, row, n);
        }
""")
    assert lines == []


@pytest.mark.parametrize("bytes_,edge", [(2, 8), (4, 4), (6, 3), (14, 2), (16, 1), (4004, 1)])
def test_rows_read_in_place(tmp_path, bytes_, edge):
    assert run(tmp_path, f'std::printf("%d", edge_rows({bytes_}));') == [str(edge)]


RING = """
  // One warp of a group that issues and uses: the kernels' own order of calls on a model of the barriers.  Batch `lost`
  // never arrives.
  for (int stages = 2; stages <= 4; ++stages)
    for (int batches = 1; batches <= 13; ++batches)
      for (int lost = -1; lost < batches; ++lost) {
        RingState r;
        int loaded = 0, used = 0, out = 0, held[4] = {-1, -1, -1, -1}, phases[4] = {1, 1, 1, 1};
        bool bad = false, seen[16] = {};
        auto arrived = [&](int s, int phase) {   // the batch that this stage holds in this phase
          const bool right = held[s] >= 0 && phases[s] == phase;
          if (!right || seen[held[s]]) bad = true;
          if (right && held[s] == lost) { ++out; return false; }
          if (right) seen[held[s]] = true;
          return right;
        };
        auto issue = [&] {
          if (!r.ok || loaded == batches) return;
          const int s = r.load(stages);
          if (held[s] >= 0 && !seen[held[s]]) bad = true;   // over a batch that may still be on its way
          held[s] = loaded++;
          phases[s] ^= 1;
        };
        for (int i = 0; i < stages - 1; ++i) issue();
        for (int b = 0; b < batches; ++b) {
          const int s = r.use(stages, arrived);
          if (s < 0 || s >= stages || (r.ok && held[s] != b)) bad = true;
          if (r.ok) ++used;
          issue();
        }
        const int before = out;
        if (!r.ok) r.drain(stages, arrived);
        for (int b = 0; b < loaded; ++b)
          if (!seen[b] && b != lost) bad = true;     // every copy on its way was waited for
        if (bad || r.ok != (lost < 0) || used != (lost < 0 ? batches : lost) || before != (lost >= 0) || out > 2)
          std::printf("%d %d %d\\n", stages, batches, lost);
      }
"""


def test_ring_stops_at_a_batch_that_does_not_arrive(tmp_path):
    """After a wait that ran out nothing is used, no further batch is loaded or waited for, and the end waits for what is
    on its way, each batch once; without one, every batch is used in order."""
    assert run(tmp_path, RING) == []
