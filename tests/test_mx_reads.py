"""Addresses of the reads of rows at odd places, run on the CPU: the code that the kernels run,
compiled for the host, on two rows of a matrix whose gaps cannot be read at all."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

SOURCE = r'''
#include <sys/mman.h>
#include <unistd.h>
#include <cstdio>
#include <cstring>
#include "mx_common.cuh"

static long fails = 0;

// what was read: element i of `w`, against element c + i of the row or zero behind it
template <typename U>
void check(const void* w, int n, const U* row, long len, long c) {
  for (int i = 0; i < n; ++i) {
    U got, want = 0;
    std::memcpy(&got, static_cast<const char*>(w) + i * sizeof(U), sizeof(U));
    if (c + i < len) want = row[c + i];
    if (got != want) ++fails;
  }
}

template <int DT, typename U>
void rows(char* page, long size, long len) {
  using T = typename b200::Elem<DT>::T;
  for (int at_end = 0; at_end < 2; ++at_end) {  // against the gap before the row, or behind it
    for (long shift = 0; shift < 16 / long(sizeof(U)); ++shift) {
      const long bytes = len * long(sizeof(U)), move = shift * long(sizeof(U));
      char* at = at_end ? page + size - bytes - move : page + move;
      if (at < page || at + bytes > page + size) continue;
      U* row = reinterpret_cast<U*>(at);
      for (long i = 0; i < len; ++i) row[i] = U(0x3C01u + 7 * i);
      for (long c = 0; c < len + 33; c += 16) {
        b200::Raw16<DT> w;
        w.load_any(reinterpret_cast<const T*>(row), len, c);
        check<U>(w.r, 16, row, len, c);
      }
      for (long c = 0; c < len; c += 16 / long(sizeof(U))) {
        uint32_t w[4];
        b200::load_words_any<DT, 4>(reinterpret_cast<const T*>(row), len, c, w);
        check<U>(w, 16 / int(sizeof(U)), row, len, c);
      }
    }
  }
}

int main() {
  const long size = sysconf(_SC_PAGESIZE);
  char* m = static_cast<char*>(mmap(nullptr, 5 * size, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
  if (m == MAP_FAILED) return 2;
  long n = 0;
  for (int p = 1; p < 5; p += 2) {  // rows in pages 1 and 3; 0, 2 and 4 fault
    if (mprotect(m + p * size, size, PROT_READ | PROT_WRITE)) return 2;
    for (long len : {1, 2, 3, 5, 7, 8, 9, 15, 16, 17, 23, 31, 32, 33, 47, 63, 64, 65, 511, 512, 513}) {
      rows<0, uint16_t>(m + p * size, size, len);
      rows<1, uint16_t>(m + p * size, size, len);
      rows<3, uint32_t>(m + p * size, size, len);
      ++n;
    }
  }
  std::printf("%ld lengths, %ld wrong\n", n, fails);
  return fails ? 1 : 0;
}
'''


def test_rows_are_read_and_nothing_beside_them(tmp_path):
    src, exe = tmp_path / "reads.cu", tmp_path / "reads"
    src.write_text(SOURCE)
    subprocess.run(["nvcc", "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a",
                    f"-I{ROOT / 'hopper-lab_b200' / 'csrc'}", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout)  # -11: it read a gap
    assert "42 lengths, 0 wrong" in r.stdout


def test_kernels_bound_their_reads_by_the_row():
    """Every caller hands over the start of a row and its length, not the matrix's span."""
    text = (ROOT / "hopper-lab_b200" / "csrc" / "mx_quant.cu").read_text()
    assert text.count("load_any(") + text.count("load16_any<") + text.count("load_words_any<") >= 6
    for span in ("(p.rows - 1) * p.ld", "(p.cols - 1) * p.ld"):
        assert span not in text
