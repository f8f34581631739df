"""Where the attention kernels of the 4-bit cache look, up to the longest sequence they admit: csrc/qf_kv4_places.h compiled for
the host, with the compiler's checks of overflow and conversion on."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MOST = 2 ** 31 - 64  # positions of a request

_STAGES = """
// One workgroup of attn_tile_kernel over stages first .. n - 1 of a sequence: every place it looks up, in its order.
static long look_ups(int end, int first, int n, int last_tile) {
  long wrong = 0;
  auto look_up = [&](int stage) {
    for (int lane = 0; lane < 64; ++lane) {
      const long want = std::min((long)stage * 64 + lane * 16, (long)last_tile);
      wrong += qfk::stage_record(stage, lane, last_tile) != want;
    }
  };
  look_up(first / 16 * 16);
  if ((first + 1) % 16 == 0) look_up(first + 1);
  for (int stage = std::max(first, n - 200); stage < n; ++stage)
    if ((stage + 2) % 16 == 0) look_up(stage + 2);
  return wrong;
}
int main() {
  for (long end : {1l, 16l, 17l, 64l, 65l, 1024l, 1025l, 2147483584l - 1024, 2147483584l - 64, 2147483584l - 63, 2147483584l - 1,
                   2147483584l}) {
    const int n = (int)((end + 63) / 64), last_tile = (int)((end - 1) / 16 * 16);
    for (int first : {0, std::max(n - 17, 0), n - 1})
      if (const long wrong = look_ups((int)end, first, n, last_tile)) printf("end %ld first %d: %ld\\n", end, first, wrong);
  }
  return 0;
}
"""


def _run(tmp_path, body):
    (tmp_path / "p.cpp").write_text('#include <algorithm>\n#include <cstdio>\n#include "qf_kv4_places.h"\n' + body)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "qwen-a100-fastpath_amd", "csrc"),
                    "-o", tmp_path / "p", tmp_path / "p.cpp"], check=True)
    return subprocess.run([tmp_path / "p"], check=True, capture_output=True, text=True, timeout=60).stdout


def test_a_stage_ahead_of_the_last_is_looked_up_inside_the_sequence(tmp_path):
    assert _run(tmp_path, _STAGES) == ""


_CHUNKS = """
// A batch of so many requests of `steps` each: the chunks that they are cut to, which have workers + requests places.
int main() {
  const long most = 1l << 26;
  for (long requests : {1l, 65l, 129l, 4096l, 65535l})
    for (long workers : {1l, 2l, 32l, 256l, 768l})
      for (long steps : {1l, 3l, 1000l, most / 2, most - 2}) {
        const long chunk = qfk::chunk_steps((uint64_t)(requests * steps), (uint32_t)workers);
        const long chunks = requests * ((steps + chunk - 1) / chunk);
        if (chunk < 1 || chunk > most || chunks > workers + requests)
          printf("%ld requests of %ld steps over %ld: %ld chunks of %ld\\n", requests, steps, workers, chunks, chunk);
      }
  return 0;
}
"""


def test_a_batch_has_no_more_chunks_than_places(tmp_path):
    assert _run(tmp_path, _CHUNKS) == ""
