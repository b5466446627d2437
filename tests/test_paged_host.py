"""The paged cache operators without a GPU: the index arithmetic of csrc/paged.cuh (which any C++ compiler takes),
and the refusals of the Python and C entry points, which come before any launch."""
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from qwen3_tts_b200 import _lib, ops

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "qwen3-tts-rsi-engine_b200" / "csrc"
BF16 = torch.bfloat16

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include "paged.cuh"
using namespace q3t;
static int bad = 0;
#define CHECK(c) do { if (!(c)) { if (bad++ < 10) printf("line %d: %s\n", __LINE__, #c); } } while (0)

int main() {
  // page table look-ups: in range, and every kind of miss; entries that are not needed are never read
  const int32_t table[3 * 5] = {7, 0, 3, 9, 9, 1, -1, 8, 2147483647, 9, -2147483647 - 1, 4, 6, 5, 9};
  PageTable t = {table, 5, 3, 4, 8, 48};  // 3 sequences, 4 of 5 columns in use, 8 pages of 48 positions
  int row;
  auto look = [&](int64_t s, int64_t p) { return t.lookup(s, p, row); };
  CHECK(look(0, 143) == 3 && row == 47 && look(2, 50) == 4 && row == 2 && look(0, 48) == 0 && row == 0);
  for (int64_t p : {int64_t(0), int64_t(47), int64_t(4294967295), int64_t(4294967296), int64_t(1) << 50})
    CHECK(t.column_of(p) == p / 48);
  CHECK(look(0, 0) == 7 && look(0, 47) == 7 && look(0, 48) == 0 && look(0, 143) == 3);
  CHECK(look(0, 144) == -1);   // page 9 of 8
  CHECK(look(0, 192) == -1);   // past the columns
  CHECK(look(1, 48) == -1 && look(1, 96) == -1 && look(1, 144) == -1 && look(2, 0) == -1);
  CHECK(look(2, 50) == 4 && look(2, -1) == -1);
  CHECK(look(-1, 0) == -1 && look(3, 0) == -1 && look(int64_t(1) << 62, 0) == -1);
  CHECK(look(0, int64_t(1) << 62) == -1 && look(0, -(int64_t(1) << 62)) == -1);
  CHECK(steps_of(-1) == 0 && steps_of(0) == 1 && steps_of(15) == 1 && steps_of(16) == 2);

  // starts of packed sequences: as given while they can be, and safe to count on from
  for (int64_t s : {int64_t(0), int64_t(-5), int64_t(1) << 35, -(int64_t(1) << 35)}) CHECK(clamped_start(s) == s);
  const int64_t last = 9223372036854775807;
  CHECK(clamped_start(last) + 2147483647 > (int64_t(1) << 34) && clamped_start(last) > (int64_t(1) << 34));
  CHECK(clamped_start(-last - 1) + 2147483647 < 0);

  // even splits: the ranges tile [0, total), differ by one at most, and split_owner inverts them
  for (int64_t total : {1, 2, 7, 8, 9, 147, 148, 149, 1000, 4097})
    for (int64_t parts : {1, 2, 8, 148, 296, 1184}) {
      const int64_t ranges = split_parts(total, parts);
      for (int64_t i = 0; i < ranges; ++i) CHECK(split_begin(i + 1, total, ranges) > split_begin(i, total, ranges));
      CHECK(ranges <= parts && split_parts(0, parts) == 0);
      CHECK(split_begin(0, total, parts) == 0 && split_begin(parts, total, parts) == total);
      for (int64_t i = 0; i < parts; ++i) {
        const int64_t b = split_begin(i, total, parts), e = split_begin(i + 1, total, parts);
        CHECK(e >= b && e - b <= (total + parts - 1) / parts);
        for (int64_t s = b; s < e; ++s) CHECK(split_owner(s, total, parts) == i);
      }
    }
  const int64_t huge = int64_t(1) << 46;
  for (int64_t i : {int64_t(0), int64_t(1), int64_t(777), int64_t(1183)}) {
    CHECK(split_owner(split_begin(i, huge, 1184), huge, 1184) == i);
    CHECK(split_owner(split_begin(i + 1, huge, 1184) - 1, huge, 1184) == i);
  }

  // the row of a flattened step, with empty rows anywhere
  srand(5);
  for (int round = 0; round < 200; ++round) {
    const int rows = 1 + rand() % 40, units = 1 + rand() % 9;
    std::vector<int32_t> prefix(1, 0);
    for (int r = 0; r < rows; ++r) prefix.push_back(prefix.back() + (rand() % 3 ? rand() % 6 : 0));
    for (int64_t at = 0; at < int64_t(prefix[rows]) * units; ++at) {
      const int r = row_of(prefix.data(), rows, at, units);
      CHECK(int64_t(prefix[r]) * units <= at && at < int64_t(prefix[r + 1]) * units);
    }
  }
  printf("%s\n", bad ? "FAILED" : "ok");
  return bad != 0;
}
"""


def test_index_arithmetic(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("g++ not found")
    source = tmp_path / "paged_index.cpp"
    source.write_text(PROGRAM)
    build = subprocess.run([compiler, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-Wall", "-I",
                            str(CSRC), "-x", "c++", str(source), "-o", str(tmp_path / "paged_index")],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    run = subprocess.run([str(tmp_path / "paged_index")], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr


# ------------------------------------------------------------------ refusals (tensor arguments)
class FakeCuda(torch.Tensor):
    """A CPU tensor that says it is on cuda:0, so that every check up to the launch runs here."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_subclass(cls, t)

    device = property(lambda self: torch.device("cuda:0"))

    def get_device(self):
        return 0

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        out = super().__torch_function__(func, types, args, kwargs or {})
        return out


def fake(*tensors):
    return [FakeCuda(t) for t in tensors]


@pytest.fixture
def no_launch(monkeypatch):
    """Calls that pass every check end here instead of in a kernel."""
    class Reached(Exception):
        pass

    def call(name, packed, device):
        raise Reached(name)

    monkeypatch.setattr(ops, "_paged_call", call)
    monkeypatch.setattr(ops, "_paged_workspace", lambda what, need, workspace, device: (None, 0, 0))
    monkeypatch.setattr(ops, "paged_decode_attention_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(ops, "paged_prefill_attention_workspace_bytes", lambda *a: 0)
    return Reached


def pool(pages=6, heads=2, size=16, dim=64, dtype=BF16):
    return torch.zeros(pages, heads, size, dim, dtype=dtype)


def table(rows=3, columns=2, dtype=torch.int32):
    return torch.zeros(rows, columns, dtype=dtype)


def index(n, dtype=torch.int64):
    return torch.zeros(n, dtype=dtype)


def decode(**change):
    a = dict(query=torch.zeros(3, 4, 64, dtype=BF16), keys=pool(), values=pool(), page_table=table(), positions=index(3),
             out=torch.zeros(3, 4, 64, dtype=BF16))
    a.update(change)
    a = {k: FakeCuda(v) for k, v in a.items()}
    return ops.paged_decode_attention(a["query"], a["keys"], a["values"], a["page_table"], a["positions"], out=a["out"])


def prompt(**change):
    a = dict(query=torch.zeros(9, 4, 64, dtype=BF16), keys=pool(), values=pool(), page_table=table(), offsets=index(4),
             starts=index(3), out=torch.zeros(9, 4, 64, dtype=BF16))
    a.update(change)
    a = {k: FakeCuda(v) for k, v in a.items()}
    return ops.paged_prefill_attention(a["query"], a["keys"], a["values"], a["page_table"], a["offsets"], a["starts"],
                                       out=a["out"])


def write(**change):
    a = dict(qkv=torch.zeros(3, 8 * 64, dtype=BF16), qw=torch.ones(64, dtype=BF16), kw=torch.ones(64, dtype=BF16),
             cos=torch.zeros(9, 64, dtype=BF16), sin=torch.zeros(9, 64, dtype=BF16), rotary=index(3), at=index(3),
             page_table=table(), keys=pool(), values=pool(), sequences=index(3), out=torch.zeros(3, 4, 64, dtype=BF16))
    a.update(change)
    a = {k: v if v is None else FakeCuda(v) for k, v in a.items()}
    return ops.paged_qk_norm_rope_kv(a["qkv"], a["qw"], a["kw"], 1e-6, a["cos"], a["sin"], a["rotary"], a["at"],
                                     a["page_table"], a["keys"], a["values"], q_heads=4, kv_heads=2, head_dim=64,
                                     sequences=a["sequences"], query_out=a["out"])


@pytest.mark.parametrize("entry", [decode, prompt, write])
def test_valid_arguments_reach_the_launch(entry, no_launch):
    with pytest.raises(no_launch):
        entry()


SHARED = [dict(keys=pool(dtype=torch.float16)), dict(values=pool(heads=1)), dict(values=pool()[:, :, ::2]),
          dict(keys=pool(size=32)[:, :, ::2]), dict(keys=pool()[0]), dict(keys=pool(pages=12)[::2]),
          dict(keys=pool(heads=0), values=pool(heads=0)), dict(keys=pool(pages=0), values=pool(pages=0)),
          dict(page_table=table(dtype=torch.int64)), dict(page_table=table(columns=4)[:, ::2]),
          dict(page_table=table(rows=2)), dict(page_table=table()[0])]
BAD = [(decode, c) for c in SHARED + [
    dict(query=torch.zeros(3, 4, 64)), dict(query=torch.zeros(3, 3, 64, dtype=BF16)),
    dict(query=torch.zeros(3, 4, 128, dtype=BF16)), dict(query=torch.zeros(3, 8, 64, dtype=BF16)[:, ::2]),
    dict(query=torch.zeros(3, 4, 128, dtype=BF16)[..., ::2]), dict(query=torch.zeros(4, 64, dtype=BF16)),
    dict(positions=index(2)), dict(positions=index(3, torch.int32)), dict(positions=index(6)[::2]),
    dict(positions=index(3)[:, None]), dict(positions=index(6)[::2]), dict(out=torch.zeros(3, 4, 64)), dict(out=torch.zeros(2, 4, 64, dtype=BF16)),
    dict(out=torch.zeros(6, 4, 64, dtype=BF16)[::2])]]
BAD += [(prompt, c) for c in SHARED + [
    dict(offsets=index(3)), dict(offsets=index(4, torch.int32)), dict(starts=index(2)), dict(starts=index(6)[::2]),
    dict(out=torch.zeros(9, 4, 64)), dict(query=torch.zeros(9, 5, 64, dtype=BF16))]]
BAD += [(write, c) for c in SHARED[:-2] + [
    dict(qkv=torch.zeros(3, 8 * 64)), dict(qkv=torch.zeros(3, 7 * 64, dtype=BF16)),
    dict(qkv=torch.zeros(3, 16 * 64, dtype=BF16)[:, ::2]), dict(qw=torch.ones(64)), dict(kw=torch.ones(32, dtype=BF16)),
    dict(cos=torch.zeros(9, 64)), dict(sin=torch.zeros(8, 64, dtype=BF16)), dict(cos=torch.zeros(9, 32, dtype=BF16)),
    dict(rotary=index(2)), dict(at=index(3, torch.int32)), dict(sequences=index(4)),
    dict(sequences=None, page_table=table(rows=2)), dict(out=torch.zeros(3, 2, 64, dtype=BF16))]]


@pytest.mark.parametrize("entry,change", BAD, ids=lambda v: getattr(v, "__name__", None) or "-".join(v))
def test_bad_arguments_are_refused_before_the_launch(entry, change, no_launch):
    with pytest.raises(ValueError):
        entry(**change)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_decode_attention(torch.zeros(3, 4, 64, dtype=BF16), pool(), pool(), table(), index(3))


# ------------------------------------------------------------------ refusals (C entry points; nothing is dereferenced)
A16 = 1 << 20  # an aligned address that no call gets to use


CACHE = dict(keys=A16, values=A16, page_stride=2048, pages=6, page_size=16, kv=2, dim=64, table=A16, table_stride=2,
             table_rows=3, columns=2, device=-1)


def c_call(name, layout, fields, change):
    """A packed call with some fields changed, in the order of the C struct."""
    assert set(change) <= {*CACHE, *fields}
    values = [0 if v is None else v for v in ({**CACHE, **fields} | change).values()]
    return getattr(_lib.load(), name)(layout.pack(*values), None, None)


def c_decode(**change):
    return c_call("q3t_paged_decode_attention", _lib.PAGED_DECODE, dict(
        query=A16, query_stride=256, rows=3, q=4, positions=A16, out=A16, context=32, scale=0.125, workspace=None,
        workspace_bytes=0), change)


def c_prompt(**change):
    return c_call("q3t_paged_prefill_attention", _lib.PAGED_PREFILL, dict(
        query=A16, query_stride=256, rows=9, q=4, offsets=A16, starts=A16, sequences=3, out=A16, scale=0.125,
        workspace=None, workspace_bytes=0), change)


def c_write(**change):
    return c_call("q3t_paged_qk_norm_rope_kv", _lib.PAGED_WRITE, dict(
        qkv=A16, stride=512, rows=3, q=4, qw=A16, kw=A16, cos=A16, sin=A16, length=9, rotary=A16, at=A16,
        sequences=None, query=A16, eps=1e-6), change)


POOLS = [(dict(keys=None), -1), (dict(values=A16 + 2), -1), (dict(page_stride=2047), -1), (dict(page_stride=1 << 41), -1),
         (dict(pages=0), -1), (dict(pages=1 << 31), -1), (dict(page_size=24), -2), (dict(page_size=0), -2),
         (dict(page_size=1 << 20), -2), (dict(kv=0), -1), (dict(dim=96), -2), (dict(table=None), -1),
         (dict(columns=0), -1), (dict(table_stride=1), -1), (dict(rows=0), -1),
         (dict(table_rows=0), -1), (dict(table_rows=2), -1),
         (dict(columns=(1 << 30) + 1, table_stride=1 << 31), -2)]
C_BAD = [(c_decode, c, rc) for c, rc in POOLS + [
    (dict(query_stride=255), -1), (dict(query_stride=260), -1), (dict(q=5), -1), (dict(query=A16 + 8), -1),
    (dict(context=33), -1), (dict(context=0), -1), (dict(positions=None), -1), (dict(rows=1 << 31), -1)]]
C_BAD += [(c_prompt, c, rc) for c, rc in POOLS + [
    (dict(offsets=None), -1), (dict(starts=None), -1), (dict(sequences=0), -1), (dict(out=A16 + 4), -1), (dict(q=3), -1)]]
C_BAD += [(c_write, c, rc) for c, rc in POOLS + [
    (dict(stride=511), -1), (dict(stride=516), -1), (dict(qw=None), -1), (dict(cos=None), -1), (dict(length=0), -1),
    (dict(qkv=A16 + 8), -1), (dict(rows=1 << 40), -1)]]


def test_packed_layouts_match_the_header(tmp_path):
    """sizeof the C structs, and the offset of the last field of each, as a C compiler sees them."""
    compiler = shutil.which("gcc")
    if compiler is None:
        pytest.skip("gcc not found")
    source = tmp_path / "sizes.c"
    source.write_text("""#include <stdio.h>
#include "q3t.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %zu %zu\\n", sizeof(q3t_paged_cache), sizeof(q3t_paged_write), sizeof(q3t_paged_decode),
         sizeof(q3t_paged_prefill), offsetof(q3t_paged_write, eps), offsetof(q3t_paged_decode, scale),
         offsetof(q3t_paged_prefill, scale));
  return 0;
}
""")
    subprocess.run([compiler, "-std=c99", "-I", str(ROOT / "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True).stdout.split()]
    sizes = [s.size for s in (_lib.PAGED_WRITE, _lib.PAGED_DECODE, _lib.PAGED_PREFILL)]
    assert got == [96, *sizes, sizes[0] - 8, sizes[1] - 24, sizes[2] - 24]


@pytest.mark.parametrize("entry,change,rc", C_BAD, ids=lambda v: getattr(v, "__name__", None) or str(v))
def test_c_entry_points_refuse(entry, change, rc):
    if not _lib.LIBRARY_PATH.exists():
        pytest.skip("libq3t_b200.so not built (run __graft_entry__.build())")
    before = _lib.launch_count()
    assert entry(**change) == rc
    assert "paged" in _lib.last_error()
    assert _lib.launch_count() == before
