"""Host logic of the residual recurrent block on the CPU: what the binding takes for shared memory, and which kernel a
product of a size takes."""

import random
import subprocess
import sys

import pytest

from daydreamer_amd import hipops


def touched(at, step, width, rows):
  return {at + k * step + j for k in range(rows) for j in range(width)}


def test_views_that_share_memory():
  """Against sets of bytes: columns of one buffer side by side, rows in between, another stride, single rows, nothing."""
  hipops.load_library()
  from daydreamer_amd import _block
  rng = random.Random(0)
  seen = {True: 0, False: 0}
  for _ in range(20000):
    views = []
    for _ in range(2):
      width, rows = rng.randint(0, 6), rng.randint(0, 5)
      step = rng.choice([8, 8, 8, 16, 24, 11, width])
      step = 0 if rows <= 1 else max(step, width)
      views.append((rng.randint(1000, 1060), step, width, rows))
    a, b = views
    want = bool(touched(*a) & touched(*b))
    assert _block.overlap(*a, *b) == want == _block.overlap(*b, *a), (a, b)
    seen[want] += 1
  assert min(seen.values()) > 2000
  for a, b, want in [((0, 4096, 64, 1 << 30), (64, 4096, 64, 1 << 30), False),       # side by side
                     ((0, 4096, 65, 1 << 30), (64, 4096, 64, 1 << 30), True),
                     ((0, 4096, 64, 1 << 30), (4096 * (1 << 30), 4096, 64, 1 << 30), False),   # one behind the other
                     ((0, 4096, 64, 1 << 30), (4096 * ((1 << 30) - 1) + 63, 0, 1, 1), True),
                     ((0, 4096, 64, 1 << 30), (4096 * ((1 << 30) - 1) + 64, 0, 1, 1), False)]:
    assert _block.overlap(*a, *b) is want
  with pytest.raises(TypeError):
    _block.overlap(1, 2, 3)


def test_the_library_loads_without_the_native_binding():
  """Without _block.so everything but the block's methods works; those say what is missing."""
  code = """
import sys
sys.modules['daydreamer_amd._block'] = None     # what an import of a missing module finds
from daydreamer_amd import hipops
lib = hipops.load_library()
assert lib.dd_version() == hipops.ABI_VERSION and hipops.load_library() is lib
ops = object.__new__(hipops.HipOps)
ops._index, ops._ws_ptr, ops.ws_bytes = 0, 0, 0
try:
  ops.quant_rows(None, None, None)
except RuntimeError as e:
  assert '_block.so not found' in str(e) and 'build()' in str(e), e
else:
  raise SystemExit('not refused')
"""
  subprocess.run([sys.executable, '-c', code], check=True, timeout=120)


def test_plans_of_products():
  """dd_linear_plan is host logic: few rows, tiles in one or two launches, the general kernel, and what it refuses."""
  import ctypes
  lib, plan = hipops.load_library(), (ctypes.c_int * 8)()

  def ask(what, M, N, K, type=1, act=0, ldr=0, z=0, ldp=None, ws=2048 << 20):
    k, q = K if what == 0 else N, K
    rc = lib.dd_linear_plan(what, type, M, N, K, ldp or k, q, act, ldr, z, ws, plan)
    return list(plan) if rc == 0 else lib.dd_last_error().decode()
  assert ask(0, 8, 2048, 1024)[:2] == [0, 16] and ask(0, 100, 2048, 1024)[:2] == [0, 128]
  assert ask(0, 100, 100, 100)[0] == 2 and ask(0, 100, 100, 100, ldp=1 << 24)[0] == 2
  assert ask(0, 8192, 8192, 8192) == [1, 256, 256, 1, 0, 0, 0, 0]
  assert ask(0, 37500, 1024, 2048, ldr=1024) == [1, 192, 128, 1, 32768, 256, 256, 1]     # whole rounds, and the rest
  assert ask(2, 37500, 1024, 2048)[3] > 1 and ask(2, 37500, 1024, 2048, ws=0)[3] == 1   # no room, no split
  assert 'dd_linear_plan' in ask(1, 8, 8, 8, type=2) and 'dd_linear_plan' in ask(0, 0, 8, 8)
  assert 'dd_linear_plan' in ask(3, 8, 8, 8) and 'dd_linear_plan' in ask(0, 8, 8, 8, type=0) and 'dd_linear_plan' in ask(0, 8, 8, 8, act=9)


def test_a_library_of_another_version_is_named(tmp_path, monkeypatch):
  """A build that lacks the newest entry points is refused for its version, before they are looked up."""
  (tmp_path / 'old.c').write_text('int dd_version(void) { return 7; }\nconst char* dd_last_error(void) { return ""; }\n')
  subprocess.run(['gcc', '-shared', '-fPIC', str(tmp_path / 'old.c'), '-o', str(tmp_path / 'old.so')], check=True)
  monkeypatch.setattr(hipops, '_LIB_PATH', tmp_path / 'old.so')
  monkeypatch.setattr(hipops, '_lib', None)
  with pytest.raises(RuntimeError, match='ABI version 7'):
    hipops.load_library()
