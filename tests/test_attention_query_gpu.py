"""A query of the runtime that fails once (shared-memory attribute, occupancy) fails
that call at most, with the runtime's message: the next call asks again.

The failure is made on the host, in a process of its own: a preloaded library
answers the nth call of one runtime function with an error and passes the
others on."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

FAKE = r"""
#define _GNU_SOURCE
#include <dlfcn.h>
#include <stdlib.h>
#include <string.h>
static int left(const char* name) {
  static int n = -1;
  const char* f = getenv("FAIL_FUNCTION");
  if (!f || strcmp(f, name)) return 0;
  if (n < 0) n = atoi(getenv("FAIL_CALL"));
  return n > 0 && --n == 0;
}
int cudaFuncSetAttribute(const void* f, int a, int v) {
  if (left("cudaFuncSetAttribute")) return 999; /* cudaErrorUnknown */
  return ((int (*)(const void*, int, int))dlsym(RTLD_NEXT, "cudaFuncSetAttribute"))(f, a, v);
}
int cudaOccupancyMaxActiveClusters(int* n, const void* f, const void* c) {
  if (left("cudaOccupancyMaxActiveClusters")) return 999;
  return ((int (*)(int*, const void*, const void*))dlsym(RTLD_NEXT, "cudaOccupancyMaxActiveClusters"))(n, f, c);
}
"""

CHILD = r"""
import sys
sys.path[:0] = [r"{root}/bonsai.cpp_b200", r"{root}/tests"]
import torch
import bonsai_b200 as bb
import test_lora_gpu as lora
import test_text_attention_gpu as attn
bb.init(0)

def paged():
    kc, vc, table = attn.make_cache(1, [3000, 70], 16, 2, 64, attn.f16)
    attn.run_paged(bb, attn.randn(2, 2, 8, 64), kc, vc, table, [0, 1, 2], [3000, 70], 16)

def prompt():
    attn.run_prompt(bb, *(attn.randn(i, 70, h, 128, dtype=attn.bf16) for i, h in enumerate((4, 2, 2))), [0, 70])

p = lora.Problem(bb, 256, 512, [16, 5])
def few():
    lora.check_f32(p, p.x(3), [0, 1, 2, 3], [0, 1, 0])
def many():
    lora.check_f32(p, p.x(300), [0, 200, 300], [0, 1])

call = dict(paged=paged, prompt=prompt, few=few, many=many)[sys.argv[1]]
failed = 0
for _ in range(3):
    try:
        call()
    except bb.BonsaiError as e:
        assert "unknown error" in str(e), e
        failed += 1
call()
assert failed <= 1, f"{{failed}} calls failed after one error"
print("failed calls:", failed)
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    d = tmp_path_factory.mktemp("fake")
    (d / "fake.c").write_text(FAKE)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(d / "fake.so"), str(d / "fake.c"), "-ldl"], check=True)
    return d / "fake.so"


OCCUPANCY, ATTRIBUTE = "cudaOccupancyMaxActiveClusters", "cudaFuncSetAttribute"


@pytest.mark.parametrize("call,function,nth", [("paged", OCCUPANCY, 1), ("paged", OCCUPANCY, 2), ("paged", ATTRIBUTE, 1),
                                               ("prompt", OCCUPANCY, 1), ("prompt", ATTRIBUTE, 2), ("few", OCCUPANCY, 1),
                                               ("few", ATTRIBUTE, 1), ("many", ATTRIBUTE, 1), ("many", ATTRIBUTE, 2)])
def test_one_failed_query_fails_one_call_at_most(gpu, fake, call, function, nth):
    env = dict(os.environ, LD_PRELOAD=str(fake), FAIL_FUNCTION=function, FAIL_CALL=str(nth))
    r = subprocess.run([sys.executable, "-c", CHILD.format(root=Path(__file__).resolve().parent.parent), call], env=env,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
