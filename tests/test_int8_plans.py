"""How 8-bit products are cut (csrc/int8_linear.hip): every kernel variant that a call of ordinary
sizes can reach is run by a listed product of tests/test_gpu_int8_plans.py.  The rule is host code;
its text is compiled here with a C++ compiler and asked."""

import os
import shutil
import subprocess

import pytest

from test_dma_waits import CSRC
from test_gpu_int8_plans import PRODUCTS

HARNESS = r"""
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
constexpr int kStep = 128;
%s
void print(const Plan& p, int64_t M, int64_t K) {
  if (p.kind == Plan::kShort) {
    puts("short");
  } else if (p.kind == Plan::kFew) {
    // the steps of the wave that has most, up to one more than the rings' four
    const int steps = (int)((K + 4 * kStep - 1) / (4 * kStep));
    printf("few cols %%d rows %%d dma %%d steps %%d cut %%d\n", (int)p.cols,
           M <= 16 ? 16 : M <= 32 ? 32 : 64, p.dma, std::min(steps, 5), K %% kStep != 0);
  } else {
    // the fewest steps of a part, up to one more than the rings' four, and whether K ends in one
    const int64_t k = p.padded ? p.padded : K;
    const int steps = (int)((k + kStep - 1) / kStep / p.parts);
    printf("tile %%dx%%d %%d dma %%d parts %%d copies %%d", kShapes[p.shape].tm, kShapes[p.shape].tn,
           kShapes[p.shape].room, p.dma, p.parts > 1, p.padded > 0);
    printf(" steps %%d cut %%d\n", std::min(steps, 5), k %% kStep != 0);
  }
}
int main(int argc, char** argv) {
  for (int i = 1; i + 3 < argc; i += 4)
    print(plan_of(atoll(argv[i]), atoll(argv[i + 1]), atoll(argv[i + 2]), atoi(argv[i + 3])),
          atoll(argv[i]), atoll(argv[i + 2]));
  if (argc > 1) return 0;
  uint64_t state = 1;
  auto random = [&] {
    state = state * 6364136223846793005u + 1442695040888963407u;
    return (double)(state >> 11) * 0x1p-53;
  };
  auto size = [&](double lo, double hi) { return (int64_t)(lo * pow(hi / lo, random())); };
  for (int i = 0; i < 1000000; ++i) {
    const int64_t M = size(1, 40000), N = size(1, 40000);
    int64_t K = size(16, 20000);
    if (random() < 0.5) K = K / 16 * 16;
    const bool aligned = K %% 16 == 0 && K >= kStep && random() < 0.5;
    print(plan_of(M, N, K, aligned), M, K);
  }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    with open(os.path.join(CSRC, "int8_linear.hip")) as f:
        text = f.read()
    rule = text[text.index("struct Shape {"):text.index("bool aligned_rows(")]
    assert "constexpr int kStep = 128;" in text
    folder = tmp_path_factory.mktemp("plans")
    source, program = folder / "plans.cpp", folder / "plans"
    source.write_text(HARNESS % rule)
    subprocess.run([cxx, "-O2", "-std=c++20", "-o", str(program), str(source)], check=True)

    def run(*args):
        out = subprocess.run([str(program), *map(str, args)], check=True, capture_output=True,
                             text=True)
        return out.stdout.splitlines()

    return run


def test_every_variant_is_among_the_listed_products(ask):
    listed = ask(*(int(a) for p in PRODUCTS for a in p))
    assert len(listed) == len(PRODUCTS)
    reached = set(ask())
    assert len(reached) > 40
    missing = sorted(reached - set(listed))
    assert not missing, missing


def test_listed_products_are_ragged(ask):
    """Tiles that the rows and the columns end inside, but for a few products of whole tiles."""

    lines = ask(*(int(a) for p in PRODUCTS for a in p))
    whole = 0
    for (M, N, _, _), line in zip(PRODUCTS, lines):
        if line.startswith("tile"):
            tm, tn = map(int, line.split()[1].split("x"))
            whole += M % tm == 0 or N % tn == 0
    assert whole <= 4
