"""How many rounds of runs an attention call over the paged cache takes: by what it reads and by its units, no GPU needed."""
import ctypes
import subprocess
from pathlib import Path

import pytest

SOURCES = Path(__file__).resolve().parent.parent / "nanokv_b200" / "csrc"
FITS, LEAST, MOST = 64 << 20, 64, 5
PROGRAM = """
#include "nkv_page_plan.h"
extern "C" int for_units(uint64_t bytes, uint32_t places, uint32_t units, int blocks, int least, int most) {
  return nkv::page::rounds_for(bytes, places, units, blocks, least, most);
}
extern "C" int by_bytes(uint64_t bytes, uint32_t places, int blocks, int least, int most) {
  return nkv::page::rounds_of(bytes, places, blocks, least, most);
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    folder = tmp_path_factory.mktemp("rounds")
    (folder / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{SOURCES}", "-o", str(folder / "plan.so"), str(folder / "plan.cpp")], check=True)
    lib = ctypes.CDLL(str(folder / "plan.so"))
    lib.for_units.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    lib.by_bytes.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    return lib


@pytest.mark.parametrize("batch,tokens,heads,length,kv_heads,rounds", [
    (1, 4680, 24, 20280, 24, 3), (1, 1560, 40, 98560, 8, 5), (1, 6000, 8, 60000, 8, 4), (1, 2048, 40, 16384, 40, 4), (4, 512, 32, 32256, 8, 5),
    (1, 1560, 24, 23400, 24, 3), (1, 4095, 32, 20000, 8, 2), (2, 1024, 24, 12288, 24, 2), (1, 600, 40, 30000, 40, 3), (8, 333, 16, 8167, 16, 1),
    (1, 300, 8, 100, 8, 1)])
def test_rounds_of_calls_whose_tokens_are_all_visible(plan, batch, tokens, heads, length, kv_heads, rounds):
    units = -(-tokens * (heads // kv_heads) // 256) * kv_heads * batch
    places = units * (-(-(length + tokens) // 128) + 5)
    assert plan.for_units(batch * (length + tokens) * 512 * kv_heads, places, units, 148, LEAST, MOST) == rounds


def test_rounds_stay_within_what_a_round_may_read_and_the_scratch(plan):
    import random
    rng = random.Random(1)
    for _ in range(5000):
        bytes_, places = int(2 ** rng.uniform(10, 36)), int(2 ** rng.uniform(0, 32)) - 1
        units, blocks, most = int(2 ** rng.uniform(0, 24)), rng.choice([1, 7, 148]), rng.randint(1, 8)
        got = plan.for_units(bytes_, places, units, blocks, LEAST, most)
        few, many = plan.by_bytes(bytes_ // 2, places, blocks, LEAST, most), plan.by_bytes(bytes_, places, blocks, LEAST, most)
        assert 1 <= few <= got <= many <= most
        assert many == 1 or places // blocks // many >= LEAST

        def away(r):
            return min(abs(r * blocks - units * k) for k in (max(1, r * blocks // units), r * blocks // units + 1))

        assert away(got) == min(away(r) for r in range(few, many + 1))
