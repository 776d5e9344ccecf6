"""How the blocks of an append are dealt out: no two thread blocks of a launch may touch one store of 16-bit rows."""
import ctypes
import subprocess
from pathlib import Path

import pytest

SOURCES = Path(__file__).resolve().parent.parent / "nanokv_b200" / "csrc"
PROGRAM = """
#include "nkv_block_plan.h"
extern "C" int blocks(int length, int count) { return nkv::append_blocks(length, count); }
extern "C" int twice(int length, int count) { return nkv::append_twice(length, count); }
extern "C" int block(int length, int count, int x, int second) { return nkv::append_block(length, count, x, second != 0); }
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    folder = tmp_path_factory.mktemp("plan")
    (folder / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{SOURCES}", "-o", str(folder / "plan.so"),
                    str(folder / "plan.cpp")], check=True)
    return ctypes.CDLL(str(folder / "plan.so"))


def launches(plan, length, count, extra=3):
    """Blocks that each launch takes; ``extra``: thread blocks that a longer sequence of the batch brings along."""
    result = [[plan.block(length, count, x, 0) for x in range(plan.blocks(length, count) + extra)]]
    result.append([plan.block(length, count, x, 1) for x in range(1 + extra)])
    return [[b for b in blocks if b >= 0] for blocks in result]


def users(blocks, length, count):
    """Of one launch: blocks that read the store of 16-bit rows (to complete the block these belong to), and blocks that write
    it (they stay open)."""
    end = length + count
    return ([b for b in blocks if 64 * b < length and 64 * b + 64 <= end], [b for b in blocks if 64 * b + 64 > end])


@pytest.mark.parametrize("count", [1, 2, 31, 63, 64, 65, 100, 127, 128, 129, 200, 1560])
def test_every_block_is_taken_once_and_the_store_by_one_thread_block(plan, count):
    for length in range(0, 260):
        first, second = launches(plan, length, count)
        assert sorted(first + second) == list(range(length // 64, (length + count - 1) // 64 + 1))
        assert bool(second) == bool(plan.twice(length, count))
        for blocks in (first, second):
            reads, writes = users(blocks, length, count)
            assert len(set(reads + writes)) <= 1, (length, count)
        # what is read is read before anything is written there
        assert not users(second, length, count)[0]


def test_calls_without_tokens_take_nothing(plan):
    assert plan.blocks(100, 0) == 0 and not any(launches(plan, 100, 0))


def test_one_launch_for_all_blocks_would_share_the_store():
    """The check above finds what it is for: 152 tokens and 60 more, both blocks in one launch."""
    reads, writes = users([2, 3], 152, 60)
    assert reads == [2] and writes == [3]
