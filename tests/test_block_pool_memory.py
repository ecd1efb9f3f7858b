"""fork and compact without host memory: whichever allocation of the call fails, nothing has changed."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from cf_hip import _abi

SOURCE = r"""
#include <dlfcn.h>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <new>
#include <string>
#include <vector>

#include "cf_hip.h"

// the armed-th allocation from now on fails
static long armed = -1;
void* operator new(std::size_t n) {
  if (armed >= 0 && armed-- == 0) throw std::bad_alloc();
  if (void* p = std::malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

#define CALL(name) ((decltype(&name))dlsym(lib, #name))
static void* lib;

struct State {
  int64_t free_blocks;
  std::vector<int64_t> rc;
  std::vector<std::vector<int32_t>> tables;
  bool operator==(const State& o) const { return free_blocks == o.free_blocks && rc == o.rc && tables == o.tables; }
};

static const char* kIds[] = {"a", "b", "c", "child with a name that no short string holds 1",
                             "child with a name that no short string holds 2", "child 3"};

static State state(void* pool) {
  State s;
  CALL(cf_bp_num_free)(pool, &s.free_blocks);
  for (int64_t b = 0; b < 64; ++b) {
    int64_t rc = 0;
    CALL(cf_bp_ref_count)(pool, b, &rc);
    s.rc.push_back(rc);
  }
  for (const char* id : kIds) {
    int32_t ids[64];
    int64_t n = -1;
    if (CALL(cf_bp_get_blocks)(pool, id, ids, 64, &n) != CF_OK) n = 0;
    s.tables.emplace_back(ids, ids + n);
  }
  return s;
}

int main(int argc, char** argv) {
  lib = dlopen(argv[1], RTLD_NOW);
  if (!lib) return std::printf("%s\n", dlerror()), 2;
  for (const int rows : {0, 16}) {
    void* pool = nullptr;
    CALL(cf_bp_create)(64, 16, &pool);
    if (rows) CALL(cf_bp_bind_rows)(pool, rows, 64);
    int32_t ids[64], copies[16], moves[128];
    int64_t n = 0;
    CALL(cf_bp_allocate)(pool, "a", 100, ids, 64, &n);
    CALL(cf_bp_allocate)(pool, "b", 200, ids, 64, &n);
    CALL(cf_bp_allocate)(pool, "c", 50, ids, 64, &n);
    CALL(cf_bp_free)(pool, "b");
    for (const bool fork : {true, false}) {
      const State before = state(pool);
      int failures = 0, rc = -1;
      for (long at = 0; at < 1000 && rc != CF_OK; ++at) {
        armed = at;
        rc = fork ? CALL(cf_bp_fork)(pool, "a", 3, kIds + 3, 90, copies, 8, &n) : CALL(cf_bp_compact)(pool, moves, 64, &n);
        armed = -1;
        if (rc == CF_OK) break;
        ++failures;
        if (!(state(pool) == before)) return std::printf("%s: changed by failure %ld, rows %d\n", fork ? "fork" : "compact", at, rows), 1;
      }
      const State after = state(pool);
      if (rc != CF_OK || after == before || failures < 5) return std::printf("rc %d, %d failures\n", rc, failures), 1;
      if (fork) {
        for (int i = 3; i < 6; ++i) {
          if (after.tables[i].size() != 6 || after.tables[i][4] != after.tables[0][4] || after.tables[i][5] == after.tables[0][5] ||
              copies[2 * (i - 3)] != after.tables[0][5] || copies[2 * (i - 3) + 1] != after.tables[i][5])
            return std::printf("child %d\n", i), 1;
        }
        if (n != 3 || after.free_blocks != before.free_blocks - 3) return 1;
      }
      std::printf("rows %d, %s: %d failures\n", rows, fork ? "fork" : "compact", failures);
    }
    CALL(cf_bp_destroy)(pool);
  }
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_fork_and_compact_change_nothing_without_memory(tmp_path):
    (tmp_path / "pool.cpp").write_text(SOURCE)
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["g++", "-std=c++17", "-O1", "-rdynamic", f"-I{include}", str(tmp_path / "pool.cpp"), "-o",
                    str(tmp_path / "pool"), "-ldl"], check=True)
    run = subprocess.run([str(tmp_path / "pool"), str(_abi._lib_path())], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout + run.stderr
