"""CPU: the index arithmetic of a slot map (csrc/r3d_map_core.hpp) compiled for the host, every workgroup and thread of it in turn,
with arrays that refuse an index outside of them and a word that was never written."""
import os
import subprocess
import textwrap

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "pcl-augmentation_amd", "csrc")

DRIVER = textwrap.dedent("""
    #include "r3d_map_core.hpp"
    #include <cstdio>
    #include <cstdlib>
    #include <random>
    #include <vector>
    using namespace r3d;

    template <class T>
    struct Checked {      // an array whose words are written before they are read
      std::vector<T> v;
      std::vector<char> there;
      explicit Checked(size_t n = 0) : v(n), there(n, 0) {}
      void put(size_t i, T x) { v.at(i) = x; there.at(i) = 1; }
      explicit operator bool() const { return !v.empty(); }
      T operator[](int64_t i) const {
        if (i < 0 || i >= (int64_t)v.size() || !there[i]) { printf("read of word %lld of %zu\\n", (long long)i, v.size()); exit(3); }
        return v[i];
      }
    };
    struct Args {
      Checked<int64_t> offsets;
      Checked<int32_t> tables, rows;
      int64_t n_seq;
      int32_t block, most, shift;
    };

    // As k_map_slots: of `capacity` tokens.  past: tokens up to the last one are walked, whatever the capacity.
    void run(const std::vector<int> &lengths, int block, bool paged, bool picked, int64_t capacity, bool past) {
      const int n = (int)lengths.size();
      int most = 1;
      for (int l : lengths) most = std::max(most, (l + block - 1) / block);
      if (!paged) { for (int l : lengths) block = std::max(block, l); most = 1; }
      Args a{Checked<int64_t>(n + 1), Checked<int32_t>(paged ? (size_t)n * most : 0), Checked<int32_t>(picked ? n : 0), n, block, most,
             (block & (block - 1)) == 0 ? __builtin_ctz(block) : -1};
      // a table holds a word for every block of its row and no more
      std::vector<int> row(n);
      for (int i = 0; i < n; ++i) row[i] = picked ? n - 1 - i : i;
      int64_t total = 0;
      for (int i = 0; i < n; ++i) {
        a.offsets.put(i, total);
        if (picked) a.rows.put(i, row[i]);
        for (int b = 0; paged && b * block < lengths[i]; ++b) a.tables.put((size_t)row[i] * most + b, 7 * row[i] + b);
        total += lengths[i];
      }
      a.offsets.put(n, total);
      for (int64_t first = 0; first < capacity; first += kMapTokens) {
        const int64_t last = std::min(first + kMapTokens, capacity), stop = std::min(last, total);
        MapPart part{0, 0, false};
        Checked<int64_t> near(kMapLds + 1);
        if (first < stop) {
          part = map_part(a.offsets, a.n_seq, first, stop);
          if (part.near) for (int64_t i = 0; i <= part.hi - part.lo; ++i) near.put(i, a.offsets[part.lo + i]);
        }
        for (int thread = 0; thread < 256; ++thread) {
          int64_t slot[kMapAhead][2];
          int32_t seq[kMapAhead][2];
          const int64_t t0 = first + thread * 2;
          map_walk(a, near, part, t0, past ? total : stop, slot, seq);
          for (int u = 0; u < kMapAhead; ++u)
            for (int j = 0; j < 2; ++j) {
              const int64_t t = t0 + u * 512 + j;
              if (t >= last) continue;
              int64_t want = -1;
              int number = -1;
              if (t < total) {
                number = 0;
                while (a.offsets[number + 1] <= t) ++number;
                const int64_t p = t - a.offsets[number];
                want = (paged ? 7 * row[number] + p / block : row[number]) * (int64_t)block + p % block;
              }
              if (slot[u][j] != want || seq[u][j] != number) { printf("token %lld\\n", (long long)t); exit(4); }
            }
        }
      }
    }

    int main(int argc, char **argv) {
      const bool past = argc > 1;
      run(std::vector<int>(600, 10), 16, true, false, 2100, past);      // 2100 of 6000 tokens
      if (past) return 0;
      std::mt19937 rng(1);
      auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
      for (int turn = 0; turn < 250; ++turn) {
        std::vector<int> lengths(1 + upto(turn % 3 ? 900 : 40));
        const int longest = turn % 5 == 0 ? 5000 : turn % 2 ? 12 : 60;
        for (int &l : lengths) l = turn % 7 == 3 && upto(3) ? 0 : upto(longest);
        if (lengths.size() > 300) for (int &l : lengths) l = std::min(l, 200);
        int64_t total = 0;
        for (int l : lengths) total += l;
        const int block = turn % 4 == 0 ? 7 : turn % 4 == 1 ? 16 : turn % 4 == 2 ? 1 : 64;
        for (int64_t capacity : {total, total + 5, total - 3, total / 2 + 1, (int64_t)upto((int)total), total + 3000})
          if (capacity > 0) run(lengths, block, turn & 1, turn & 2, capacity, false);
      }
      puts("ok");
      return 0;
    }
""")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("slot_map")
    source, out = folder / "walk.cpp", folder / "walk"
    source.write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(source), "-o", str(out)], check=True, timeout=120)
    return str(out)


def test_every_index_of_a_slot_map_is_inside(program):
    run = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stdout


def test_the_check_sees_a_walk_beyond_the_capacity(program):
    run = subprocess.run([program, "past"], capture_output=True, text=True, timeout=120)
    assert run.returncode == 3 and "read of word" in run.stdout
