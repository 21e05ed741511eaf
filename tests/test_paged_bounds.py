"""What the device arrays of a paged cache can lead to, on the CPU: the part of
the kernels that turns them into addresses, compiled as plain C++ and run with
arrays full of anything."""
from __future__ import annotations

import os
import shutil
import subprocess
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = textwrap.dedent(r'''
    #include <cstdio>
    #include <cstdlib>
    #include <random>
    #include <vector>
    #include "zn_paged.h"
    // as the runtime's: x / d for 0 <= x < 2^31
    static void divisor(uint32_t d, uint32_t &mul, uint32_t &shift) {
        uint32_t l = 0;
        while ((1ull << l) < d) ++l;
        mul = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
        shift = l;
    }
    #define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
    int main() {
        std::mt19937_64 rng(11);
        auto pick = [&](int64_t lo, int64_t hi) { return lo + (int64_t)(rng() % (uint64_t)(hi - lo + 1)); };
        const int wild[] = {0, 1, -1, 2147483647, -2147483647 - 1, 5, 1 << 30, -(1 << 30)};
        for (int round = 0; round < 20000; ++round) {
            ZnPagedCache c = {};
            c.batch = (int)pick(1, 5);
            c.pages = (int)pick(0, 7);
            c.page_size = (int)pick(1, 300);
            c.max_pages = (int)pick(1, 6);
            c.kv_heads = (int)pick(1, 4);
            c.dim = (int)pick(1, 128);
            c.tokens = (int)pick(0, 50);
            c.cap = c.pages ? (int)pick(0, (int64_t)c.max_pages * c.page_size) : 0;
            c.stride[2] = c.dim + pick(0, 4);
            c.stride[1] = c.stride[2] * c.page_size;
            c.stride[0] = c.stride[1] * c.kv_heads;
            const int64_t size = c.pages * c.stride[0];
            divisor((uint32_t)c.page_size, c.div_mul, c.div_shift);
            std::vector<int32_t> table((size_t)c.batch * c.max_pages), lens(c.batch), starts(c.batch + 1);
            for (auto *v : {&table, &lens, &starts})
                for (auto &x : *v) x = rng() % 3 ? (int32_t)pick(-2, 60) : wild[rng() % 8];
            c.table = table.data();
            c.kv_lens = lens.data();
            c.starts = starts.data();
            for (int b = 0; b < c.batch; ++b) {
                const PagedSeq s(c, b);
                CHECK(s.t0 >= 0 && s.ql >= 0 && s.t0 + s.ql <= c.tokens);
                CHECK(s.kl >= 0 && s.kl <= c.cap && s.first == s.kl - s.ql);
                for (int j = 0; j < s.kl; ++j) {
                    const int page = table[(size_t)b * c.max_pages + j / c.page_size];
                    const bool in = page >= 0 && page < c.pages;
                    for (int kh = 0; kh < c.kv_heads; kh += 3) {
                        const int64_t at = paged_at(c, b, kh, j);
                        CHECK((at >= 0) == in);
                        if (in) CHECK(at == page * c.stride[0] + kh * c.stride[1] + j % c.page_size * c.stride[2] && at + c.dim <= size);
                    }
                }
            }
        }
        // far: the largest page numbers, positions and strides that a call takes
        ZnPagedCache c = {};
        const int32_t table[1] = {(1 << 30) - 2};
        c.batch = c.max_pages = c.kv_heads = 1;
        c.pages = (1 << 30) - 1;
        c.page_size = (1 << 30) - 1;
        c.stride[0] = (int64_t)1 << 16;
        c.stride[2] = 128;
        c.table = table;
        divisor((uint32_t)c.page_size, c.div_mul, c.div_shift);
        CHECK(paged_at(c, 0, 0, (1 << 30) - 2) == ((int64_t)((1 << 30) - 2) << 16) + (int64_t)((1 << 30) - 2) * 128);
        std::printf("OK\n");
        return 0;
    }
''')


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_addresses_stay_inside(tmp_path):
    src = tmp_path / "bounds.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "bounds"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "zigneuron_amd", "csrc", "kernels"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr
