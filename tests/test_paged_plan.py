"""How a call of the attention over a paged cache is cut up, on the CPU: the runtime's rule, compiled as plain C++, against the parts
that batches of all kinds turn out to have."""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

COMMON = textwrap.dedent(r'''
    #include <cstdio>
    #include <cstring>
    #include <random>
    #include <vector>
    #include "kernels/zn_paged.h"
    #include "runtime/zn_paged_plan.h"
    #define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

    static ZnPagedArgs call(int64_t batch, int64_t kv_heads, int64_t group, int dim, int64_t tokens, int64_t max_q, int64_t cap, int causal) {
        ZnPagedArgs a;
        std::memset(&a, 0, sizeof(a));
        a.c.batch = (int32_t)batch;
        a.c.kv_heads = (int32_t)kv_heads;
        a.c.dim = dim;
        a.c.tokens = (int32_t)tokens;
        a.c.cap = (int32_t)cap;
        a.q_heads = (int32_t)(kv_heads * group);
        a.group = (int32_t)group;
        a.causal = causal;
        a.max_q = (int32_t)(max_q < tokens ? max_q : tokens);
        return a;
    }
''')

PROGRAM = COMMON + textwrap.dedent(r'''
    int main() {
        std::mt19937_64 rng(3);
        auto pick = [&](int64_t lo, int64_t hi) { return lo + (int64_t)(rng() % (uint64_t)(hi - lo + 1)); };
        int mixed = 0;
        for (int round = 0; round < 20000; ++round) {
            const int64_t batch = pick(1, rng() % 2 ? 8 : 600), kv = pick(1, 8), group = pick(1, rng() % 3 ? 8 : 40), pad = pick(0, 5);
            const int64_t most = pick(1, rng() % 2 ? 20 : 1500), cap = pick(0, 5000);
            const int dim = (int)pick(8, 128), type = (int)pick(0, 1);
            std::vector<int64_t> n(batch), kl(batch);
            int64_t tokens = pad, longest = 0;
            for (int64_t b = 0; b < batch; ++b) {
                n[b] = rng() % 3 ? pick(0, 2) : pick(0, most);
                kl[b] = std::min(cap, std::max(n[b], pick(0, cap)));
                tokens += n[b];
                longest = std::max(longest, n[b]);
            }
            const int64_t max_q = rng() % 2 ? longest : longest + pick(0, 50);
            if (tokens == 0 || max_q == 0) continue;
            ZnPagedArgs a = call(batch, kv, group, dim, tokens, max_q, cap, (int)pick(0, 1));
            const PagedPlan p = paged_plan(a, type, 256);
            CHECK(p.fits() && p.kernel >= 0 && p.kernel < kNumPaged);
            if (p.all_few) {
                CHECK(group * a.max_q <= kPagedRows[p.kernel] && a.few == group * a.max_q && a.few_splits >= 1);
                continue;
            }
            mixed += a.few > 0;
            CHECK(a.tile == kPagedRows[p.kernel] && a.tile_splits >= 1 && (int64_t)a.tile_splits * a.tile_len >= cap);
            // the parts of the tiles, as the kernel numbers them
            int64_t parts = 0;
            for (int64_t b = 0; b < batch; ++b) {
                const int64_t rows = std::min<int64_t>(n[b], a.max_q) * group;
                if (rows > a.few) parts += (rows + a.tile - 1) / a.tile * std::max<int64_t>(1, (kl[b] + a.tile_len - 1) / a.tile_len);
            }
            const int64_t few = a.few ? (int64_t)a.few_heads * a.few_splits : 0;
            CHECK(parts * kv + few <= p.wgs);
            // sequences of few rows have no tile
            CHECK(p.wgs - few <= (tokens * group / a.tile + tokens * group / (a.few + 1)) * kv * a.tile_splits);
        }
        CHECK(mixed > 1000);
        // as many sequences as a call takes, one of them with a chunk
        for (int64_t kv : {1, 2, 8, 64})
            for (int type : {0, 1})
                for (int dim : {8, 64, 128}) {
                    const int64_t batch = ((int64_t)1 << 22) / kv, tokens = batch + 499;
                    ZnPagedArgs a = call(batch, kv, 1, dim, tokens, 500, 512, 1);
                    CHECK(tokens < 1 << 24 && paged_plan(a, type, 256).fits());
                }
        std::printf("OK\n");
        return 0;
    }
''')


# Prints each kernel that calls of all kinds take, once.
TAKEN = COMMON + textwrap.dedent(r'''
    int main() {
        std::mt19937_64 rng(5);
        auto log = [&](double lo, double hi) {
            return (int64_t)std::llround(std::exp(std::log(lo) + (std::log(hi) - std::log(lo)) * (double)(rng() % 1000000) / 1e6));
        };
        bool seen[kNumPaged][2][4] = {};
        for (int round = 0; round < 200000; ++round) {
            const int64_t batch = log(1, 2000), kv = log(1, 16), group = log(1, 64), max_q = log(1, 8192), cap = log(1, 65536);
            const int64_t tokens = std::min<int64_t>((1 << 24) - 1, rng() % 2 ? batch * max_q : max_q + (batch - 1) * log(1, (double)max_q));
            if (tokens * kv * group > INT32_MAX / 2) continue;
            const int dim = (int)log(8, 128), type = (int)(rng() % 2);
            ZnPagedArgs a = call(batch, kv, group, dim, tokens, max_q, cap, (int)(rng() % 2));
            const PagedPlan p = paged_plan(a, type, 256);
            bool &s = seen[p.kernel][type][(dim - 1) / 32];
            if (!s) std::printf("%s_%s_%d\n", kPagedName[p.kernel], kCacheName[type], 32 * ((dim - 1) / 32 + 1));
            s = true;
        }
        return 0;
    }
''')


# The kernel of each call that is read: batch, kv_heads, group, dim, tokens, max_q, cap, causal, type.
NAMES = COMMON + textwrap.dedent(r'''
    int main() {
        long long batch, kv, group, dim, tokens, max_q, cap, causal, type;
        while (std::scanf("%lld %lld %lld %lld %lld %lld %lld %lld %lld", &batch, &kv, &group, &dim, &tokens, &max_q, &cap, &causal, &type) == 9) {
            ZnPagedArgs a = call(batch, kv, group, (int)dim, tokens, max_q, cap, (int)causal);
            const PagedPlan p = paged_plan(a, (int)type, 256);
            std::printf("%s_%s_%d\n", kPagedName[p.kernel], kCacheName[type], (int)(32 * ((dim - 1) / 32 + 1)));
        }
        return 0;
    }
''')


def run(tmp_path, program, *flags, given=""):
    src = tmp_path / "plan.cpp"
    src.write_text(program)
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-O1", "-std=c++17", *flags, "-I", os.path.join(ROOT, "zigneuron_amd", "csrc"), str(src), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], input=given, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def built():
    """The kernels of the code object."""
    with open(os.path.join(ROOT, "zigneuron_amd", "lib", "zn_attention_gfx950.hsaco"), "rb") as f:
        names = re.findall(rb"zn_paged_(?:few|few2|few4|tile|wide)_(?:f32|bf16)_\d+(?:_p)?(?=\.kd)", f.read())
    return {n.decode() for n in names}


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_workgroups_cover_the_parts_and_no_more_sequences_than_can_have_them(tmp_path):
    assert run(tmp_path, PROGRAM, "-fsanitize=undefined", "-fno-sanitize-recover=all").strip() == "OK"


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_every_kernel_that_is_built_is_taken(tmp_path):
    """... for pages of any size and of multiples of 16 positions alike, and none is taken that is not built."""
    taken = run(tmp_path, TAKEN).split()
    assert built() == {n + p for n in taken for p in ("", "_p")}


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_the_gpu_tests_reach_every_kernel(tmp_path):
    """tests/test_gpu_paged_kernels.py: each call is taken by the kernel that it names, and none is left out."""
    from paged_cases import cases
    calls, names = [], []
    for name, lens, counts, hq, hk, page, dim, dtype in cases():
        for causal in (0, 1):
            calls.append((len(lens), hk, hq // hk, dim, sum(counts) + 2, max(counts), max(lens), causal, int(dtype == "bf16")))
            names.append((name, "_p" if page % 16 == 0 else ""))
    got = run(tmp_path, NAMES, given="\n".join(" ".join(map(str, c)) for c in calls)).split()
    assert len(got) == len(calls)
    assert [n for n, _ in names] == [g + p for g, (_, p) in zip(got, names)]
    assert built() == {n for n, _ in names}
