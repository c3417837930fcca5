"""Runs of rows in the paged-cache attention (csrc/paged.h), compiled for the
host: every visible key of every row lies in exactly one tile of its run, the
shares cover every tile of every run once, and cut units are joined from
exactly the pieces they were left in."""
import os
import subprocess

from conftest import ROOT

SOURCE = r"""
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>
#include "paged.h"

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

static int shares(std::mt19937 &rng, int rows, int span, int units, int longest, int ctas) {
    auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    iris_gpu_kv_cache_t c = {};
    c.kv_heads = units;
    c.num_seqs = pick(1, 4);
    c.page_size = pick(1, 40);
    c.max_blocks = longest / c.page_size + 1;
    std::vector<int32_t> seq(rows), pos(rows);
    const int stay = pick(0, 9);
    for (int t = 0; t < rows; t++) {
        seq[t] = t && pick(0, 9) < stay ? seq[t - 1] : pick(0, 9) == 0 ? (pick(0, 1) ? -1 : c.num_seqs + pick(0, 5))
                                                                       : pick(0, c.num_seqs - 1);
        pos[t] = pick(0, 9) == 0 ? -pick(1, 3) : pick(0, 19) == 0 ? 0x7FFFFFFF : pick(0, longest);
    }
    const int32_t *S = seq.data(), *P = pos.data();
    std::vector<int> n(rows), of(rows, -1);
    int64_t total = 0, tiles = 0;
    for (int t = 0; t < rows; t++) {
        int len = -1;
        const int count = iris_paged_run(&c, S, P, rows, span, t, &len);
        n[t] = iris_paged_run_places(&c, S, P, rows, span, t);
        CHECK(count >= 0 && count <= span && t + count <= rows && len >= 0);
        CHECK(n[t] == (len ? iris_paged_tiles(len) + IRIS_PAGED_EXTRA : 0));
        int most = 0;
        for (int r = t; r < t + count; r++) {
            CHECK(of[r] < 0 && seq[r] == seq[t] && r / span == t / span);
            of[r] = t;
            const int l = iris_paged_len(&c, pos[r]);
            most = l > most ? l : most;
        }
        CHECK(most == len);
        total += (int64_t)n[t] * units;
        tiles += (int64_t)(n[t] ? n[t] - IRIS_PAGED_EXTRA : 0) * units;
    }
    for (int t = 0; t < rows; t++) CHECK((of[t] >= 0) == (seq[t] >= 0 && seq[t] < c.num_seqs));
    const int64_t share = iris_paged_share(total, ctas);
    std::set<std::tuple<int, int, int>> done;
    std::map<std::pair<int, int>, std::set<int>> pieces, wanted;
    std::map<std::pair<int, int>, int> whole;
    for (int cta = 0; cta < ctas; cta++) {
        const int64_t start = cta * share;
        if (start >= total) continue;
        iris_paged_at_t at = {};
        at.rows = rows;
        at.span = span;
        int64_t before = 0;
        while (start >= before + (int64_t)n[at.t] * units) before += (int64_t)n[at.t++] * units;
        const int64_t mine = share < total - start ? share : total - start;
        if (!iris_paged_start(&at, start - before, mine, units, &c, S, P)) continue;
        if (const int later = iris_paged_join(&at, share)) {
            CHECK(cta > 0 && wanted.find({at.t, at.u}) == wanted.end());
            auto &w = wanted[{at.t, at.u}];
            w.insert(2 * cta - 1);
            for (int p = 0; p < later; p++) w.insert(2 * (cta + p));
        }
        bool fresh = true, begun = false;
        for (bool more = true; more;) {
            more = iris_paged_more(&at);
            CHECK(at.t < rows && of[at.t] == at.t && at.u < units && at.i < at.n && at.s == seq[at.t] && at.left > 0);
            int len;
            CHECK(at.count == iris_paged_run(&c, S, P, rows, span, at.t, &len) && at.len == len && at.count > 0);
            if (fresh) begun = at.i == 0, fresh = false;
            CHECK(done.insert({at.t, at.u, at.i}).second);
            const bool ends = at.i == at.n - 1;
            if (ends || !more) {
                if (ends && begun) whole[{at.t, at.u}]++;
                else CHECK((pieces[{at.t, at.u}].insert(2 * cta + (begun ? 1 : 0)).second));
                fresh = true;
            }
            if (more) iris_paged_next(&at, units, &c, S, P);
        }
    }
    CHECK((int64_t)done.size() == tiles);
    CHECK(pieces == wanted);
    for (int t = 0; t < rows; t++)
        for (int u = 0; n[t] && u < units; u++) CHECK(whole.count({t, u}) + pieces.count({t, u}) == 1);
    return 0;
}

int main() {
    std::mt19937 rng(2);
    auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    for (int j = 0; j < 500; j++)
        if (shares(rng, pick(1, 150), pick(1, 64), pick(1, 5), j % 3 ? pick(0, 3000) : pick(0, 90), pick(1, j % 2 ? 12 : 300)))
            return 1;
    // rows up to the end of int
    iris_gpu_kv_cache_t c = {};
    c.num_seqs = 1;
    c.page_size = 1 << 16;
    c.max_blocks = 1 << 16;
    const int32_t seq[3] = {0, 0, 0}, pos[3] = {-1, 0x7FFFFFFF, 5};
    int len = 0;
    CHECK(iris_paged_run(&c, seq, pos, 3, 64, 0, &len) == 3 && len == 0x7FFFFFFF);
    CHECK(iris_paged_run(&c, seq, pos, 3, 64, 1, &len) == 0 && len == 0);
    CHECK(iris_paged_run(&c, seq, pos, 3, 2, 2, &len) == 1 && len == 6);
    std::puts("ok");
    return 0;
}
"""


def test_shares_of_runs(tmp_path):
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    src, exe = tmp_path / "runs.cpp", tmp_path / "runs"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    f"-I{ROOT}/include", f"-I{ROOT}/iris.c_b200/csrc", f"-I{cuda}/include", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
