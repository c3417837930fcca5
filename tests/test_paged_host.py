"""Index arithmetic of the paged-cache attention (csrc/paged.h), compiled for the
host: shares cover every tile of every row once, cut units are joined from
exactly the pieces they were left in, and no table entry or page outside the
cache is ever used."""
import os
import subprocess

from conftest import ROOT

SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>
#include "paged.h"

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

static int shares(std::mt19937 &rng, int rows, int heads, int kv_heads, int longest, int ctas) {
    auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    iris_gpu_kv_cache_t c = {};
    c.kv_heads = kv_heads;
    c.num_seqs = rows + 2;
    c.page_size = pick(1, 40);
    c.max_blocks = longest / c.page_size + 1;
    std::vector<int32_t> seq(rows), pos(rows);
    for (int t = 0; t < rows; t++) {
        seq[t] = pick(0, 9) == 0 ? (pick(0, 1) ? -1 : c.num_seqs + pick(0, 5)) : pick(0, c.num_seqs - 1);
        pos[t] = pick(0, 9) == 0 ? -pick(1, 3) : pick(0, 9) == 0 ? 0x7FFFFFFF : pick(0, longest);
    }
    const int units = iris_paged_units(&c, heads);
    CHECK(units == kv_heads * (heads / kv_heads <= 16 ? 1 : (heads / kv_heads + 15) / 16));
    int64_t total = 0, tiles = 0;
    std::vector<int> n(rows);
    for (int t = 0; t < rows; t++) {
        n[t] = iris_paged_row_places(&c, seq.data(), pos.data(), t);
        const bool live = seq[t] >= 0 && seq[t] < c.num_seqs && pos[t] >= 0;
        CHECK((n[t] > 0) == live);
        const int real = n[t] ? n[t] - IRIS_PAGED_EXTRA : 0;
        CHECK(!live || (real > 0 && (int64_t)(real - 1) * IRIS_PAGED_TILE < (int64_t)c.max_blocks * c.page_size));
        total += (int64_t)n[t] * units;
        tiles += (int64_t)real * units;
    }
    const int64_t share = iris_paged_share(total, ctas);
    CHECK(share * ctas >= total && share == iris_paged_share32((uint32_t)total, ctas));
    std::set<std::tuple<int, int, int>> done;                 // row, unit, tile
    std::map<std::pair<int, int>, std::set<int>> pieces;      // unit -> slots left
    std::map<std::pair<int, int>, int> whole, joined;
    std::map<std::pair<int, int>, std::set<int>> wanted;
    for (int cta = 0; cta < ctas; cta++) {
        const int64_t start = cta * share;
        if (start >= total) continue;
        iris_paged_at_t at = {};
        int64_t before = 0;
        while (start >= before + (int64_t)n[at.t] * units) before += (int64_t)n[at.t++] * units;
        const int64_t mine = share < total - start ? share : total - start;
        if (!iris_paged_start(&at, start - before, mine, units, &c, seq.data(), pos.data())) continue;
        if (const int later = iris_paged_join(&at, share)) {
            CHECK(cta > 0);
            joined[{at.t, at.u}]++;
            auto &w = wanted[{at.t, at.u}];
            w.insert(2 * cta - 1);
            for (int p = 0; p < later; p++) w.insert(2 * (cta + p));
        }
        bool fresh = true, begun = false;
        for (bool more = true; more;) {
            more = iris_paged_more(&at);
            CHECK(at.t < rows && at.u < units && at.i < at.n && at.s == seq[at.t] && at.left > 0);
            if (fresh) begun = at.i == 0, fresh = false;
            CHECK(done.insert({at.t, at.u, at.i}).second);
            const bool ends = at.i == at.n - 1;
            if (ends || !more) {
                if (ends && begun) whole[{at.t, at.u}]++;
                else CHECK((pieces[{at.t, at.u}].insert(2 * cta + (begun ? 1 : 0)).second));
                fresh = true;
            }
            if (more) iris_paged_next(&at, units, &c, seq.data(), pos.data());
        }
    }
    CHECK((int64_t)done.size() == tiles);
    for (auto &p : pieces) {
        CHECK(whole.find(p.first) == whole.end());
        CHECK(joined[p.first] == 1);
        CHECK(wanted[p.first] == p.second);
        for (int slot : p.second) CHECK(slot >= 0 && slot < 2 * ctas);
    }
    CHECK(pieces.size() == wanted.size());
    int64_t begin = 0;
    for (int t = 0; t < rows; t++)
        for (int u = 0; n[t] && u < units; u++, begin += n[t]) {
            int border = 0;
            const int later = iris_paged_cut(begin, n[t] - IRIS_PAGED_EXTRA, share, &border);
            CHECK((later > 0) == (wanted.count({t, u}) > 0));
            if (!later) continue;
            std::set<int> slots = {2 * border - 1};
            for (int p = 0; p < later; p++) slots.insert(2 * (border + p));
            CHECK((wanted[{t, u}] == slots));
        }
    for (int t = 0; t < rows; t++)
        for (int u = 0; n[t] && u < units; u++) CHECK(whole.count({t, u}) + pieces.count({t, u}) == 1);
    return 0;
}

static int pages(std::mt19937 &rng) {
    auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    iris_gpu_kv_cache_t c = {};
    c.num_pages = pick(1, 50);
    c.page_size = pick(1, 70);
    c.num_seqs = pick(1, 4);
    c.max_blocks = pick(1, 9);
    c.table_stride = c.max_blocks + pick(0, 3);
    c.token_stride = 512;
    c.page_stride = 512 * (int64_t)c.page_size;
    std::vector<int32_t> table((size_t)c.num_seqs * c.table_stride, 1 << 30);   // the gaps between rows: no page
    std::vector<std::vector<int>> good(c.num_seqs, std::vector<int>(c.max_blocks));
    for (int s = 0; s < c.num_seqs; s++)
        for (int b = 0; b < c.max_blocks; b++) {
            const int kind = pick(0, 5);
            const int v = kind == 0 ? -pick(1, 1 << 30) : kind == 1 ? c.num_pages + pick(0, 1 << 30) : pick(0, c.num_pages - 1);
            table[s * c.table_stride + b] = v;
            good[s][b] = v >= 0 && v < c.num_pages ? v : -1;
        }
    c.table = table.data();
    const int64_t room = (int64_t)c.page_size * c.max_blocks;
    CHECK(iris_paged_len(&c, 0x7FFFFFFF) == room);
    CHECK(iris_paged_len(&c, -1) == 0 && iris_paged_len(&c, (int)0x80000000) == 0 && iris_paged_len(&c, 0) == 1);
    for (int j = 0; j < 400; j++) {
        const int s = pick(0, c.num_seqs - 1);
        const int p = j < 100 ? pick(0, (int)room + 200) : j == 100 ? 0x7FFFFFFF : pick(0, (int)room - 1);
        const int block = iris_paged_block(iris_paged_div(c.page_size), p), page = iris_paged_page(&c, s, block);
        CHECK(block == p / c.page_size);
        CHECK(page == (p < room ? good[s][p / c.page_size] : -1));
        if (page >= 0) {
            const int64_t o = iris_paged_offset(&c, page, p - block * c.page_size);
            CHECK(o >= 0 && o < c.num_pages * c.page_stride && o % 512 == 0);
            CHECK(o == page * c.page_stride + (p % c.page_size) * c.token_stride);
        }
    }
    return 0;
}

int main() {
    std::mt19937 rng(1);
    auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    for (int j = 0; j < 300; j++) {
        const int kv = pick(1, 5), heads = kv * pick(1, 20);
        if (shares(rng, pick(1, 40), heads, kv, j % 3 ? pick(0, 3000) : pick(0, 90), pick(1, j % 2 ? 12 : 300))) return 1;
        if (pages(rng)) return 1;
    }
    // a line of tiles past 32 bits, and positions at the end of int
    iris_gpu_kv_cache_t c = {};
    c.kv_heads = 1;
    c.num_seqs = 1;
    c.page_size = 1 << 16;
    c.max_blocks = 1 << 16;
    CHECK(iris_paged_len(&c, 0x7FFFFFFF) == 0x7FFFFFFF);
    CHECK(iris_paged_tiles(0x7FFFFFFF) == 33554432);
    CHECK(iris_paged_share((int64_t)33554432 * 4096, 296) * 296 >= (int64_t)33554432 * 4096);
    // blocks of every position, pages of any size
    for (int j = 0; j < 4000; j++) {
        const int ps = j < 600 ? j + 1 : j < 660 ? (1 << (j - 600) / 2) - 1 + j % 2 : pick(1, 0x7FFFFFFF);
        if (ps < 1) continue;
        const iris_paged_div_t d = iris_paged_div(ps);
        for (int i = 0; i < 60; i++) {
            const int64_t m = (int64_t)ps * pick(0, 0x7FFFFFFF / ps) + (i % 3 - 1);
            const int p = i == 0 ? 0x7FFFFFFF : i == 1 ? 0 : m < 0 || m > 0x7FFFFFFF ? pick(0, 0x7FFFFFFF) : (int)m;
            CHECK(iris_paged_block(d, p) == p / ps);
        }
    }
    std::puts("ok");
    return 0;
}
"""


def test_shares_and_pages(tmp_path):
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    src, exe = tmp_path / "paged.cpp", tmp_path / "paged"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    f"-I{ROOT}/include", f"-I{ROOT}/iris.c_b200/csrc", f"-I{cuda}/include", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
