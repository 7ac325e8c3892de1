"""How attention of a chunk over a paged cache is dealt out (webgpu_b200/csrc/paged_schedule.h), on the CPU: for batches of all kinds
the shares of the CTAs are the whole line of items, each key tile once, in order, and none is much longer than the mean."""
import pathlib
import subprocess

ROOT = pathlib.Path(__file__).resolve().parents[1]

PROGRAM = r"""
#include "webgpu_b200/csrc/paged_schedule.h"
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>
using namespace luxcuda;

static bool before(const ChunkPlace& a, const ChunkPlace& b) {
    if (a.seq != b.seq) return a.seq < b.seq;
    if (a.head != b.head) return a.head < b.head;
    if (a.tile != b.tile) return a.tile < b.tile;
    return a.key_tile < b.key_tile;
}

int main() {
    std::mt19937 rng(7);
    auto pick = [&](uint32_t lo, uint32_t hi) { return lo + rng() % (hi - lo + 1); };
    for (int n = 0; n < 4000; n++) {
        ChunkShape h{pick(1, 9), n % 5 == 0 ? 1u : pick(1, 130), n % 2 ? 64u : 128u, pick(1, 300), pick(1, 4), rng() % 4 ? 1u : 0u};
        const uint32_t seqs = pick(1, 6), grid = pick(1, 40);
        std::vector<uint32_t> tokens(seqs), keys(seqs);
        for (uint32_t s = 0; s < seqs; s++) {
            tokens[s] = rng() % 4 ? pick(0, 3) : pick(0, 700);
            keys[s] = rng() % 8 ? tokens[s] + pick(0, 2000) : pick(0, 300);       // contexts shorter than the chunk too
        }
        uint64_t total = 0;
        std::vector<uint64_t> cost(seqs);
        for (uint32_t s = 0; s < seqs; s++) {
            // the closed form against the sum
            uint64_t sum = 0;
            for (uint32_t t = 0; t < tiles_of(h, tokens[s]); t++) {
                if (cost_before(h, tokens[s], keys[s], t) != sum) return std::printf("cost of %u tiles: %u tokens, %u keys\n", t, tokens[s], keys[s]), 1;
                sum += h.fixed + tile_sees(h, tokens[s], keys[s], t);
            }
            cost[s] = sequence_cost(h, tokens[s], keys[s]);
            if (cost[s] != sum * h.heads) return std::printf("cost of a sequence\n"), 1;
            total += cost[s];
        }
        std::vector<ChunkPlace> place(grid + 1, ChunkPlace{seqs, 0, 0, 0});
        for (uint32_t c = 0; c <= grid; c++) {
            const uint64_t at = total / grid * c + total % grid * c / grid;
            uint64_t from = 0;
            for (uint32_t s = 0; s < seqs; from += cost[s++])
                if (at >= from && at - from < cost[s]) place[c] = place_in(h, s, tokens[s], keys[s], at - from);
        }
        // the walk of all CTAs one after the other goes through every item and every key tile once
        ChunkPlace want{0, 0, 0, 0};
        auto settle = [&] {
            while (want.seq < seqs && want.tile >= tiles_of(h, tokens[want.seq])) {
                want.tile = 0;
                if (tiles_of(h, tokens[want.seq]) == 0 || ++want.head == h.heads) want.head = 0, want.seq++;
            }
        };
        settle();
        uint64_t longest = 0;
        for (uint32_t c = 0; c < grid; c++) {
            uint64_t work = 0;
            if (before(place[c + 1], place[c])) return std::printf("boundaries out of order\n"), 1;
            while (want.seq < seqs && before(want, place[c + 1])) {
                const uint32_t sees = tile_sees(h, tokens[want.seq], keys[want.seq], want.tile), all = (sees + h.tile_keys - 1) / h.tile_keys;
                const uint32_t k1 = same_item(want, place[c + 1]) ? place[c + 1].key_tile : all;
                if (want.key_tile > all || k1 > all) return std::printf("a boundary behind its item\n"), 1;
                if (want.key_tile && all - want.key_tile < h.snap) return std::printf("too short an end\n"), 1;
                work += (uint64_t)(k1 - want.key_tile) * h.tile_keys + h.fixed;
                if (k1 < all) { want.key_tile = k1; break; }
                want.tile++;
                want.key_tile = 0;
                settle();
            }
            longest = std::max(longest, work);
        }
        if (want.seq < seqs) return std::printf("not all is dealt out\n"), 1;
        // a share passes the mean by what boundaries move: at most `snap` tiles (2 snap for short items) and half a tile on either side,
        // keys rounded up to tiles, and the fixed cost of a cut item
        if (n % 5 && longest > 0 && total) {
            const uint64_t slack = 2ull * (2 * h.snap + 2) * h.tile_keys + 2 * h.fixed;
            // an item's cost grows by less than a tile: the ratio is bounded by (fixed + tile) / fixed on items without many keys
            const uint64_t mean = total / grid + 1;
            const uint64_t most = mean + mean * h.tile_keys / (h.fixed + 1) + slack;
            if (longest > most) return std::printf("a share of %llu, mean %llu, bound %llu\n", (unsigned long long)longest, (unsigned long long)mean, (unsigned long long)most), 1;
        }
    }
    std::puts("ok");
    return 0;
}
"""


def test_shares_cover_every_key_tile_once(tmp_path):
    src = tmp_path / "schedule.cpp"
    src.write_text(PROGRAM)
    exe = tmp_path / "schedule"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", str(ROOT), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
