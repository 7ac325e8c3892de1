// How the attention of a chunk over a paged cache is dealt out to the CTAs of one wave (paged_chunk.cu, paged_chunk_tc.cu).
// Host and device; the lengths are known on the device only, so every CTA works out its own share.
//
// A sequence's new tokens go in tiles of `tile_tokens`, and a (sequence, KV head, tile) is an item: the rows of a tile are
// the query heads that share the KV head times the tokens.  An item costs the keys that its last row sees plus `fixed`
// (what a start and an end take, in keys); a caller may weigh the sequences' costs.  Items in the order sequence, KV head, tile lie one behind the other on
// a line of costs; CTA c of n owns the piece from total * c / n on.  A boundary inside an item falls between two tiles
// of `tile_keys` keys, or, nearer than `snap` tiles to an end of the item, on that end: both CTAs on either side compute the same.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define LUX_HD __host__ __device__ __forceinline__
#else
#define LUX_HD inline
#endif

namespace luxcuda {

struct ChunkShape {
    uint32_t heads;          // KV heads (or parts of them) per sequence
    uint32_t tile_tokens, tile_keys;
    uint32_t fixed, snap;
    uint32_t causal;
};

// Keys that the last row of tile t sees; `tokens` new ones of `keys` in all (fewer keys than tokens: the first rows see none).
LUX_HD uint32_t tile_sees(const ChunkShape& h, uint32_t tokens, uint32_t keys, uint32_t t) {
    if (!h.causal) return keys;
    const uint64_t end = (uint64_t)(t + 1) * h.tile_tokens;
    const int64_t sees = (int64_t)keys - (int64_t)tokens + (int64_t)(end < tokens ? end : tokens);
    return sees > 0 ? (uint32_t)sees : 0u;
}
LUX_HD uint32_t tiles_of(const ChunkShape& h, uint32_t tokens) { return tokens / h.tile_tokens + (tokens % h.tile_tokens != 0); }
// Cost of the first n tiles of a head, n <= tiles_of().  (U: 32 bits where no call of these sizes can cost more than they hold.)
template <typename U = uint64_t> LUX_HD U cost_before(const ChunkShape& h, uint32_t tokens, uint32_t keys, uint32_t n) {
    U cost = (U)n * h.fixed;
    if (!n) return 0;
    if (!h.causal) return cost + (U)n * keys;
    // the last tile apart (it may be short), the others rise by tile_tokens each from the first one that sees a key
    cost += tile_sees(h, tokens, keys, n - 1);
    const uint32_t full = n - 1;
    uint32_t blind = 0;
    if (tokens > keys) {
        const uint32_t b = (tokens - keys) / h.tile_tokens;
        blind = b < full ? b : full;
    }
    const U m = full - blind;
    if (m) {
        const U first = tile_sees(h, tokens, keys, blind);
        cost += m * first + (U)h.tile_tokens * (m * (m - 1) / 2);
    }
    return cost;
}
template <typename U = uint64_t> LUX_HD U sequence_cost(const ChunkShape& h, uint32_t tokens, uint32_t keys) {
    return (U)h.heads * cost_before<U>(h, tokens, keys, tiles_of(h, tokens));
}

// A place on the line: key tile `key_tile` of an item.
struct ChunkPlace {
    uint32_t seq, head, tile, key_tile;
};
LUX_HD bool same_item(const ChunkPlace& a, const ChunkPlace& b) { return a.seq == b.seq && a.head == b.head && a.tile == b.tile; }

// The place `rest` behind the beginning of sequence `seq` (rest < its cost); beyond the sequence: (seq + 1, 0, 0, 0).
template <typename U = uint64_t> LUX_HD ChunkPlace place_in(const ChunkShape& h, uint32_t seq, uint32_t tokens, uint32_t keys, U rest) {
    const uint32_t tiles = tiles_of(h, tokens);
    const U per_head = cost_before<U>(h, tokens, keys, tiles);
    uint32_t head = (uint32_t)(rest / per_head);
    rest -= head * per_head;
    uint32_t lo = 0, hi = tiles;                           // the last tile that begins at or before rest
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (cost_before<U>(h, tokens, keys, mid) <= rest) lo = mid;
        else hi = mid;
    }
    rest -= cost_before<U>(h, tokens, keys, lo);
    const uint32_t sees = tile_sees(h, tokens, keys, lo), key_tiles = sees / h.tile_keys + (sees % h.tile_keys != 0);
    const uint32_t key = rest < sees ? (uint32_t)rest : sees;
    uint32_t at = (uint32_t)(((U)key + h.tile_keys / 2) / h.tile_keys);
    if (at > key_tiles) at = key_tiles;
    bool over;                                             // the end of the item: the beginning of the next one
    if (!key_tiles) {
        over = rest > 0;
    } else if (key_tiles < 2 * h.snap) {                   // too short to be cut
        over = at * 2 >= key_tiles;
        at = 0;
    } else {
        if (at < h.snap) at = 0;
        over = key_tiles - at < h.snap || at == key_tiles;
    }
    if (over) {
        at = 0;
        if (++lo == tiles) {
            lo = 0;
            if (++head == h.heads) {
                head = 0;
                seq++;
            }
        }
    }
    return ChunkPlace{seq, head, lo, at};
}

}  // namespace luxcuda
