// How the norm and rotation kernels (fpt_qk_rope.cu) cut their tokens into tiles and share tiles out over blocks: plain host
// arithmetic on sizes, so that it can be checked without a device.
#pragma once
#include <algorithm>
#include <cstdint>

namespace fpt {

constexpr uint32_t kMaxTileTokens = 32;
constexpr uint32_t kBwdTrig = 512;      // tokens x pairs of a tile of the backward pass (two entries a thread, two tiles)

// Tokens of a tile, a power of two: every group gets at least `rounds` heads of its token.  Measured for the forward pass (2 x 4096
// tokens of 32 + 8 heads x 128 and 15840 such tokens, us at 2, 4, 8 heads): with the norm 37.3, 29.0, 29.6; rotation alone 55.9,
// 50.0, 51.2.
inline uint32_t tile_tokens(uint32_t groups, uint32_t heads, uint32_t pairs, uint32_t rounds, uint32_t trig) {
    uint32_t t = 1;
    while (2 * t <= std::min(kMaxTileTokens, groups) && 2 * t * pairs <= trig && t * heads < rounds * groups) t *= 2;
    return t;
}

struct BwdShare {                       // queries or keys in the backward pass
    uint32_t blocks, tiles, tile_tokens;
};

// Tiles of the backward pass and its blocks, `total` at most (as many as are resident with 16-bit data, and as many as the
// workspace has rows for), shared out between queries and keys.  A tile takes as many steps as its groups have heads, and
// kTileCost more (sines, addresses, a barrier); the shares are those for which the side that takes longest, in whole rounds of tiles, is done first.
// Measured against shares by heads alone (a tile's own cost as one head): 2 x 4096 tokens of 32 + 8 heads of 128 the backward pass
// 55 us and 46, 3063 tokens of 12 + 4 heads of 64 with the forward pass 17.0 and 15.5, 8192 tokens of 8 + 1 heads of 256 53 and
// 35, of 40 + 8 heads of 80 58 and 62.  The constant: 0.5 .. 3 differ by less than that.
// reach(side, tokens): whether that side's tiles of so many tokens can be addressed.
constexpr float kTileCost = 1.5f;
template <class Reach>
void share_blocks(BwdShare& q, uint32_t q_heads, BwdShare& k, uint32_t k_heads, uint32_t tokens, uint32_t groups, uint32_t pairs,
                  uint32_t total, Reach&& reach) {
    BwdShare* const sides[2] = {&q, &k};
    const uint32_t heads[2] = {q_heads, k_heads};
    float cost[2] = {0.0f, 0.0f};       // of a token
    for (int s = 0; s < 2; ++s) {
        *sides[s] = BwdShare{0, 0, 1};
        if (!heads[s]) continue;
        sides[s]->tile_tokens = tile_tokens(groups, heads[s], pairs, 8, kBwdTrig);
        cost[s] = float(heads[s]) + kTileCost * float(groups) / float(sides[s]->tile_tokens);
    }
    for (int s = 0; s < 2; ++s) {
        BwdShare& d = *sides[s];
        if (!heads[s]) continue;
        // no more tokens a tile than keep every block busy
        const float blocks = float(total) * cost[s] / (cost[0] + cost[1]);
        while (d.tile_tokens > 1 && float(tokens / d.tile_tokens) < blocks) d.tile_tokens /= 2;
        if (!reach(s, d.tile_tokens)) d.tile_tokens = 1u;
        d.tiles = (tokens + d.tile_tokens - 1) / d.tile_tokens;
        d.blocks = std::min(total, d.tiles);
    }
    if (!q_heads || !k_heads) return;
    q.blocks = std::min(total - 1, q.tiles);        // where nothing below fits: so many query tiles that the keys' share is under a block
    k.blocks = std::min(total - q.blocks, k.tiles);
    const auto steps = [&](int s) {
        const uint32_t step = groups / sides[s]->tile_tokens;
        return float((heads[s] + step - 1) / step) + kTileCost;
    };
    const float q_tile = steps(0), k_tile = steps(1);
    const float even = (float(q.tiles) * q_tile + float(k.tiles) * k_tile) / float(total);      // time with nothing left over
    const uint32_t most = std::max(1u, uint32_t(std::min(even / q_tile, float(q.tiles))));
    float least = 1e30f;
    for (uint32_t rounds = most > 2 ? most - 2 : 1; rounds < most + 6; ++rounds) {
        const uint32_t blocks = (q.tiles + rounds - 1) / rounds;
        if (blocks >= total) continue;
        const float time = std::max(float(rounds) * q_tile, float((k.tiles + total - blocks - 1) / (total - blocks)) * k_tile);
        if (time < least) {
            least = time;
            q.blocks = blocks;
            k.blocks = std::min(total - blocks, k.tiles);
        }
    }
}

}  // namespace fpt
