// kv_plan.h -- how kv_attention.cu spreads a call over the device: a function
// of the call's sizes and the number of SMs alone.
#pragma once

#include "common.h"

#include <algorithm>

namespace hbfb {

constexpr u32 kWarps = 4;
constexpr u32 kShare = 8;           // tiles of a share at least: two per warp
// Tiles of a segment that one CTA of so many warps may take whole, at most.  With two row tiles or
// more the sums of their weights cost CTAs on an SM: 400 segments of 125 tiles and 16 rows took 78
// us whole and 58 us split.
constexpr u32 whole_tiles(u32 nt, u32 warps) { return nt == 1 || warps > kWarps ? 128 : 32; }
// Few longer segments are finished by teams of up to 8 CTAs (a cluster) that join through
// distributed shared memory: from 64 tiles on, 16 to a CTA at least (38 tiles took 11.0 us by two
// CTAs and 9.7 us by one), as long as all teams are resident at once: clusters do not fill every
// processing cluster, so 7 of 8 SMs count.
constexpr u32 kTeamFrom = 64, kTeamTiles = 16;
constexpr u32 team_places(u32 sms) { return sms * 7 / 8; }

// Row tiles of 8 rows that a pass takes.  Wide passes widen the cache's values
// less often but leave fewer warps on an SM: 24 rows of 128 channels in one
// pass took 45 us where two passes of 16 took 49, 40 rows in three passes of
// 16 took 63 where two of 24 took 69 (8 sequences of 700 to 9001 tokens, 8
// heads).  At 256 channels the accumulators leave room for 16 rows.
constexpr u32 pass_width(u32 eights, u32 dim) { return eights <= 2 || (eights == 3 && dim < 256) ? eights : 2; }

// CTAs per SM, by registers and about 192 KB of rings.
constexpr u32 per_sm(u32 dim, u32 nt)
{
    return dim == 256 ? 2 : dim == 128 ? (nt == 3 ? 2 : 3) : (nt <= 2 ? 4 : 3);
}

// Tiles of each CTA of a team, whole blocks.
HD constexpr u32 part_of(u32 tiles, u32 team, u32 block_tiles)
{
    return (tiles + team * block_tiles - 1) / (team * block_tiles) * block_tiles;
}

// Sizes of a call; `group` query heads to a key/value head, lists of `top` blocks or none.
struct PlanCall {
    u32 seqs, tokens, heads, group, dim, block, width, top;
    bool lists, weights;
};

struct Plan {
    u32 nt, lists, rows, row_tiles, units, per_unit, workers, tiles, whole, warps, team;
    u64 segments, part_o, part_ml, part_ref, span, tile_sums, bytes;
};

// The form of a call on a device of `sms` SMs.
inline Plan plan_of(const PlanCall& c, u32 sms)
{
    Plan p{};
    p.lists = c.lists ? c.tokens : 1;
    p.rows = c.lists ? c.group : c.group * c.tokens;
    p.nt = pass_width((p.rows + 7) / 8, c.dim);
    const u32 R = 8 * p.nt;
    p.row_tiles = (p.rows + R - 1) / R;
    p.tiles = (c.lists ? c.top : c.width) * (c.block / 16);
    p.units = c.lists ? c.seqs * c.tokens * c.heads : c.seqs;
    p.per_unit = c.lists ? p.row_tiles : c.heads * p.row_tiles;
    p.segments = static_cast<u64>(p.units) * p.per_unit;
    // as many CTAs as are resident at once, fewer for little work
    const u64 most = (p.segments * p.tiles + kShare - 1) / kShare;
    const u64 resident = static_cast<u64>(per_sm(c.dim, p.nt)) * sms;
    p.workers = static_cast<u32>(std::max<u64>(1, std::min<u64>(most, resident)));
    // Short segments (by the table's width or the lists' length) are finished where they are
    // summed: one launch, where the even split takes two and joins.  With an SM for each, they get
    // CTAs of 8 warps: 64 of 38 tiles (128 channels) take 9.9 us, 12.4 us with 4 warps and 15.8 us
    // split.  Longer ones get teams of CTAs: 8 of 128 tiles take 10.0 us and 13.2 us split, 32 of
    // 256 tiles 14.4 and 22.0 us, 8 of 1024 tiles 20.0 and 21.4 us.  The more tiles a CTA has, the
    // more CTAs there have to be: 64 of 128 tiles take 17.7 us by one CTA each and 21.5 us split.
    p.warps = p.segments <= sms ? 2 * kWarps : kWarps;
    p.team = 1;  // CTAs of 4 warps take a segment each
    while (p.warps > kWarps && p.team < 8 && p.tiles >= kTeamFrom && p.segments * p.team * 2 <= team_places(sms) &&
           p.tiles >= p.team * 2 * kTeamTiles)
        p.team *= 2;
    const u32 each = part_of(p.tiles, p.team, c.block / 16);
    // With 4 warps: 400 of 128 tiles take 36.6 us whole and 41.2 us split.  More long ones than are
    // resident at once should fill their last turn: 1600 lists of 128 tiles take 152 and 169 us,
    // 512 on 444 places 74 and 64 us (512 of 21 to 63 tiles 32.0 and 36.7 us).
    const u64 places = (p.segments + resident - 1) / resident * resident;
    p.whole = each <= whole_tiles(p.nt, p.warps) &&
              (p.segments <= sms ? each <= p.segments * p.team + 64 : 2 * p.tiles <= p.segments + 64) &&
              (p.tiles <= 64 || p.segments <= resident || p.segments * 5 >= places * 4) &&
              (!c.weights || p.lists * p.row_tiles == 1);
    if (p.whole) {
        p.workers = static_cast<u32>(p.segments) * p.team;
        return p;  // no workspace
    }
    u64 at = 0;
    auto take = [&](u64 bytes) {
        const u64 here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.part_o = take((p.segments + p.workers) * R * c.dim * 4);
    p.part_ml = take((p.segments + p.workers) * R * 8);
    p.part_ref = take((p.segments + p.workers) * R * 4);
    p.span = take(p.segments * 8);
    p.tile_sums = take(c.weights ? p.segments * p.tiles * R * 8 : 0);
    p.bytes = at;
    return p;
}

}  // namespace hbfb
