/*
 * How the attention over the 4-bit cache is launched (cache4_attend_impl.h), and the room that its parts take. Plain host code without a HIP header: the
 * tests look at batches that no device memory holds.
 */
#ifndef KMX_CACHE4_PLAN_H
#define KMX_CACHE4_PLAN_H

#include <cstddef>
#include <cstdint>

namespace kmx {

constexpr uint32_t MOST_PARTS = 128;    /* of the tokens of a row */
constexpr uint32_t TICKETS = 8192;      /* units (sequence, head, tile of rows) of a call that takes its tokens in parts */
constexpr uint64_t MOST_UNITS = 1 << 23; /* of a call */
constexpr uint32_t MANY_ROWS = 64;      /* rows of a head: above it 256 a work-group (2 sequences of up to 16384 tokens, 8 heads, 64 rows: 39 us by 16, 41 by 256; 128 rows: 62 and 44) */
constexpr uint32_t MANY_LEAST = 4, MANY_COST = 8; /* tiles of a part at least; tiles that a part costs beside its own (2, 4, 8: 128.7, 128.4, 123.6 us for 54 units of 178 tiles) */
constexpr uint32_t SHARE_LEAST = 64;    /* tiles for each work-group of a call divided in shares (16 tiles: 57 us in parts, 62 in shares; 128 and more: see plan_attend4) */
/* rounds of work-groups, as many as the chip holds at a time, that many rows in parts are launched as at most: what each leaves to be joined is 133 KB at 128
 * channels, 270 MB of them, 540 MB at 256 (1056 queries, 64 heads on 8 of 128, 131072 tokens: 5.69 ms in 7 parts, 5.51 in 16, which take 0.6 GB; of 256
 * channels 14.36 and 13.96, 1.1 GB) */
constexpr uint32_t MANY_ROUNDS = 8;

struct Shape4 {
	uint32_t J, heads, group; /* 32 J channels; heads of the cache, query heads of each */
	uint32_t sequences, max_queries, max_length, page_shift, top, compute_units;
};

/* launch shape: units (sequence, head, tile of rows), tiles of 16 or (many) 256 rows, parts of the tokens, tiles of 64 tokens a part. many: splits is the
 * number of work-groups; tiles_per_split 0: shares. joined: parts are left to the kernel that joins them */
struct Plan4 { uint64_t units; uint32_t row_tiles, splits, tiles_per_split; bool many, joined; };

constexpr size_t part_floats(uint32_t J, bool many) { return (many ? 256 : 16) * (32 * (size_t)J + 2); } /* sums, maximum and sum of probabilities of each row */

/*
 * Tiles of 16 rows, or of 256 where there are many, and how many parts the tokens are taken in.
 * 16 rows: two work-groups a compute unit in all, none below one tile a wavefront (64 sequences of 8192 tokens, 8 heads: 124 us in one part, 133 in
 * four; one sequence of 131072: 32 us with one work-group a unit, 28.7 with two, 29.4 with four).
 * 256 rows: lengths are known on the device only. Several sequences whose lengths may differ by much are divided in equal shares there, one for each
 * work-group that the chip holds (2 x 1024 queries over 16384 and fewer tokens, 8 heads: of 128 channels 568 -> 521 us, 64: 375 -> 325, 256: 1598 ->
 * 1475; 5 x 700 over up to 9000: 505 -> 463; but equal lengths 588 -> 622). Not one sequence (323 -> 347), nor where units are many and fill the chip
 * as they come (1024 units: 477 -> 534), nor short ones: there as many parts as make the rounds of work-groups short, at most MANY_ROUNDS of them.
 */
inline Plan4 plan_attend4(const Shape4& s)
{
	Plan4 plan{};
	const uint64_t rows = (uint64_t)s.max_queries * s.group;
	plan.many = !s.top && rows > MANY_ROWS;
	const uint64_t row_tiles = s.top ? s.max_queries * (((uint64_t)s.group + 15) / 16) : plan.many ? (rows + 255) / 256 : (rows + 15) / 16;
	const uint64_t entries = s.sequences * row_tiles, units = row_tiles >= MOST_UNITS || entries >= MOST_UNITS ? MOST_UNITS : entries * s.heads;
	plan.units = units;
	plan.row_tiles = (uint32_t)row_tiles;
	plan.splits = 1;
	if (units >= MOST_UNITS) return plan; /* (refused) */
	/* of a list no more pages are looked at than a sequence has (tiles_of) */
	const uint64_t pages = ((uint64_t)s.max_length + (1u << s.page_shift) - 1) >> s.page_shift, tokens = s.top ? (s.top < pages ? s.top : pages) << s.page_shift : s.max_length;
	const uint32_t tiles = (uint32_t)((tokens + 63) / 64);
	if (plan.many) {
		const uint64_t slots = (s.J <= 2 ? 2 : 1) * (uint64_t)s.compute_units; /* work-groups on the chip at a time */
		if (s.sequences > 1 && units <= 2 * slots && units * tiles >= SHARE_LEAST * slots && rows <= 0x7FFFFF00u && units * tiles <= 0x7FFFFFFFu) {
			plan.splits = (uint32_t)slots;
			plan.joined = true;
			return plan;
		}
		uint64_t best = ~0ull, parts = 1;
		for (uint64_t p = 1; p <= 16 && (p == 1 || (p * MANY_LEAST <= tiles && units * p <= MANY_ROUNDS * slots)); ++p) {
			const uint64_t time = (units * p + slots - 1) / slots * ((tiles + p - 1) / p + MANY_COST);
			if (time < best) { best = time; parts = p; }
		}
		plan.tiles_per_split = tiles ? (uint32_t)((tiles + parts - 1) / parts) : 1;
		plan.splits = (uint32_t)(units * parts);
		plan.joined = parts > 1;
		return plan;
	}
	uint64_t parts = (2 * (uint64_t)s.compute_units + units - 1) / (units ? units : 1);
	if (parts > (tiles + 3) / 4) parts = (tiles + 3) / 4;
	if (parts > MOST_PARTS) parts = MOST_PARTS;
	if (parts == 0 || units > TICKETS) parts = 1;
	plan.tiles_per_split = tiles ? (uint32_t)(((tiles + parts - 1) / parts + 3) / 4 * 4) : 4; /* a tile for each wavefront */
	plan.splits = tiles ? (tiles + plan.tiles_per_split - 1) / plan.tiles_per_split : 1;
	return plan;
}

/* slots of the parts of many rows: one a work-group, of shares two (the end of one unit and the begin of another) */
inline size_t many_slots(const Plan4& plan) { return plan.tiles_per_split ? plan.splits : 2 * (size_t)plan.splits; }

/* floats of work space: slots and two words a unit, or the parts of all units */
inline size_t plan_floats(const Plan4& plan, uint32_t J)
{
	if (plan.units >= MOST_UNITS) return 0;
	if (plan.many) return plan.joined ? many_slots(plan) * part_floats(J, true) + 2 * plan.units : 0;
	return plan.splits > 1 ? plan.units * plan.splits * part_floats(J, false) : 0;
}

/*
 * The most that this takes for any batch that is no larger: fewer units are taken in more parts. Of few rows units with parts are fewer than 2 compute_units, and
 * there are at most 2 compute_units / units + 1 parts of each; of many rows MANY_ROUNDS rounds of parts, or shares, one for each work-group that the chip holds.
 */
inline size_t most_floats(const Shape4& s)
{
	constexpr uint64_t PLENTY = (uint64_t)1 << 40;
	const auto times = [](uint64_t a, uint64_t b) { return a == 0 || b == 0 ? 0 : a > PLENTY / b ? PLENTY : a * b; };
	const auto least = [](uint64_t a, uint64_t b) { return a < b ? a : b; };
	const uint64_t pages = ((uint64_t)s.max_length + (1u << s.page_shift) - 1) >> s.page_shift;
	const uint64_t tiles = ((pages << s.page_shift) + 63) / 64; /* (of lists, whose last page counts as a whole) */
	const uint64_t rows = (uint64_t)s.max_queries * s.group, heads = times(s.sequences, s.heads), slots = (s.J <= 2 ? 2 : 1) * (uint64_t)s.compute_units;
	const uint64_t listed = s.top ? times(s.max_queries, ((uint64_t)s.group + 15) / 16) : 0, few = (least(rows, MANY_ROWS) + 15) / 16;
	size_t most = tiles > 4 ? least(4 * (uint64_t)s.compute_units, times(times(heads, listed > few ? listed : few), (tiles + 3) / 4)) * part_floats(s.J, false) : 0;
	if (rows > MANY_ROWS) {
		const uint64_t units = times(heads, (rows + 255) / 256), parts = least(16, tiles / MANY_LEAST);
		const size_t floats = parts > 1 ? least(MANY_ROUNDS * slots, times(units, parts)) * (part_floats(s.J, true) + 1) : 0; /* (two words a unit, of two parts at least) */
		const size_t shared = s.sequences > 1 && times(units, tiles) >= SHARE_LEAST * slots ? slots * (2 * part_floats(s.J, true) + 4) : 0;
		if (floats > most) most = floats;
		if (shared > most) most = shared;
	}
	return most;
}

} // namespace kmx

#endif
