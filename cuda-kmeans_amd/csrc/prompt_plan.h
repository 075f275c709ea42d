/*
 * How the attention over prompts is launched (prompt_attend_impl.h), and the room that its parts take. Plain host code without a HIP header.
 */
#ifndef KMX_PROMPT_PLAN_H
#define KMX_PROMPT_PLAN_H

#include <cmath>
#include <cstddef>
#include <cstdint>

namespace kmx {

struct PromptShape { uint32_t J, heads, group, sequences, max_queries, max_tokens, compute_units; }; /* 32 J channels */

/* units: rows of 128 (wide: 256) of a head of a sequence; parts of the tokens of each, of so many tiles of 32; units 0: too many for a call */
struct PromptPlan { uint32_t row_tiles, units, parts, tiles_per_part; bool wide; };

constexpr uint32_t PROMPT_LEAST = 2; /* tiles of a part at least */

/*
 * Rows of 256 a work-group where heads have 160 or 192 channels (128 of them do not have the registers), and where heads have 96 or 128 and there are more than two rounds of
 * work-groups of 256; else 128. 8192 tokens, 32 heads of 128: 525 us by 256, 550 by 128; 4 x 500: 25.4 and 22.9; 6 prompts of up to 4096, 24 heads of 64 channels, 268 and 202 when both were built.
 *
 * Parts where the work-groups do not fill the chip. A tile takes a work-group about STEP us, so P parts save STEP tiles (1 - 1 / P); their sums, in 32 bits, are written and read again
 * and joined in a launch of its own, ROWS us for each part of all rows and 4 us once. P is where both together are least: sqrt(STEP tiles / ROWS).
 */
inline PromptPlan plan_prompt(const PromptShape& s)
{
	PromptPlan plan{};
	plan.parts = 1;
	plan.tiles_per_part = 0x4000000; /* all of them */
	const uint64_t rows = (uint64_t)s.max_queries * s.group, pairs = (uint64_t)s.heads * s.sequences;
	if (rows > 0x7FFFFF00u || pairs > 0x7FFFFFFFu) return plan;
	plan.wide = s.J == 5 || s.J == 6 || ((s.J == 3 || s.J == 4) && rows * pairs > 512 * (uint64_t)s.compute_units);
	const uint32_t unit_rows = plan.wide ? 256 : 128;
	const uint64_t row_tiles = (rows + unit_rows - 1) / unit_rows, units = row_tiles * pairs;
	if (units > 0x7FFFFFFFu) return plan;
	plan.row_tiles = (uint32_t)row_tiles;
	plan.units = (uint32_t)units;
	const uint64_t slots = (s.J <= 4 && !plan.wide ? 2 : 1) * (uint64_t)s.compute_units; /* work-groups on the chip at a time */
	if (units == 0 || 2 * units > slots) return plan;
	const uint32_t tiles = s.max_tokens / 32 + (s.max_tokens % 32 ? 1 : 0);
	const double step = 0.3 + 0.06 * s.J, row = (double)(rows * pairs) * s.J * 256 / 4e6; /* 4 TB/s */
	double parts = sqrt(step * tiles / row);
	if (parts > (double)(slots / units)) parts = (double)(slots / units);
	if (parts > (double)(tiles / PROMPT_LEAST)) parts = (double)(tiles / PROMPT_LEAST);
	if (parts < 2 || step * tiles * (1 - 1 / parts) < 4 + row * parts) return plan;
	plan.tiles_per_part = (uint32_t)((double)tiles / parts + 0.999);
	plan.parts = (tiles + plan.tiles_per_part - 1) / plan.tiles_per_part;
	return plan;
}

/* a launch has fewer than 2^32 threads: 2^24 work-groups of 128 rows, 2^23 of 256 */
inline bool prompt_launches(const PromptPlan& plan) { return plan.units && (uint64_t)plan.units * plan.parts <= 0xFFFFFFFFu / (plan.wide ? 512u : 256u); }

/* floats of work space of a call, and the most of any (no more work-groups than the chip holds have parts: 51 MB at 192 channels) */
inline size_t prompt_floats(const PromptPlan& plan, uint32_t J) { return plan.parts > 1 ? (size_t)plan.units * plan.parts * (plan.wide ? 256 : 128) * (32 * (size_t)J + 2) : 0; }
inline size_t most_prompt_floats(uint32_t J, uint32_t compute_units) { return (J <= 6 ? 256 : 128) * (size_t)compute_units * (32 * (size_t)J + 2); }

} // namespace kmx

#endif
