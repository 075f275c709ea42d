/*
 * Attention over prompts on the device (kmx_prompt_attend of include/kmx.h): what its kernels are handed.
 */
#ifndef KMX_PROMPT_ATTEND_H
#define KMX_PROMPT_ATTEND_H

#include "cache4.h"
#include "prompt_plan.h"

namespace kmx {

struct PromptAttend {
	const int32_t* query_starts; const int32_t* token_starts; /* sequences + 1 */
	uint32_t sequences, heads, group, query_heads; /* heads of the keys, query heads of each and in all */
	uint32_t queries, tokens, max_queries, max_tokens;
	const void* q; size_t q_token, q_head;
	const void* k; const void* v; size_t token_stride, head_stride;
	void* out; size_t out_token, out_head;
	float* lse;
	float factor;             /* |scale| log2(e) */
	uint32_t q_keep, q_turn;  /* bits of two queries that stay, and those that are turned over */
	bool causal, vec;         /* vec: rows of 16-byte pieces */
	uint32_t row_tiles, units, parts, tiles_per_part; /* (filled in by the launcher) */
	float* partial;           /* sums of parts, where there are any */
};
template <int J> int launch_prompt_attend(const PromptAttend& a, bool bf16, const PromptPlan& plan);

} // namespace kmx

#endif
