/* kmx_prompt_attend of include/kmx.h: checks and dispatch (kernels: prompt_attend_impl.h). */
#include "prompt_attend.h"

#include <cmath>

using namespace kmx;

extern "C" {

int kmx_prompt_attend(const kmx_prompt* prompt, int type, const void* q, size_t q_token_stride, size_t q_head_stride,
                      const void* keys, const void* values, size_t token_stride, size_t head_stride,
                      void* out, size_t out_token_stride, size_t out_head_stride, float* lse, float scale, int causal)
{
	clear_error();
	if (!prompt) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: null prompt");
	const kmx_prompt& b = *prompt;
	if (b.heads == 0 || b.query_heads == 0 || b.query_heads % b.heads) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: %u query heads are no multiple of %u heads", b.query_heads, b.heads);
	if (b.dim == 0 || b.dim % 32 || b.dim > 256) return fail(KMX_ERR_UNSUPPORTED, "kmx_prompt_attend: dim %u is no multiple of 32 up to 256", b.dim);
	if (type == KMX_F32) return fail(KMX_ERR_UNSUPPORTED, "kmx_prompt_attend: rows are KMX_F16 or KMX_BF16");
	if (type != KMX_F16 && type != KMX_BF16) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: unknown element type %d", type);
	if (causal != 0 && causal != 1) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: causal is 0 or 1");
	if (!(std::fabs(scale) <= 3.4e38f)) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: the scale is not finite");
	if (b.sequences == 0 || b.queries == 0 || b.max_queries == 0) return KMX_OK;
	if (!b.query_starts || !b.token_starts) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: null device pointer in the prompt");
	if (b.queries > 0x7FFFFFFFu || b.tokens > 0x7FFFFFFFu) return fail(KMX_ERR_UNSUPPORTED, "kmx_prompt_attend: queries and tokens are counted in 31 bits");
	if (!q || !out || (b.tokens && (!keys || !values))) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: null device pointer");
	if ((uintptr_t)q % 2 || (uintptr_t)keys % 2 || (uintptr_t)values % 2 || (uintptr_t)out % 2) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: rows start at multiples of 2 bytes");
	if (b.query_heads > 1 && out_head_stride < b.dim) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: head stride of the output %zu < dim %u", out_head_stride, b.dim);
	if (b.queries > 1 && out_token_stride < b.dim) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_attend: token stride of the output %zu < dim %u", out_token_stride, b.dim);
	PromptAttend a{};
	a.query_starts = b.query_starts;
	a.token_starts = b.token_starts;
	a.sequences = b.sequences;
	a.heads = b.heads;
	a.group = b.query_heads / b.heads;
	a.query_heads = b.query_heads;
	a.queries = b.queries;
	a.tokens = b.tokens;
	a.max_queries = b.max_queries < b.queries ? b.max_queries : b.queries; /* a bound may be as loose as it likes */
	a.max_tokens = b.max_tokens < b.tokens ? b.max_tokens : b.tokens;
	a.q = q;
	a.q_token = q_token_stride;
	a.q_head = q_head_stride;
	a.k = keys;
	a.v = values;
	a.token_stride = token_stride;
	a.head_stride = head_stride;
	a.out = out;
	a.out_token = out_token_stride;
	a.out_head = out_head_stride;
	a.lse = lse;
	/* a score below 2^127 times the factor stays a number; a scale of 0 takes the queries away */
	const float factor = std::fabs(scale) * 1.44269504088896341f;
	a.factor = factor < 1.2e-38f ? 1.2e-38f : factor > 0x1p100f ? 0x1p100f : factor;
	a.q_keep = scale == 0.0f ? 0u : 0xFFFFFFFFu;
	a.q_turn = scale < 0.0f ? 0x80008000u : 0u;
	a.causal = causal != 0;
	const auto aligned = [](const void* p, size_t token, size_t head) { return (uintptr_t)p % 16 == 0 && token % 8 == 0 && head % 8 == 0; };
	a.vec = aligned(q, q_token_stride, q_head_stride) && aligned(keys, token_stride, head_stride) && aligned(values, token_stride, head_stride) && aligned(out, out_token_stride, out_head_stride);
	/* offsets of pieces are counted in 32 bits, from the end of a sequence as far on as it is long among them */
	if ((uint64_t)a.max_tokens + 192 > 0x7FFFFFFFu / 2 / (token_stride ? token_stride : 1)) a.vec = false;
	const DeviceInfo* dev = nullptr;
	const int rc = device_info(&dev);
	if (rc) return rc;
	const uint32_t J = b.dim / 32;
	const PromptPlan plan = plan_prompt(PromptShape{ J, a.heads, a.group, a.sequences, a.max_queries, a.max_tokens, dev->compute_units });
	if (!prompt_launches(plan)) return fail(KMX_ERR_UNSUPPORTED, "kmx_prompt_attend: %u sequences of up to %u queries are too many for one call", b.sequences, a.max_queries);
	if (const size_t floats = prompt_floats(plan, J)) {
		const int rc2 = place_cache4("kmx_prompt_attend", floats, &a.partial, "kmx_prompt_reserve");
		if (rc2) return rc2;
	}
	const bool bf16 = type == KMX_BF16;
	switch (J) {
	case 1: return launch_prompt_attend<1>(a, bf16, plan);
	case 2: return launch_prompt_attend<2>(a, bf16, plan);
	case 3: return launch_prompt_attend<3>(a, bf16, plan);
	case 4: return launch_prompt_attend<4>(a, bf16, plan);
	case 5: return launch_prompt_attend<5>(a, bf16, plan);
	case 6: return launch_prompt_attend<6>(a, bf16, plan);
	case 7: return launch_prompt_attend<7>(a, bf16, plan);
	default: return launch_prompt_attend<8>(a, bf16, plan);
	}
}

int kmx_prompt_reserve(uint32_t dim)
{
	clear_error();
	if (recording_graph()) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_prompt_reserve: not allowed between kmx_graph_begin and kmx_graph_end");
	if (dim == 0 || dim % 32 || dim > 256) return fail(KMX_ERR_UNSUPPORTED, "kmx_prompt_reserve: dim %u is no multiple of 32 up to 256", dim);
	const DeviceInfo* dev = nullptr;
	const int rc = device_info(&dev);
	if (rc) return rc;
	Workspace* scratch = nullptr;
	if (noalloc_workspace(&scratch)) clear_error(); /* the address of the scratch array that recorded calls use (they do without if it has none) */
	float* partials = nullptr;
	return place_cache4("kmx_prompt_reserve", most_prompt_floats(dim / 32, dev->compute_units), &partials);
}

} // extern "C"
