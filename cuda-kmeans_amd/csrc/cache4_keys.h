/*
 * The order in which kmx_cache4_select (cache4.hip) takes pages, as unsigned words: larger for a better page. Plain code that the tests compile for
 * the host: the room of a list rests on no score having the key of a page that is always taken.
 */
#ifndef KMX_CACHE4_KEYS_H
#define KMX_CACHE4_KEYS_H

#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstring>

#ifdef __HIPCC__
#define KMX_HOST_DEVICE __host__ __device__ inline __attribute__((always_inline))
#else
#define KMX_HOST_DEVICE inline
#endif

namespace kmx {

/* floats in the order of unsigned words */
KMX_HOST_DEVICE uint32_t ordered(float v)
{
	uint32_t u;
	memcpy(&u, &v, 4);
	return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr uint32_t FORCED_KEY = 0xFF800000u;  /* ordered(infinity): the first and last pages, of which a list has room for all */
constexpr uint32_t MISSING_KEY = 0x007FFFFFu; /* ordered(-infinity): a page that is not there */

/* The score best * scale. Bounds that nobody made may hold anything, so the scale may be infinite or no number: the score is held to the finite
 * numbers, NaN to the lowest of them. */
KMX_HOST_DEVICE uint32_t page_key(bool forced, bool known, int best, float scale)
{
	const float score = (float)best * scale + 0.0f; /* (+ 0: one zero) */
	const uint32_t key = ordered(fminf(fmaxf(score, -FLT_MAX), FLT_MAX));
	return forced ? FORCED_KEY : known ? key : MISSING_KEY;
}

} // namespace kmx

#endif
