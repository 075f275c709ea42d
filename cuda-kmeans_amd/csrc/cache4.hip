/*
 * The 4-bit cache: rows quantised as they are written and read back, bounds of its pages, the choice of pages by an 8-bit score, and the
 * C entry points of all of it (include/kmx.h, kmx_cache4_*). The attention that reads it is in cache4_attend_impl.h.
 */
#include "cache4.h"
#include "cache4_keys.h"

#include <cmath>
#include <cstring>

namespace kmx {

/* ---------------------------------------------------------------- writing and reading rows ------- */

struct Rows4 {
	Cache4 cache;
	void* keys; void* values;
	size_t token_stride, head_stride;
	const int32_t* slots;
	uint32_t tokens;
	bool vec;
};

/* the scale of a group: its largest magnitude with 5 significant bits (ties to the even one), at most 31 * 2^11 */
__device__ __forceinline__ _Float16 group_scale(float largest)
{
	uint32_t u = __builtin_bit_cast(uint32_t, fminf(largest, 65504.0f));
	u = (u + 0x3FFFFu + ((u >> 19) & 1u)) & ~0x7FFFFu;
	return (_Float16)fminf(__builtin_bit_cast(float, u), 63488.0f);
}

/* the 8 codes of one lane's channels, nibble i for channel i: the number of edges scale * (L_j + L_j+1) / 2 that |x| lies above (three
 * comparisons; NaN lies above none), and the sign */
__device__ __forceinline__ uint32_t codes8(const float x[8], float scale, const float middle[7])
{
	float edge[7];
	for (int j = 0; j < 7; ++j) edge[j] = scale * middle[j];
	uint32_t codes = 0;
	for (int i = 0; i < 8; ++i) {
		const float size = fabsf(x[i]);
		const bool b2 = size > edge[3];
		const float low = b2 ? edge[4] : edge[0], half = b2 ? edge[5] : edge[1], high = b2 ? edge[6] : edge[2];
		const bool b1 = size > half;
		const bool b0 = size > (b1 ? high : low);
		codes |= (b2 ? 4u << (4 * i) : 0u) | (b1 ? 2u << (4 * i) : 0u);
		codes |= (b0 ? 1u << (4 * i) : 0u) | (x[i] < 0.0f ? 8u << (4 * i) : 0u);
	}
	return codes;
}

__device__ __forceinline__ uint32_t nibbles_to_bytes(uint32_t w) /* four nibbles, one a byte */
{
	w = (w | w << 8) & 0x00FF00FFu;
	return (w | w << 4) & 0x0F0F0F0Fu;
}

/* 8 elements of a row as they lie there, and in floats */
template <typename T>
struct Raw8 { u32x4 w[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Raw8<T> fetch8(const T* p, bool vec)
{
	Raw8<T> r;
	if (vec) {
		for (uint32_t i = 0; i < sizeof(T) / 2; ++i) r.w[i] = __builtin_nontemporal_load((const u32x4*)p + i);
	} else if constexpr (sizeof(T) == 4) {
		for (int i = 0; i < 8; ++i) r.w[i / 4][i % 4] = ((const uint32_t*)p)[i];
	} else {
		for (int i = 0; i < 4; ++i) r.w[0][i] = ((const uint16_t*)p)[2 * i] | (uint32_t)((const uint16_t*)p)[2 * i + 1] << 16;
	}
	return r;
}
template <typename T>
__device__ __forceinline__ void floats8(const Raw8<T>& r, float x[8])
{
	for (int i = 0; i < 8; ++i) {
		if constexpr (sizeof(T) == 4) {
			const uint32_t w = r.w[i / 4][i % 4];
			x[i] = __builtin_bit_cast(float, w);
		} else {
			const uint32_t w = r.w[0][i / 2];
			if constexpr (__is_same(T, __bf16)) x[i] = __builtin_bit_cast(float, i % 2 ? w & 0xFFFF0000u : w << 16);
			else x[i] = (float)__builtin_bit_cast(half2v, w)[i % 2];
		}
	}
}

/*
 * A wavefront takes 16 tokens of one head, 64 pieces of 8 channels at a time: piece n is channels 8 (n % 4 J) of token n / 4 J, so that a load of all
 * lanes is whole rows side by side and a group of 32 channels four lanes, its maximum two exchanges inside them. The keys' words go where they
 * belong (a token's lie together); the values' bytes pass through LDS, 16 tokens of a pair side by side, and leave as 16 bytes a lane where the 16
 * tokens fill a block in order, else byte by byte. Rows go past the caches: nobody comes back to them. Bound by the vector units: 26 instructions a number,
 * 99 % of their time: 16384 tokens of 8 heads of 128 in bf16 (86 MB) 27 us, 3.2 TB/s.
 */
template <int J, typename T>
__global__ void __launch_bounds__(256)
write4_kernel(Rows4 a)
{
	constexpr uint32_t D = 32 * J;
	__shared__ __attribute__((aligned(16))) uint8_t lds[4][16 * 16 * J];
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE;
	const uint64_t unit = (uint64_t)blockIdx.x * 4 + wave;
	const uint32_t head = (uint32_t)(unit % a.cache.heads);
	const uint64_t first = unit / a.cache.heads * 16;
	if (first >= a.tokens) return; /* (no barriers below: a wavefront's LDS is its own) */
	const uint64_t places = (uint64_t)a.cache.page_count << a.cache.page_shift;
	const uint32_t page_mask = (1u << a.cache.page_shift) - 1;
	const int32_t slot = first + lane % 16 < a.tokens ? a.slots[first + lane % 16] : -1; /* lane n: of token n % 16 */
	uint8_t* const mine = lds[wave];
	auto block_of = [&](int32_t s) { return a.cache.blocks + block_offset<J>(a.cache, (uint32_t)s >> a.cache.page_shift, head, ((uint32_t)s & page_mask) / 16); };

	for (int which = 0; which < 2; ++which) {
		Raw8<T> raw[J];
		int32_t place[J];
#pragma unroll
		for (int n = 0; n < J; ++n) {
			const uint32_t piece = WAVE * n + lane, t = piece / (4 * J), c = piece % (4 * J);
			place[n] = __shfl(slot, (int)t);
			if ((uint64_t)(int64_t)place[n] >= places) place[n] = -1; /* (negative ones too) */
			const uint64_t token = min(first + t, (uint64_t)a.tokens - 1);
			raw[n] = fetch8((const T*)(which ? a.values : a.keys) + token * a.token_stride + head * a.head_stride + 8 * c, a.vec);
		}
		float middle[7];
		{
			const uint16_t* l = a.cache.levels + ((size_t)head * 2 + which) * 8;
			float below = (float)__builtin_bit_cast(_Float16, l[0]);
			for (int j = 0; j < 7; ++j) {
				const float above = (float)__builtin_bit_cast(_Float16, l[j + 1]);
				middle[j] = (below + above) * 0.5f;
				below = above;
			}
		}
#pragma unroll
		for (int n = 0; n < J; ++n) {
			const uint32_t piece = WAVE * n + lane, t = piece / (4 * J), c = piece % (4 * J), j = c / 4, g = c % 4;
			float x[8];
			floats8<T>(raw[n], x);
			float largest = 0.0f; /* fmaxf leaves NaN out */
			for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(x[i]));
			largest = fmaxf(largest, dpp<DPP_XOR1>(largest));
			largest = fmaxf(largest, dpp<DPP_XOR2>(largest));
			const _Float16 scale = group_scale(largest);
			const uint32_t codes = codes8(x, (float)scale, middle);
			const uint32_t at = (uint32_t)place[n] % 16;
			if (which == 0) {
				if (place[n] >= 0) {
					uint8_t* const block = block_of(place[n]);
					((uint32_t*)(block + at * (D / 2)))[g * J + j] = nibbles_to_bytes(codes & 0xFFFFu) | nibbles_to_bytes(codes >> 16) << 4;
					if (g == 0) ((_Float16*)(block + 16 * D))[at * J + j] = scale;
				}
			} else {
				/* lanes g and g + 2 hold the two channels of 8 pairs: each makes the bytes of four */
				const uint32_t other = dpp<DPP_XOR2>(codes), half = g / 2;
				const uint32_t low = (half ? other : codes) >> (16 * half), high = (half ? codes : other) >> (16 * half);
				const uint32_t bytes = nibbles_to_bytes(low & 0xFFFFu) | nibbles_to_bytes(high & 0xFFFFu) << 4;
				const uint32_t pair = 16 * j + 8 * (g & 1) + 4 * half;
				for (int b = 0; b < 4; ++b) mine[(pair + b) * 16 + t] = (uint8_t)(bytes >> (8 * b));
				if (place[n] >= 0 && g == 0) ((_Float16*)(block_of(place[n]) + 17 * D))[16 * j + at] = scale;
			}
		}
	}
	wave_sync();
	const int32_t slot0 = __builtin_amdgcn_readfirstlane(slot);
	const bool in_order = (uint64_t)(int64_t)slot0 < places && slot0 % 16 == 0 && __ballot(slot != slot0 + (int32_t)(lane % 16)) == 0;
	if (in_order) {
		uint8_t* const block = block_of(slot0);
		for (uint32_t p = lane; p < D / 2; p += WAVE) *(u32x4*)(block + 8 * D + p * 16) = *(const u32x4*)(mine + p * 16);
	} else {
		for (uint32_t p = lane; p < D / 2; p += WAVE) {
			const u32x4 w = *(const u32x4*)(mine + p * 16);
#pragma unroll
			for (int n = 0; n < 16; ++n) {
				const int32_t s = __builtin_amdgcn_readlane(slot, n);
				if ((uint64_t)(int64_t)s < places) (block_of(s) + 8 * D + (uint32_t)s % 16)[p * 16] = (uint8_t)(w[n / 4] >> (8 * (n % 4)));
			}
		}
	}
}

/* The same pieces backwards; a place outside the cache reads as zeros. Bound by the rows that it writes: 32768 tokens of 8 heads of 128 in bf16 (172 MB)
 * 28 us, 6.1 TB/s; through the caches 34. */
template <int J, typename T>
__global__ void __launch_bounds__(256)
read4_kernel(Rows4 a)
{
	constexpr uint32_t D = 32 * J, ROW = D / 2 + 8; /* LDS: the values' bytes token by token, rows 8 bytes apart in the banks */
	__shared__ __attribute__((aligned(16))) uint8_t lds[4][16 * ROW];
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE;
	const uint64_t unit = (uint64_t)blockIdx.x * 4 + wave;
	const uint32_t head = (uint32_t)(unit % a.cache.heads);
	const uint64_t first = unit / a.cache.heads * 16;
	if (first >= a.tokens) return;
	const uint64_t places = (uint64_t)a.cache.page_count << a.cache.page_shift;
	const uint32_t page_mask = (1u << a.cache.page_shift) - 1;
	const int32_t slot = first + lane % 16 < a.tokens ? a.slots[first + lane % 16] : -1;
	uint8_t* const mine = lds[wave];
	auto block_of = [&](int32_t s) { return a.cache.blocks + block_offset<J>(a.cache, (uint32_t)s >> a.cache.page_shift, head, ((uint32_t)s & page_mask) / 16); };

	/* the keys' words and the scales under way, then the values' bytes into LDS */
	uint32_t codes[J];
	uint16_t scales[2][J];
	int32_t place[J];
#pragma unroll
	for (int n = 0; n < J; ++n) {
		const uint32_t piece = WAVE * n + lane, t = piece / (4 * J), c = piece % (4 * J), j = c / 4, g = c % 4;
		place[n] = __shfl(slot, (int)t);
		if ((uint64_t)(int64_t)place[n] >= places) place[n] = -1;
		codes[n] = 0;
		scales[0][n] = scales[1][n] = 0;
		if (place[n] >= 0) {
			const uint8_t* const block = block_of(place[n]);
			const uint32_t at = (uint32_t)place[n] % 16;
			codes[n] = ((const uint32_t*)(block + at * (D / 2)))[g * J + j];
			scales[0][n] = ((const uint16_t*)(block + 16 * D))[at * J + j];
			scales[1][n] = ((const uint16_t*)(block + 17 * D))[16 * j + at];
		}
	}
	const int32_t slot0 = __builtin_amdgcn_readfirstlane(slot);
	const bool in_order = (uint64_t)(int64_t)slot0 < places && slot0 % 16 == 0 && __ballot(slot != slot0 + (int32_t)(lane % 16)) == 0;
	if (in_order) {
		const uint8_t* const block = block_of(slot0);
		for (uint32_t p = lane; p < D / 2; p += WAVE) {
			const u32x4 w = *(const u32x4*)(block + 8 * D + p * 16);
			for (int n = 0; n < 16; ++n) mine[n * ROW + p] = (uint8_t)(w[n / 4] >> (8 * (n % 4)));
		}
	} else {
		for (uint32_t p = lane; p < D / 2; p += WAVE) {
			uint8_t w[16]; /* all 16 under way before the first is waited for */
#pragma unroll
			for (int n = 0; n < 16; ++n) {
				const int32_t s = __builtin_amdgcn_readlane(slot, n);
				w[n] = (uint64_t)(int64_t)s < places ? (block_of(s) + 8 * D + (uint32_t)s % 16)[p * 16] : 0;
			}
#pragma unroll
			for (int n = 0; n < 16; ++n) mine[n * ROW + p] = w[n];
		}
	}
	wave_sync();
	for (int which = 0; which < 2; ++which) {
		const Magnitudes m = load_magnitudes(a.cache.levels, head, which);
#pragma unroll
		for (int n = 0; n < J; ++n) {
			const uint32_t piece = WAVE * n + lane, t = piece / (4 * J), c = piece % (4 * J), j = c / 4, g = c % 4;
			if (first + t >= a.tokens) continue;
			uint32_t w[4];
			if (which == 0) {
				unpack4<false>(codes[n], m, w[0], w[1]);
				unpack4<true>(codes[n], m, w[2], w[3]);
			} else {
				const u32x2 b = *(const u32x2*)(mine + t * ROW + 16 * j + 8 * (g & 1));
				unpack4<false>(b[0] >> (4 * (g / 2)), m, w[0], w[1]);
				unpack4<false>(b[1] >> (4 * (g / 2)), m, w[2], w[3]);
			}
			const float scale = (float)__builtin_bit_cast(_Float16, scales[which][n]);
			float x[8];
			for (int i = 0; i < 8; ++i) x[i] = place[n] >= 0 ? scale * (float)__builtin_bit_cast(half2v, w[i / 2])[i % 2] : 0.0f;
			store8((T*)(which ? a.values : a.keys) + (first + t) * a.token_stride + head * a.head_stride + 8 * c, a.vec, x);
		}
	}
}

template <typename T>
static int launch_rows4(bool write, const Rows4& a, uint32_t J)
{
	const uint64_t units = ((uint64_t)a.tokens + 15) / 16 * a.cache.heads, groups = (units + 3) / 4;
	if (groups > 0x7FFFFFFFu) return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_%s: %u tokens of %u heads are too many for one call", write ? "write" : "read", a.tokens, a.cache.heads);
	const dim3 grid((unsigned)groups), block(256);
	switch (J) {
#define KMX_CASE(N)                                                                                                     \
	case N:                                                                                                               \
		if (write) KMX_LAUNCH_KERNEL((write4_kernel<N, T>), grid, block, 0, stream(), a);                                  \
		else KMX_LAUNCH_KERNEL((read4_kernel<N, T>), grid, block, 0, stream(), a);                                         \
		break;
		KMX_CASE(1) KMX_CASE(2) KMX_CASE(3) KMX_CASE(4) KMX_CASE(5) KMX_CASE(6) KMX_CASE(7) KMX_CASE(8)
#undef KMX_CASE
	}
	KMX_LAUNCH_CHECK("write4_kernel / read4_kernel");
	return KMX_OK;
}

/* ---------------------------------------------------------------- bounds of pages ---------------- */

/*
 * 1, 2 or 4 wavefronts (as many as a page has blocks, at most 4) take a page and head. A wavefront unpacks a block, lane = 4 token + g as in the
 * block, and turns it over in LDS: its lanes go on with the channels, 16 tokens each. Values are products of half-precision numbers, exact in
 * floats, and maxima know no order. Few pages are made at a time (those that were written to), so that its own latency bounds it: 4 to 7 us, of which
 * 3.5 are a launch with its first load and last store.
 */
template <int J>
__global__ void __launch_bounds__(256)
bound4_kernel(Cache4 c, const int32_t* __restrict__ pages, const int32_t* __restrict__ counts, uint32_t count, uint32_t waves)
{
	constexpr uint32_t D = 32 * J, ROW = D + 4;
	__shared__ __attribute__((aligned(16))) float turned[4][16 * ROW];
	__shared__ float high[4][D], low[4][D];
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE, t = lane / 4, g = lane % 4;
	const uint32_t set = wave / waves, mine = wave % waves; /* the work-group's 4 / waves pages, and the wavefronts of each */
	const uint64_t unit = (uint64_t)blockIdx.x * (4 / waves) + set, entry = unit / c.heads;
	const uint32_t head = (uint32_t)(unit % c.heads);
	const int32_t page = entry < count ? pages[entry] : -1;
	const bool there = page >= 0 && (uint32_t)page < c.page_count;
	const int32_t room = 1 << c.page_shift;
	const int32_t tokens = !there || counts[entry] < 0 ? 0 : counts[entry] < room ? counts[entry] : room;
	const Magnitudes m = load_magnitudes(c.levels, head, 0);
	constexpr int EACH = (D + WAVE - 1) / WAVE; /* channels a lane */
	float hi[EACH], lo[EACH];
#pragma unroll
	for (int i = 0; i < EACH; ++i) { hi[i] = -__builtin_inff(); lo[i] = __builtin_inff(); }
	for (int32_t from = 16 * mine; from < tokens; from += 16 * waves) {
		const uint8_t* block = c.blocks + block_offset<J>(c, (uint32_t)page, head, from / 16);
		uint32_t codes[J], scales[(J + 1) / 2];
		{
			const uint32_t* p = (const uint32_t*)(block + 4 * J * lane);
			const uint16_t* s = (const uint16_t*)(block + 16 * D) + t * J;
#pragma unroll
			for (int j = 0; j < J; ++j) codes[j] = p[j];
#pragma unroll
			for (int j = 0; j < J; ++j) scales[j / 2] = j % 2 ? scales[j / 2] | (uint32_t)s[j] << 16 : s[j];
		}
		wave_sync();
#pragma unroll
		for (int j = 0; j < J; ++j) {
			uint32_t w[4];
			unpack4<false>(codes[j], m, w[0], w[1]);
			unpack4<true>(codes[j], m, w[2], w[3]);
			const float scale = (float)__builtin_bit_cast(_Float16, (uint16_t)(scales[j / 2] >> (16 * (j % 2))));
			float x[8];
			for (int i = 0; i < 8; ++i) x[i] = scale * (float)__builtin_bit_cast(half2v, w[i / 2])[i % 2];
			float* row = turned[wave] + t * ROW + 32 * j + 8 * g;
			*(f32x4*)row = f32x4{ x[0], x[1], x[2], x[3] };
			*(f32x4*)(row + 4) = f32x4{ x[4], x[5], x[6], x[7] };
		}
		wave_sync();
		const int32_t rows = min(16, tokens - from);
#pragma unroll
		for (int i = 0; i < EACH; ++i) {
			const uint32_t ch = min(lane + WAVE * i, D - 1);
#pragma unroll
			for (int n = 0; n < 16; ++n) {
				const float x = turned[wave][n * ROW + ch];
				hi[i] = n < rows ? fmaxf(hi[i], x) : hi[i];
				lo[i] = n < rows ? fminf(lo[i], x) : lo[i];
			}
		}
	}
#pragma unroll
	for (int i = 0; i < EACH; ++i)
		if (lane + WAVE * i < D) { high[wave][lane + WAVE * i] = hi[i]; low[wave][lane + WAVE * i] = lo[i]; }
	__syncthreads();
	if (mine != 0) return;
	float top = 0.0f;
#pragma unroll
	for (int i = 0; i < EACH; ++i) {
		const uint32_t ch = min(lane + WAVE * i, D - 1);
		for (uint32_t w = 1; w < waves; ++w) { hi[i] = fmaxf(hi[i], high[wave + w][ch]); lo[i] = fminf(lo[i], low[wave + w][ch]); }
		if (tokens == 0) hi[i] = lo[i] = 0.0f;
		if (lane + WAVE * i < D) top = fmaxf(top, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
	}
	for (int d = 1; d < WAVE; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
	if (!there) return;
	const float by = top > 0.0f ? 1.0f / top * 127.0f : 0.0f;
	int8_t* out = c.bounds + ((size_t)page * c.heads + head) * (2 * D);
#pragma unroll
	for (int i = 0; i < EACH; ++i) {
		const uint32_t ch = lane + WAVE * i;
		if (ch >= D) continue;
		out[ch] = (int8_t)fminf(fmaxf(ceilf(hi[i] * by), -127.0f), 127.0f); /* outwards, so that a bound stays one */
		out[D + ch] = (int8_t)fminf(fmaxf(floorf(lo[i] * by), -127.0f), 127.0f);
	}
	if (lane == 0) c.bound_scales[(size_t)page * c.heads + head] = top / 127.0f;
}

/* ---------------------------------------------------------------- the choice of pages ------------ */

struct Select4 {
	Cache4 cache;
	Batch4 batch;
	const void* q; size_t q_token, q_head;
	uint32_t* keys;     /* [token][head][table_stride], larger for a better page */
	int32_t* chosen;    /* [token][head][top] */
	uint32_t top, first, last;
	uint32_t span, span_bits; /* query heads of a token side by side: the power of two from `group` on, at most 16 */
	uint32_t per;       /* tokens of a tile of queries: a power of two, at most 16 / span and 8 */
	uint32_t token_tiles, chunks, chunk; /* tiles of queries a sequence; parts of the pages and how many times 64 each */
	bool bf16, vec;
};

/*
 * The scores of pages: the bound on q . k over a page, in 8 bits. 16 rows of queries (tokens of one head of the cache, their query heads side by
 * side) are 8-bit columns of v_mfma_i32_16x16x64_i8: the positive parts against the largest values, the negative ones against the smallest.
 * Whole numbers below 2^24, the same in any order. A lane holds 16 of each 64 of the 2 dim numbers of row or page lane % 16. The work-group
 * rounds the rows once, in LDS, for all its wavefronts (768 instructions a wavefront if each does it for itself).
 */
template <int J>
struct Scorer4 {
	static constexpr uint32_t D = 32 * J, ROW = 2 * D + 16; /* LDS: 8 rows one below the other lie in 8 different groups of banks */
	struct Lds {
		__attribute__((aligned(16))) int8_t rows[16 * ROW];
		uint32_t largest[8];
	};
	const Select4& a;
	const Sequence& seq;
	uint32_t head, tile, col, kg, i; /* i: the query of the lane's row */
	bool token_there;
	i32x4 q8[J];

	__device__ __forceinline__ Scorer4(const Select4& args, const Sequence& sequence, uint32_t cache_head, uint32_t tile_of_queries, uint32_t lane)
	    : a(args), seq(sequence), head(cache_head), tile(tile_of_queries), col(lane % 16), kg(lane / 16), i(tile * args.per + (lane % 16 >> args.span_bits))
	{
		token_there = (lane % 16 >> a.span_bits) < a.per && i < seq.queries;
	}
	/* 8 channels of a row of the 16 from query head g0 on; zeros where there is none */
	__device__ __forceinline__ u32x4 load(uint32_t g0, uint32_t row, uint32_t channel) const
	{
		const uint32_t token = tile * a.per + (row >> a.span_bits), h = g0 + (row & (a.span - 1));
		if ((row >> a.span_bits) >= a.per || token >= seq.queries || h >= a.batch.group) return u32x4{ 0, 0, 0, 0 };
		return load_raw8((const uint16_t*)a.q + (size_t)(seq.first + token) * a.q_token + (size_t)(head * a.batch.group + h) * a.q_head + channel, a.vec);
	}
	/* the largest magnitude of each token, over all its query heads; by all threads of the work-group */
	__device__ __forceinline__ void measure(Lds& lds, uint32_t threads) const
	{
		if (threadIdx.x < 8) lds.largest[threadIdx.x] = 0;
		__syncthreads();
		for (uint32_t g0 = 0; g0 < a.batch.group; g0 += 16)
			for (uint32_t item = threadIdx.x; item < a.per * a.span * (D / 8); item += threads) {
				const u32x4 raw = load(g0, item / (D / 8), item % (D / 8) * 8);
				float largest = 0.0f;
				for (int e = 0; e < 8; ++e) {
					const uint32_t w = raw[e / 2];
					largest = fmaxf(largest, fabsf(raw_element(w, e % 2, a.bf16)));
				}
				atomicMax(&lds.largest[item / (D / 8) >> a.span_bits], __builtin_bit_cast(uint32_t, largest)); /* (not negative: in the order of their words) */
			}
		__syncthreads();
	}
	/* the 16 rows from query head g0 on in 8 bits, into LDS and then the lanes */
	__device__ __forceinline__ void round(Lds& lds, uint32_t g0, uint32_t threads)
	{
		for (uint32_t item = threadIdx.x; item < 16 * (D / 8); item += threads) {
			const uint32_t row = item / (D / 8), channel = item % (D / 8) * 8;
			const float largest = __builtin_bit_cast(float, lds.largest[min((row >> a.span_bits), 7u)]);
			const float by = largest > 0.0f ? 1.0f / largest * 127.0f : 0.0f;
			const u32x4 raw = load(g0, row, channel);
			u32x2 up{ 0, 0 }, down{ 0, 0 };
			for (int e = 0; e < 8; ++e) {
				const uint32_t w = raw[e / 2];
				float v = raw_element(w, e % 2, a.bf16) * by;
				v = v != v ? 0.0f : fminf(fmaxf(rintf(v), -127.0f), 127.0f);
				up[e / 4] |= (uint32_t)((int)fmaxf(v, 0.0f) & 0xFF) << (8 * (e % 4));
				down[e / 4] |= (uint32_t)((int)fminf(v, 0.0f) & 0xFF) << (8 * (e % 4));
			}
			*(u32x2*)(lds.rows + row * ROW + channel) = up;
			*(u32x2*)(lds.rows + row * ROW + D + channel) = down;
		}
		__syncthreads();
#pragma unroll
		for (int c = 0; c < J; ++c) q8[c] = *(const i32x4*)(lds.rows + col * ROW + 64 * c + 16 * kg);
	}
	/* the whole numbers of 16 pages: lane (col, kg) gets those of its row and the pages 4 kg + r, of the rows from query head g0 on */
	__device__ __forceinline__ void dots(const i32x4 b[J], uint32_t g0, int best[4]) const
	{
		i32x4 dot{ 0, 0, 0, 0 };
#pragma unroll
		for (int c = 0; c < J; ++c) dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[c], q8[c], dot, 0, 0, 0);
		const bool there = token_there && g0 + (col & (a.span - 1)) < a.batch.group;
		for (int r = 0; r < 4; ++r) best[r] = there ? dot[r] : INT32_MIN;
		for (uint32_t d = 1; d < a.span; d *= 2) /* the largest over the token's query heads */
			for (int r = 0; r < 4; ++r) best[r] = max(best[r], __shfl_xor(best[r], (int)d));
	}
	/* pages of the sequence with a token that the lane's query sees */
	__device__ __forceinline__ uint32_t seen() const { return token_there ? (visible_to(a.batch, seq, i) + (1u << a.cache.page_shift) - 1) >> a.cache.page_shift : 0; }
	/* the lane that writes number r of its page: the lanes of a token share them out */
	__device__ __forceinline__ bool writes(int r) const { return token_there && ((col & (a.span - 1))) < 4 && ((uint32_t)r & (a.span - 1) & 3) == (col & (a.span - 1) & 3); }
	__device__ __forceinline__ uint32_t key(uint32_t page, uint32_t pages, int best, float scale, bool known) const
	{
		return page_key(page < a.first || page + a.last >= pages, known, best, scale);
	}
};

/*
 * All scores of a work-group's pages [from, end), a wavefront 16 TILES pages at a time and `stride` pages further each time; the bounds of the next ones are under way
 * while it works on those. put(query, page, key) takes them. More than 16 query heads to a head: again for each 16, the largest kept.
 */
template <int J, int TILES, typename GET, typename PUT>
__device__ __forceinline__ void score_pages(Scorer4<J>& scorer, typename Scorer4<J>::Lds& lds, const int32_t* table, uint32_t from, uint32_t end, uint32_t pages, uint32_t stride, uint32_t threads, const GET& get, const PUT& put)
{
	const Select4& a = scorer.a;
	const uint32_t col = scorer.col, kg = scorer.kg;
	auto page_at = [&](uint32_t p) { return (uint32_t)table[min(p, pages - 1)]; };
	uint32_t page[TILES], after[TILES];
	float scale[TILES];
	i32x4 b[TILES][J];
	auto fetch = [&]() {
#pragma unroll
		for (int t = 0; t < TILES; ++t) {
			const bool there = page[t] < a.cache.page_count;
			const size_t at = (size_t)(there ? page[t] : 0) * a.cache.heads + scorer.head;
			scale[t] = a.cache.bound_scales[at];
			const int8_t* bounds = a.cache.bounds + at * (64 * J) + 16 * kg;
#pragma unroll
			for (int c = 0; c < J; ++c) b[t][c] = *(const i32x4*)(bounds + 64 * c);
		}
	};
	auto begin = [&]() {
#pragma unroll
		for (int t = 0; t < TILES; ++t) page[t] = page_at(from + 16 * t + col);
#pragma unroll
		for (int t = 0; t < TILES; ++t) after[t] = page_at(from + stride + 16 * t + col);
		fetch();
	};
	begin();
	scorer.measure(lds, threads);
	const uint32_t seen = scorer.seen();
	for (uint32_t g0 = 0; g0 < a.batch.group; g0 += 16) {
		if (g0) {
			__syncthreads(); /* (the rows before have been read) */
			begin();
		}
		scorer.round(lds, g0, threads);
		for (uint32_t p0 = from; p0 < end; p0 += stride) {
			int best[TILES][4];
			float scales[TILES];
			bool known[TILES];
#pragma unroll
			for (int t = 0; t < TILES; ++t) {
				scorer.dots(b[t], g0, best[t]);
				scales[t] = scale[t];
				known[t] = page[t] < a.cache.page_count;
				page[t] = after[t];
			}
			fetch();
#pragma unroll
			for (int t = 0; t < TILES; ++t) after[t] = page_at(p0 + 2 * stride + 16 * t + col);
#pragma unroll
			for (int t = 0; t < TILES; ++t)
#pragma unroll
				for (int r = 0; r < 4; ++r) {
					const float sc = __shfl(scales[t], (int)(4 * kg + r)); /* (lanes 0 to 15 hold the scales of the 16 pages) */
					const int there = __shfl(known[t] ? 1 : 0, (int)(4 * kg + r));
					const uint32_t p = p0 + 16 * t + 4 * kg + r;
					if (!scorer.writes(r) || p >= min(seen, end)) continue;
					const uint32_t k = scorer.key(p, seen, best[t][r], sc, there);
					put(p, g0 ? max(get(p), k) : k);
				}
		}
	}
}

/* Many pages for few queries: scores in one kernel, a part of the pages a work-group, the choice in the next. Latency of the chain queries - rounding -
 * products bounds both: 1024 pages of 8 heads, 16 sequences (34 MB of bounds) 12 us and 7.7. */
template <int J>
__global__ void __launch_bounds__(256)
score4_kernel(Select4 a)
{
	__shared__ typename Scorer4<J>::Lds lds;
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE;
	const uint32_t head = blockIdx.x, s = blockIdx.y, tile = a.token_tiles == 1 ? 0 : blockIdx.z % a.token_tiles, part = a.token_tiles == 1 ? blockIdx.z : blockIdx.z / a.token_tiles;
	const Sequence seq = sequence_of(a.batch, s, a.cache.page_shift);
	if (tile * a.per >= seq.queries) return;
	const uint32_t page_tokens = 1u << a.cache.page_shift, last_i = min(seq.queries, (tile + 1) * a.per) - 1;
	const uint32_t pages = (visible_to(a.batch, seq, last_i) + page_tokens - 1) >> a.cache.page_shift;
	if (part * a.chunk * 64 >= pages) return;
	Scorer4<J> scorer(a, seq, head, tile, lane);
	uint32_t* const keys = a.keys + ((size_t)(seq.first + (scorer.token_there ? scorer.i : 0)) * a.cache.heads + head) * a.batch.table_stride;
	score_pages<J, 1>(scorer, lds, a.batch.table + (size_t)s * a.batch.table_stride, (part * a.chunk * 4 + wave) * 16, min(pages, (part + 1) * a.chunk * 64), pages, 64, 256,
	                  [&](uint32_t p) { return keys[p]; }, [&](uint32_t p, uint32_t k) { keys[p] = k; });
}

/*
 * The `top` best of n keys, ascending. The keys' range is cut into 512 steps, whose numbers of keys tell the step with the threshold, that step again
 * into 512, until all of a step is wanted or its keys are equal (four passes over 8 bits each, whatever the keys, took 9 us for 1024 keys; this
 * mostly ends after one). Then one pass in the order of the pages keeps what lies above the threshold and as many at it as are left, the lowest
 * first. All threads of the work-group come here, `threads` of them (whole wavefronts, thread `tid` of them) to each list. Pages that are always taken
 * are no more than `top` (page_key gives their key to no score); nothing is written behind the list whatever the keys.
 */
struct ChooseLds { uint32_t histogram[512], low, high, forced, step[3]; }; /* of a list */
template <typename KEY>
__device__ __forceinline__ void choose_top(const KEY& key, uint32_t n, uint32_t top, int32_t* out, uint32_t tid, uint32_t threads, ChooseLds& lds, uint32_t* above, uint32_t* equal)
{
	const uint32_t wave = tid / WAVE, lane = tid % WAVE, waves = threads / WAVE;
	const bool all = n <= top; /* (n = 0 and out = null where there is no list) */
	if (all)
		for (uint32_t e = tid; out && e < top; e += threads) out[e] = e < n ? (int32_t)e : -1;
	const uint32_t some = all ? 0 : n;
	if (tid == 0) { lds.low = 0xFFFFFFFFu; lds.high = 0; lds.forced = 0; }
	for (uint32_t e = tid; e < 512; e += threads) lds.histogram[e] = 0;
	__syncthreads();
	{
		uint32_t low = 0xFFFFFFFFu, high = 0, forced = 0;
		for (uint32_t p = tid; p < some; p += threads) {
			const uint32_t k = key(p);
			if (k == FORCED_KEY) ++forced;
			else { low = min(low, k); high = max(high, k); }
		}
		for (int d = 1; d < WAVE; d *= 2) {
			low = min(low, (uint32_t)__shfl_xor((int)low, d));
			high = max(high, (uint32_t)__shfl_xor((int)high, d));
			forced += __shfl_xor((int)forced, d);
		}
		if (lane == 0 && !all) { atomicMin(&lds.low, low); atomicMax(&lds.high, high); atomicAdd(&lds.forced, forced); }
	}
	__syncthreads();
	/* kept: the keys above `threshold`, and the first `rest` of those equal to it */
	uint32_t low = lds.low, width = 0xFFFFFFFFu, rest = top - (all ? top : min(lds.forced, top)), threshold = lds.high; /* the threshold lies in [low, low + width) */
	int shift = all || lds.high <= low ? 0 : 32 - __clz(lds.high - low);
	shift = shift > 9 ? shift - 9 : 0;
	bool done = all || rest == 0;
	while (__syncthreads_or(!done)) {
		if (!done)
			for (uint32_t p = tid; p < some; p += threads) {
				const uint32_t k = key(p);
				if (k != FORCED_KEY && k >= low && k - low < width) atomicAdd(&lds.histogram[(k - low) >> shift], 1u);
			}
		__syncthreads();
		if (wave == 0 && !done) { /* lane l: steps 511 - 8 l and the seven below */
			uint32_t sum = 0;
			for (int e = 0; e < 8; ++e) sum += lds.histogram[511 - 8 * lane - e];
			uint32_t upto = sum;
			for (int d = 1; d < WAVE; d *= 2) {
				const uint32_t v = __shfl_up(upto, d);
				if (lane >= (uint32_t)d) upto += v;
			}
			uint32_t before = upto - sum;
			if (before < rest && rest <= upto)
				for (int e = 0; e < 8; ++e) {
					const uint32_t h = lds.histogram[511 - 8 * lane - e];
					if (rest <= before + h) {
						lds.step[0] = 511 - 8 * lane - e;
						lds.step[1] = rest - before;
						lds.step[2] = h;
						break;
					}
					before += h;
				}
		}
		__syncthreads();
		if (!done) {
			low += lds.step[0] << shift;
			width = 1u << shift;
			rest = lds.step[1];
			if (lds.step[2] == rest) { /* all of the step */
				threshold = low - 1;
				rest = 0;
				done = true;
			} else if (shift == 0) {
				threshold = low;
				done = true;
			}
			shift = shift > 9 ? shift - 9 : 0;
			for (uint32_t e = tid; e < 512; e += threads) lds.histogram[e] = 0;
		}
	}
	/* a wavefront takes a stretch of the pages: how many of it lie above the threshold and at it, then where they go */
	const uint32_t stretch = ((some + waves - 1) / waves + WAVE - 1) / WAVE * WAVE, from = wave * stretch, to = min(some, from + stretch);
	uint32_t gt = 0, eq = 0;
	for (uint32_t p0 = from; p0 < to; p0 += WAVE) {
		const uint32_t p = p0 + lane, k = p < to ? key(p) : 0;
		gt += __popcll(__ballot(p < to && k > threshold));
		eq += __popcll(__ballot(p < to && k == threshold));
	}
	if (lane == 0) { above[wave] = gt; equal[wave] = eq; }
	__syncthreads();
	uint32_t written = lane < wave ? above[lane] : 0, ties = lane < wave ? equal[lane] : 0; /* before this stretch (at most 16 wavefronts) */
	for (int d = 1; d < 16; d *= 2) { written += __shfl_xor((int)written, d); ties += __shfl_xor((int)ties, d); }
	written = (uint32_t)__builtin_amdgcn_readfirstlane((int)written);
	ties = (uint32_t)__builtin_amdgcn_readfirstlane((int)ties);
	const uint64_t below = ((uint64_t)1 << lane) - 1;
	for (uint32_t p0 = from; p0 < to; p0 += WAVE) {
		const uint32_t p = p0 + lane, k = p < to ? key(p) : 0;
		const bool is_above = p < to && k > threshold, is_equal = p < to && k == threshold;
		const uint64_t ballot_above = __ballot(is_above), ballot_equal = __ballot(is_equal);
		const uint32_t my_eq = ties + __popcll(ballot_equal & below), my_gt = written + __popcll(ballot_above & below);
		const uint32_t at = my_gt + min(my_eq, rest);
		if ((is_above || (is_equal && my_eq < rest)) && at < top) out[at] = (int32_t)p;
		written += __popcll(ballot_above);
		ties += __popcll(ballot_equal);
	}
}

__global__ void __launch_bounds__(512)
choose4_kernel(Select4 a)
{
	constexpr uint32_t CACHED = 8192;
	__shared__ uint32_t above[8], equal[8], cached[CACHED];
	__shared__ ChooseLds lds;
	const uint32_t head = blockIdx.x, s = blockIdx.y, i = blockIdx.z;
	const Sequence seq = sequence_of(a.batch, s, a.cache.page_shift);
	if (i >= seq.queries) return;
	const uint32_t n = (visible_to(a.batch, seq, i) + (1u << a.cache.page_shift) - 1) >> a.cache.page_shift;
	const size_t row = (size_t)(seq.first + i) * a.cache.heads + head;
	const uint32_t* keys = a.keys + row * a.batch.table_stride;
	if (n > CACHED) {
		choose_top([&](uint32_t p) { return keys[p]; }, n, a.top, a.chosen + row * a.top, threadIdx.x, 512, lds, above, equal);
		return;
	}
	if (n > a.top)
		for (uint32_t p = threadIdx.x; p < n; p += 512) cached[p] = keys[p];
	choose_top([&](uint32_t p) { return cached[p]; }, n, a.top, a.chosen + row * a.top, threadIdx.x, 512, lds, above, equal);
}

/*
 * Both in one kernel, where the keys of a tile of queries fit LDS and a work-group reads them fast enough: it takes `per` tokens of one
 * head, all pages. 625 pages, 2 x 128 queries, 16 query heads on 4 of 64: 17 us.
 */
constexpr uint32_t select_threads(uint32_t J, bool small) { return small ? 256 : J <= 4 ? 1024 : 512; } /* few pages, or as many wavefronts as the registers allow */
constexpr uint32_t SELECT_FEW = 512, SELECT_PAGES = 768;

template <int J, bool FEW>
__global__ void __launch_bounds__(select_threads(J, FEW))
select4_kernel(Select4 a, uint32_t stride)
{
	extern __shared__ uint32_t keys[]; /* [per][stride] */
	constexpr uint32_t THREADS = select_threads(J, FEW);
	__shared__ typename Scorer4<J>::Lds lds;
	__shared__ ChooseLds choose[8];
	__shared__ uint32_t above[THREADS / WAVE], equal[THREADS / WAVE];
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE;
	const uint32_t head = blockIdx.x, s = blockIdx.y, tile = blockIdx.z;
	const Sequence seq = sequence_of(a.batch, s, a.cache.page_shift);
	if (tile * a.per >= seq.queries) return;
	const uint32_t page_tokens = 1u << a.cache.page_shift, last_i = min(seq.queries, (tile + 1) * a.per) - 1;
	const uint32_t pages = (visible_to(a.batch, seq, last_i) + page_tokens - 1) >> a.cache.page_shift;
	if (pages > a.top) {
		Scorer4<J> scorer(a, seq, head, tile, lane);
		uint32_t* const mine = keys + (scorer.token_there ? (scorer.col >> a.span_bits) : 0) * stride;
		constexpr int TILES = THREADS == 512 ? 2 : 1;
		score_pages<J, TILES>(scorer, lds, a.batch.table + (size_t)s * a.batch.table_stride, 16 * TILES * wave, pages, pages, 16 * TILES * (THREADS / WAVE), THREADS,
		                      [&](uint32_t p) { return mine[p]; }, [&](uint32_t p, uint32_t k) { mine[p] = k; });
	}
	__syncthreads();
	const uint32_t threads = THREADS / a.per, list = threadIdx.x / threads, tid = threadIdx.x % threads, i = tile * a.per + list;
	const bool there = i < seq.queries;
	const uint32_t n = there ? (visible_to(a.batch, seq, i) + page_tokens - 1) >> a.cache.page_shift : 0;
	int32_t* out = there ? a.chosen + ((size_t)(seq.first + i) * a.cache.heads + head) * a.top : nullptr;
	const uint32_t* from = keys + list * stride;
	choose_top([&](uint32_t p) { return from[p]; }, n, a.top, out, tid, threads, choose[list], above + list * (threads / WAVE), equal + list * (threads / WAVE));
}

} // namespace kmx

using namespace kmx;

/* ---------------------------------------------------------------- entry points ------------------- */

static int check_cache4(const char* who, const kmx_cache4* cache, Cache4* out)
{
	if (!cache) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: null cache", who);
	if (cache->heads == 0) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: heads must be positive", who);
	if (cache->dim == 0 || cache->dim % 32 || cache->dim > 256) return fail(KMX_ERR_UNSUPPORTED, "%s: dim %u is not a multiple of 32 up to 256", who, cache->dim);
	const uint32_t p = cache->page_tokens;
	if (p < 16 || p > 256 || (p & (p - 1))) return fail(KMX_ERR_UNSUPPORTED, "%s: pages of %u tokens (16, 32, 64, 128 or 256)", who, p);
	uint32_t shift = 4;
	while ((1u << shift) < p) ++shift;
	if ((uint64_t)cache->page_count << shift > 0x7FFFFFFFu) return fail(KMX_ERR_UNSUPPORTED, "%s: %u pages of %u tokens are more places than 31 bits count", who, cache->page_count, p);
	if (out) {
		if (!cache->blocks || !cache->levels) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: null device pointer in the cache", who);
		if ((uintptr_t)cache->blocks % 16 || (uintptr_t)cache->levels % 16 || (uintptr_t)cache->bounds % 16)
			return fail(KMX_ERR_INVALID_ARGUMENT, "%s: the cache's buffers start at multiples of 16 bytes", who);
		const size_t codes = (size_t)cache->page_count * cache->heads * 2 * cache->dim;
		*out = Cache4{ (uint8_t*)cache->blocks, (int8_t*)cache->bounds, cache->bounds ? (float*)((int8_t*)cache->bounds + codes) : nullptr, cache->levels, cache->heads, cache->page_count, shift };
	}
	return KMX_OK;
}

static int check_type(const char* who, int type, bool floats)
{
	if (type == KMX_F16 || type == KMX_BF16 || (floats && type == KMX_F32)) return KMX_OK;
	if (type == KMX_F32) return fail(KMX_ERR_UNSUPPORTED, "%s: queries are KMX_F16 or KMX_BF16", who);
	return fail(KMX_ERR_INVALID_ARGUMENT, "%s: unknown element type %d", who, type);
}

static bool aligned_rows(const void* p, size_t token_stride, size_t head_stride, size_t size)
{
	return (uintptr_t)p % 16 == 0 && token_stride * size % 16 == 0 && head_stride * size % 16 == 0;
}

static int rows4(const char* who, bool write, const kmx_cache4* cache, int type, void* keys, void* values, size_t token_stride, size_t head_stride, const int32_t* slots, uint32_t tokens)
{
	Rows4 a{};
	int rc = check_cache4(who, cache, &a.cache);
	if (rc) return rc;
	rc = check_type(who, type, true);
	if (rc) return rc;
	if (tokens == 0) return KMX_OK;
	if (!keys || !values || !slots) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: null device pointer", who);
	if (!write && head_stride < cache->dim && cache->heads > 1) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: head stride %zu < dim %u", who, head_stride, cache->dim);
	if (!write && token_stride < cache->dim && tokens > 1) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: token stride %zu < dim %u", who, token_stride, cache->dim);
	if (cache->page_count == 0 && write) return KMX_OK; /* no place is in it */
	const size_t size = type == KMX_F32 ? 4 : 2;
	if ((uintptr_t)keys % size || (uintptr_t)values % size) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: rows start at multiples of their element's size", who);
	a.keys = keys;
	a.values = values;
	a.token_stride = token_stride;
	a.head_stride = head_stride;
	a.slots = slots;
	a.tokens = tokens;
	a.vec = aligned_rows(keys, token_stride, head_stride, size) && aligned_rows(values, token_stride, head_stride, size);
	const uint32_t J = cache->dim / 32;
	if (type == KMX_F32) return launch_rows4<float>(write, a, J);
	if (type == KMX_F16) return launch_rows4<_Float16>(write, a, J);
	return launch_rows4<__bf16>(write, a, J);
}

/* a bound may be as loose as it likes: no sequence has more queries than there are */
static uint32_t most_queries(const kmx_cache4_batch* b) { return b->max_queries < b->tokens ? b->max_queries : b->tokens; }

static int check_batch4(const char* who, const kmx_cache4* cache, const kmx_cache4_batch* batch, int causal, Batch4* out)
{
	if (!batch) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: null batch", who);
	if (batch->query_heads == 0 || batch->query_heads % cache->heads)
		return fail(KMX_ERR_INVALID_ARGUMENT, "%s: %u query heads are no multiple of the cache's %u", who, batch->query_heads, cache->heads);
	if (causal != 0 && causal != 1) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: causal is 0 or 1", who);
	if (batch->sequences && batch->tokens && batch->max_queries) {
		if (!batch->starts || !batch->lengths || (batch->table_stride && !batch->table)) return fail(KMX_ERR_INVALID_ARGUMENT, "%s: null device pointer in the batch", who);
		if (batch->max_length > 0x7FFFFFFFu || batch->tokens > 0x7FFFFFFFu) return fail(KMX_ERR_UNSUPPORTED, "%s: lengths and tokens are counted in 31 bits", who);
	}
	*out = Batch4{ batch->starts, batch->lengths, batch->table, batch->sequences, batch->tokens, most_queries(batch), batch->table_stride,
		       batch->max_length, batch->query_heads / cache->heads, batch->query_heads, causal != 0 };
	if (cache->page_count == 0) out->table_stride = 0; /* nothing is cached */
	return KMX_OK;
}

/*
 * Work space of a call. A recording keeps the addresses of its moment, and the work space moves when a later call needs more of it: recorded calls take the static
 * scratch array of recorded updates where it has room (64 MB: all attention of few rows, and choices of 16M scores), else the work space.
 */
static int place_cache4(const char* who, size_t floats, float** partials)
{
	const bool recorded = launches_recorded();
	const Workspace* fixed = recorded ? fixed_scratch() : nullptr;
	if (fixed && floats <= fixed->partials_cap) {
		*partials = fixed->partials;
		scratch_recorded();
		return KMX_OK;
	}
	Workspace* ws = nullptr;
	int rc = workspace(&ws);
	if (rc) return rc;
	if (recorded && floats > ws->partials_cap)
		return fail(KMX_ERR_INVALID_ARGUMENT, "%s: the call needs a larger work space, which cannot be allocated while it is recorded: kmx_cache4_reserve, or the same call once before", who);
	if (recorded) scratch_recorded();
	rc = reserve_partials(ws, floats);
	*partials = ws->partials;
	return rc;
}

/* the numbers of a call that decide how it is launched */
static Shape4 shape_of(const kmx_cache4* cache, const kmx_cache4_batch* b, uint32_t table_stride, uint32_t top, const DeviceInfo& dev)
{
	uint32_t shift = 4;
	while ((1u << shift) < cache->page_tokens) ++shift;
	const uint64_t most = (uint64_t)table_stride << shift;
	return Shape4{ cache->dim / 32, cache->heads, b->query_heads / cache->heads, b->sequences, most_queries(b), b->max_length < most ? b->max_length : (uint32_t)most, shift, top, dev.compute_units };
}

static uint32_t table_pages(const kmx_cache4_batch* b, uint32_t page_tokens)
{
	const uint32_t need = b->max_length / page_tokens + (b->max_length % page_tokens ? 1 : 0);
	return need < b->table_stride ? need : b->table_stride;
}

extern "C" {

int kmx_cache4_sizes(const kmx_cache4* cache, size_t* blocks, size_t* bounds)
{
	clear_error();
	int rc = check_cache4("kmx_cache4_sizes", cache, nullptr);
	if (rc) return rc;
	const size_t pages = (size_t)cache->page_count * cache->heads;
	if (blocks) *blocks = pages * (cache->page_tokens / 16) * 18 * cache->dim;
	if (bounds) *bounds = pages * (2 * cache->dim + 4);
	return KMX_OK;
}

int kmx_cache4_round_levels(const float* in, uint32_t sets, uint16_t* out)
{
	clear_error();
	if (sets == 0) return KMX_OK;
	if (!in || !out) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_round_levels: null pointer");
	for (uint32_t n = 0; n < sets; ++n) {
		for (int i = 0; i < 8; ++i) {
			const float v = in[8 * (size_t)n + i];
			if (!(v >= 0.0f && v <= 1.0f)) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_round_levels: level %d of set %u is not within 0 and 1", i, n);
			if (i && v < in[8 * (size_t)n + i - 1]) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_round_levels: set %u does not ascend at level %d", n, i);
			int power = 0;
			const float part = std::frexp(v, &power);
			/* 6 significant bits, fewer below 2^-14, where half precision has its last place at 2^-24 */
			const int place = power - 6 < -24 ? -24 : power - 6;
			const float rounded = std::ldexp(std::nearbyint(std::ldexp(part, power - place)), place);
			const _Float16 h = (_Float16)rounded;
			std::memcpy(out + 8 * (size_t)n + i, &h, 2);
		}
	}
	return KMX_OK;
}

int kmx_cache4_write(const kmx_cache4* cache, int type, const void* keys, const void* values, size_t token_stride, size_t head_stride, const int32_t* slots, uint32_t tokens)
{
	clear_error();
	return rows4("kmx_cache4_write", true, cache, type, (void*)keys, (void*)values, token_stride, head_stride, slots, tokens);
}

int kmx_cache4_read(const kmx_cache4* cache, int type, void* keys, void* values, size_t token_stride, size_t head_stride, const int32_t* slots, uint32_t tokens)
{
	clear_error();
	return rows4("kmx_cache4_read", false, cache, type, keys, values, token_stride, head_stride, slots, tokens);
}

int kmx_cache4_bound(const kmx_cache4* cache, const int32_t* pages, const int32_t* counts, uint32_t count)
{
	clear_error();
	Cache4 c;
	int rc = check_cache4("kmx_cache4_bound", cache, &c);
	if (rc) return rc;
	if (!cache->bounds) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_bound: the cache keeps no bounds");
	if (count == 0) return KMX_OK;
	if (!pages || !counts) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_bound: null device pointer");
	const uint32_t waves = cache->page_tokens >= 64 ? 4 : cache->page_tokens / 16;
	const uint64_t groups = ((uint64_t)count * c.heads + 4 / waves - 1) / (4 / waves);
	if (groups > 0x7FFFFFFFu) return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_bound: %u pages of %u heads are too many for one call", count, c.heads);
	switch (cache->dim / 32) {
#define KMX_CASE(N)                                                                                                      \
	case N: KMX_LAUNCH_KERNEL((bound4_kernel<N>), dim3((unsigned)groups), dim3(256), 0, stream(), c, pages, counts, count, waves); break;
		KMX_CASE(1) KMX_CASE(2) KMX_CASE(3) KMX_CASE(4) KMX_CASE(5) KMX_CASE(6) KMX_CASE(7) KMX_CASE(8)
#undef KMX_CASE
	}
	KMX_LAUNCH_CHECK("bound4_kernel");
	return KMX_OK;
}

int kmx_cache4_select(const kmx_cache4* cache, const kmx_cache4_batch* batch, int type, const void* q, size_t q_token_stride, size_t q_head_stride,
                      int32_t* chosen, uint32_t top, uint32_t first, uint32_t last, int causal)
{
	clear_error();
	Select4 a{};
	int rc = check_cache4("kmx_cache4_select", cache, &a.cache);
	if (rc) return rc;
	if (!cache->bounds) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_select: the cache keeps no bounds");
	rc = check_batch4("kmx_cache4_select", cache, batch, causal, &a.batch);
	if (rc) return rc;
	rc = check_type("kmx_cache4_select", type, false);
	if (rc) return rc;
	if (top == 0 || (uint64_t)first + last > top) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_select: top %u has no room for the %u first and %u last pages", top, first, last);
	if (batch->sequences == 0 || batch->tokens == 0 || batch->max_queries == 0) return KMX_OK;
	if (!q || !chosen) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_select: null device pointer");
	if ((uintptr_t)q % 2) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_select: queries start at multiples of 2 bytes");
	const uint32_t pages = table_pages(batch, cache->page_tokens);
	a.q = q;
	a.q_token = q_token_stride;
	a.q_head = q_head_stride;
	a.chosen = chosen;
	a.top = top;
	a.first = first;
	a.last = last;
	a.bf16 = type == KMX_BF16;
	a.vec = aligned_rows(q, q_token_stride, q_head_stride, 2);
	a.span = 1;
	while (a.span < a.batch.group && a.span < 16) { a.span *= 2; ++a.span_bits; }
	/* Scores and choice in one kernel where the pages are few, by 4 wavefronts or by 16 (64 sequences of 128 pages: 65 us by 16, 57 in two kernels; two
	 * sequences of 625 pages, 128 queries: 37 us against 41); two kernels where one work-group would read for long (1 x 1024 pages: 29 us against 34) */
	const bool one = pages <= SELECT_PAGES, few = pages <= SELECT_FEW;
	a.per = 1;
	while (a.per < a.batch.max_queries && a.per < (one && few ? 4 : 8) && a.per * a.span < 16) a.per *= 2;
	a.token_tiles = (a.batch.max_queries + a.per - 1) / a.per;
	const uint64_t units = (uint64_t)batch->sequences * a.token_tiles * a.cache.heads;
	if (batch->sequences > 65535 || a.batch.max_queries > 65535)
		return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_select: %u sequences of %u queries are too many for one call", batch->sequences, a.batch.max_queries);
	if (one) {
		const uint32_t stride = pages | 1, bytes = 4 * a.per * stride; /* at most 24.6 KB */
		switch (cache->dim / 32) {
#define KMX_CASE(N)                                                                                                      \
	case N:                                                                                                               \
		if (few) KMX_LAUNCH_KERNEL((select4_kernel<N, true>), dim3(a.cache.heads, batch->sequences, a.token_tiles), dim3(select_threads(N, true)), bytes, stream(), a, stride); \
		else KMX_LAUNCH_KERNEL((select4_kernel<N, false>), dim3(a.cache.heads, batch->sequences, a.token_tiles), dim3(select_threads(N, false)), bytes, stream(), a, stride); \
		break;
			KMX_CASE(1) KMX_CASE(2) KMX_CASE(3) KMX_CASE(4) KMX_CASE(5) KMX_CASE(6) KMX_CASE(7) KMX_CASE(8)
#undef KMX_CASE
		}
		KMX_LAUNCH_CHECK("select4_kernel");
		return KMX_OK;
	}
	/* parts of the pages: enough work-groups to fill the chip, of 128 pages at least */
	const uint32_t tiles = (pages + 63) / 64; /* of 16 pages a wavefront */
	uint64_t parts = (1024 + units - 1) / units;
	if (parts > (tiles + 1) / 2) parts = (tiles + 1) / 2;
	a.chunk = (uint32_t)((tiles + parts - 1) / parts);
	a.chunks = (tiles + a.chunk - 1) / a.chunk;
	if ((uint64_t)a.token_tiles * a.chunks > 65535) return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_select: %u queries are too many for one call", a.batch.max_queries);
	float* keys = nullptr;
	rc = place_cache4("kmx_cache4_select", (size_t)batch->tokens * a.cache.heads * batch->table_stride, &keys);
	if (rc) return rc;
	a.keys = (uint32_t*)keys;
	switch (cache->dim / 32) {
#define KMX_CASE(N)                                                                                                      \
	case N: KMX_LAUNCH_KERNEL((score4_kernel<N>), dim3(a.cache.heads, batch->sequences, a.token_tiles * a.chunks), dim3(256), 0, stream(), a); break;
		KMX_CASE(1) KMX_CASE(2) KMX_CASE(3) KMX_CASE(4) KMX_CASE(5) KMX_CASE(6) KMX_CASE(7) KMX_CASE(8)
#undef KMX_CASE
	}
	KMX_LAUNCH_CHECK("score4_kernel");
	KMX_LAUNCH_KERNEL(choose4_kernel, dim3(a.cache.heads, batch->sequences, a.batch.max_queries), dim3(512), 0, stream(), a);
	KMX_LAUNCH_CHECK("choose4_kernel");
	return KMX_OK;
}

int kmx_cache4_attend(const kmx_cache4* cache, const kmx_cache4_batch* batch, int type, const void* q, size_t q_token_stride, size_t q_head_stride,
                      void* out, size_t out_token_stride, size_t out_head_stride, float* lse, float scale, int causal, const int32_t* chosen, uint32_t top)
{
	clear_error();
	Attend4 a{};
	int rc = check_cache4("kmx_cache4_attend", cache, &a.cache);
	if (rc) return rc;
	rc = check_batch4("kmx_cache4_attend", cache, batch, causal, &a.batch);
	if (rc) return rc;
	rc = check_type("kmx_cache4_attend", type, false);
	if (rc) return rc;
	if (chosen && top == 0) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_attend: chosen pages, but top is 0");
	if (!(std::fabs(scale) <= 3.4e38f)) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_attend: the scale is not finite");
	if (batch->sequences == 0 || batch->tokens == 0 || batch->max_queries == 0) return KMX_OK;
	if (!q || !out) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_attend: null device pointer");
	if ((uintptr_t)q % 2 || (uintptr_t)out % 2) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_attend: rows start at multiples of 2 bytes");
	if (batch->query_heads > 1 && out_head_stride < cache->dim) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_attend: head stride of the output %zu < dim %u", out_head_stride, cache->dim);
	if (batch->tokens > 1 && out_token_stride < cache->dim) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_attend: token stride of the output %zu < dim %u", out_token_stride, cache->dim);
	a.q = q;
	a.q_token = q_token_stride;
	a.q_head = q_head_stride;
	a.out = out;
	a.out_token = out_token_stride;
	a.out_head = out_head_stride;
	a.lse = lse;
	a.chosen = chosen;
	a.top = chosen ? top : 0;
	a.scale = scale;
	a.bf16 = type == KMX_BF16;
	a.vec = aligned_rows(q, q_token_stride, q_head_stride, 2) && aligned_rows(out, out_token_stride, out_head_stride, 2);
	const DeviceInfo* dev = nullptr;
	rc = device_info(&dev);
	if (rc) return rc;
	const Plan4 plan = plan_attend4(shape_of(cache, batch, a.batch.table_stride, a.top, *dev));
	if (plan.units >= MOST_UNITS) return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_attend: too many queries for one call");
	const size_t floats = plan_floats(plan, cache->dim / 32);
	if (floats) {
		rc = place_cache4("kmx_cache4_attend", floats, &a.partial);
		if (rc) return rc;
	}
	switch (cache->dim / 32) {
	case 1: return launch_attend4<1>(a, plan);
	case 2: return launch_attend4<2>(a, plan);
	case 3: return launch_attend4<3>(a, plan);
	case 4: return launch_attend4<4>(a, plan);
	case 5: return launch_attend4<5>(a, plan);
	case 6: return launch_attend4<6>(a, plan);
	case 7: return launch_attend4<7>(a, plan);
	default: return launch_attend4<8>(a, plan);
	}
}

int kmx_cache4_reserve(const kmx_cache4* cache, const kmx_cache4_batch* batch, uint32_t top)
{
	clear_error();
	if (recording_graph()) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_reserve: not allowed between kmx_graph_begin and kmx_graph_end");
	int rc = check_cache4("kmx_cache4_reserve", cache, nullptr);
	if (rc) return rc;
	if (!batch) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_reserve: null batch");
	if (batch->query_heads == 0 || batch->query_heads % cache->heads)
		return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_reserve: %u query heads are no multiple of the cache's %u", batch->query_heads, cache->heads);
	const DeviceInfo* dev = nullptr;
	rc = device_info(&dev);
	if (rc) return rc;
	size_t floats = most_floats(shape_of(cache, batch, batch->table_stride, top, *dev));
	if (top && table_pages(batch, cache->page_tokens) > SELECT_PAGES) { /* scores of the choice in two kernels */
		const size_t keys = (size_t)batch->tokens * cache->heads * batch->table_stride;
		if (keys > floats) floats = keys;
	}
	Workspace* scratch = nullptr;
	if (noalloc_workspace(&scratch)) clear_error(); /* the address of the scratch array that recorded calls use (they do without if it has none) */
	float* partials = nullptr;
	return floats ? place_cache4("kmx_cache4_reserve", floats, &partials) : KMX_OK;
}

} // extern "C"
