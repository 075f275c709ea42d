/*
 * Attention over the 4-bit cache, kernels for J groups of 32 channels (one object per J: cache4_attend_inst.hip).
 *
 * For a row r (a query head of a token) that sees the tokens t < vis:  o_r = sum_t p_rt v_t / l_r,  p_rt = 2^(s_rt - m_r),
 * s_rt = scale log2(e) q_r . k_t,  m_r = max_t s_rt,  l_r = sum_t p_rt;  lse_r = ln 2 (m_r + log2 l_r). One pass over the cache with the running
 * maximum and sum; parts of the tokens (wavefronts, and work-groups where there are few rows) are joined at the end. (The kernels keep p and l times 2^15.)
 */
#ifndef KMX_CACHE4_ATTEND_IMPL_H
#define KMX_CACHE4_ATTEND_IMPL_H

#include "cache4.h"

#include <type_traits>

namespace kmx {

/* 2^v by the instruction: results below 2^-126 are 0, which no sum here notices */
__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }

/* parts done of each unit of a call, zero between calls: in the code's own memory, so that no call allocates or clears it */
static __device__ uint32_t tickets[TICKETS];

struct Row4 { uint32_t token, head; bool there; }; /* query number inside its sequence, query head inside its group */

/* (divisions are some twenty instructions and come before the first load: none where a sequence has one query) */
__device__ __forceinline__ Row4 row_of(const Attend4& a, const Sequence& seq, uint32_t row_tile, uint32_t r)
{
	Row4 row;
	if (a.batch.max_queries == 1) {
		row.token = 0;
		row.head = row_tile * 16 + r;
		row.there = seq.queries && row.head < a.batch.group;
	} else if (a.chosen) { /* the tokens' pages differ: a tile has rows of one token */
		const uint32_t tiles = (a.batch.group + 15) / 16;
		row.token = row_tile / tiles;
		row.head = row_tile % tiles * 16 + r;
		row.there = row.token < seq.queries && row.head < a.batch.group;
	} else { /* (at most MANY_ROWS of them) */
		const uint32_t x = row_tile * 16 + r;
		row.token = x / a.batch.group;
		row.head = x % a.batch.group;
		row.there = row.token < seq.queries;
	}
	return row;
}

/* rows of a tile that are there: the first ones */
__device__ __forceinline__ uint32_t rows_of(const Attend4& a, const Sequence& seq, uint32_t row_tile)
{
	if (a.chosen) return min(16u, a.batch.group - row_tile % ((a.batch.group + 15) / 16) * 16);
	const uint32_t rows = seq.queries * a.batch.group, first = row_tile * 16;
	return first < rows ? min(16u, rows - first) : 0;
}

/* the query of a tile's rows that sees the most */
__device__ __forceinline__ uint32_t last_query_of(const Attend4& a, const Sequence& seq, uint32_t row_tile)
{
	if (a.batch.max_queries == 1) return 0;
	return a.chosen ? row_tile / ((a.batch.group + 15) / 16) : min(seq.queries - 1, (row_tile * 16 + 15) / a.batch.group);
}

__device__ __forceinline__ uint64_t pair_of(float x, float y) { return (uint64_t)__builtin_bit_cast(uint32_t, y) << 32 | __builtin_bit_cast(uint32_t, x); }

/* tiles of 64 tokens that a tile of rows looks at */
__device__ __forceinline__ uint32_t tiles_of(const Attend4& a, const Sequence& seq, uint32_t row_tile)
{
	if (!a.chosen && row_tile * 16 >= seq.queries * a.batch.group) return 0;
	const uint32_t query = last_query_of(a, seq, row_tile);
	if (query >= seq.queries) return 0;
	const uint32_t sees = visible_to(a.batch, seq, query);
	if (!a.chosen) return (sees + 63) / 64;
	/* lists ascend: pages with a token that the query sees come first, and there are no more of them than the sequence has */
	const uint32_t pages = (sees + (1u << a.cache.page_shift) - 1) >> a.cache.page_shift;
	return (uint32_t)((((uint64_t)min(a.top, pages) << (a.cache.page_shift - 4)) + 3) / 4);
}

template <int J>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t w[J])
{
	if constexpr (J % 4 == 0) {
		for (int i = 0; i < J / 4; ++i) { const u32x4 v = ((const u32x4*)p)[i]; for (int e = 0; e < 4; ++e) w[4 * i + e] = v[e]; }
	} else if constexpr (J % 2 == 0) {
		for (int i = 0; i < J / 2; ++i) { const u32x2 v = ((const u32x2*)p)[i]; w[2 * i] = v[0]; w[2 * i + 1] = v[1]; }
	} else {
		for (int i = 0; i < J; ++i) w[i] = ((const uint32_t*)p)[i];
	}
}

/* J halves, two a word */
template <int J>
__device__ __forceinline__ void load_halves(const uint8_t* p, uint32_t w[(J + 1) / 2])
{
	if constexpr (J % 8 == 0) {
		const u32x4 v = *(const u32x4*)p;
		for (int e = 0; e < 4; ++e) w[e] = v[e];
	} else if constexpr (J % 4 == 0) {
		const u32x2 v = *(const u32x2*)p;
		w[0] = v[0];
		w[1] = v[1];
	} else if constexpr (J % 2 == 0) {
		for (int i = 0; i < J / 2; ++i) w[i] = ((const uint32_t*)p)[i];
	} else {
		for (int i = 0; i < (J + 1) / 2; ++i) {
			w[i] = ((const uint16_t*)p)[2 * i];
			if (2 * i + 1 < J) w[i] |= (uint32_t)((const uint16_t*)p)[2 * i + 1] << 16;
		}
	}
}

/* N pieces of 8 channels of a row, `apart` channels from one to the next */
template <int N>
__device__ __forceinline__ void load_pieces(const uint16_t* p, uint32_t apart, bool vec, u32x4 raw[N])
{
	if (vec) {
#pragma unroll
		for (int n = 0; n < N; ++n) raw[n] = load_raw8(p + apart * n, true);
	} else {
#pragma unroll
		for (int n = 0; n < N; ++n) raw[n] = load_raw8(p + apart * n, false);
	}
}
template <int N>
__device__ __forceinline__ void floats_of(const u32x4 raw[N], bool bf16, float x[N][8])
{
	if (bf16) {
#pragma unroll
		for (int n = 0; n < N; ++n)
			for (int e = 0; e < 8; ++e) { const uint32_t w = raw[n][e / 2]; x[n][e] = raw_element(w, e % 2, true); }
	} else {
#pragma unroll
		for (int n = 0; n < N; ++n)
			for (int e = 0; e < 8; ++e) { const uint32_t w = raw[n][e / 2]; x[n][e] = raw_element(w, e % 2, false); }
	}
}

template <int J>
constexpr int values_words() { return J > 4 * ((J + 3) / 4) ? J : 4 * ((J + 3) / 4); } /* words of codes a lane holds: J of keys, or 4 for each of its pairs of channels */

/* What queries of that largest magnitude are multiplied with to become halves of at most 2 in magnitude (bf16 has more exponents), with the sign
 * of the scale; *row_scale takes a score of theirs, below 2^26, to the exponent of 2, which stays a number: at most 2^100, where any two scores that
 * differ do so by far more than a softmax tells from infinity */
__device__ __forceinline__ float query_scale(float scale, float largest, float* row_scale)
{
	int power = (int)(__builtin_bit_cast(uint32_t, largest) >> 23) - 127;
	power = power < -126 ? -126 : power > 126 ? 126 : power; /* (queries below 2^-126 too) */
	const float by = __builtin_bit_cast(float, (uint32_t)(127 - power) << 23);
	*row_scale = fminf(fmaxf(fabsf(scale) * 1.44269504088896341f * __builtin_bit_cast(float, (uint32_t)(127 + power) << 23), 1.2e-38f), 0x1p100f);
	return scale > 0.0f ? by : scale < 0.0f ? -by : 0.0f;
}

/*
 * Probabilities are rounded to half precision for their product with the values: 11 bits from 2^-14 on, none below 2^-25. They are taken times 2^15, so
 * that the largest is as large as half precision allows for: then 11 bits reach down to 2^-29 of it and the last one to 2^-39, and what all
 * tokens of a long row add up to below one that stands far out is there. Sums are of the same size; only lse takes the factor off.
 */
constexpr float RAISE = 15.0f, LOWERED = 0x1p-15f;

/*
 * What is added to row_scale times the scores so that the largest, m, becomes RAISE. One fused operation a score, whose error is that of m row_scale,
 * 2^-24 of it: in rows where that is no longer small the scores give m up themselves, exactly at the largest. Whether a row of the wavefront is
 * such a one is found where a maximum rises (found for each tile: 533 us of the many-rows kernel in place of 524; see also EXACT there).
 */
constexpr float FAR_SCORE = 1024.0f;
__device__ __forceinline__ bool far_score(float m, float row_scale) { return m != -__builtin_inff() && fabsf(m * row_scale) > FAR_SCORE; } /* (-inf: nothing seen yet) */
template <typename LOWER>
__device__ __forceinline__ float below_most(float m, float row_scale, bool any_far, const LOWER& lower)
{
	float base = m == -__builtin_inff() ? RAISE : fmaf(-m, row_scale, RAISE);
	if (any_far) {
		const bool far = far_score(m, row_scale);
		lower(far ? m : 0.0f);
		base = far ? RAISE : base;
	}
	return base;
}

/* 4 channels of an output row */
__device__ __forceinline__ void store_out4(const Attend4& a, char* row, uint32_t channel, const float v[4])
{
	uint32_t b[4];
	for (int i = 0; i < 4; ++i) b[i] = a.bf16 ? bf16_bits(v[i]) : bits16<_Float16>(v[i]);
	if (a.vec) *(u32x2*)(row + 2 * channel) = u32x2{ b[0] | b[1] << 16, b[2] | b[3] << 16 };
	else
		for (int i = 0; i < 4; ++i) ((uint16_t*)row)[channel + i] = (uint16_t)b[i];
}

/* What a wavefront loads for 64 tokens. A lane is row i = lane % 16 of the operands and holds their piece kg = lane / 16. */
template <int J>
struct Tile4 {
	uint32_t kc[4][J];        /* codes of token 4 u + i % 4 of block i / 4, channels 32 j + 8 kg .. + 7 */
	u32x4 vc[J];              /* codes of channels 32 j + i and + 16 + i, the 16 tokens of block kg */
	u32x4 sc[(J + 3) / 4];    /* 16 bytes of the 64 J of the scales of block kg, which go through LDS to the lanes that need them */
};

/*
 * A work-group of four wavefronts takes 16 rows of one head of the cache (the query heads of a token side by side, then the next token's) and
 * a part of the tokens; a wavefront takes every fourth tile of 64 tokens. The registers of a tile's keys are loaded with the next tile's as soon as
 * the scores are there, those of its values as soon as the sums are: each load has the other half of a tile's work to arrive in, and three
 * wavefronts fit a SIMD (two above 128 channels). Both products have the cache as their first operand (v_mfma_f32_16x16x32_f16): scores come out as
 * [token][row], so a lane has all its 16 scores in one row -- maxima and sums are its own but for two exchanges -- and its probabilities are, as they
 * stand, its piece of the second operand of [channel][row] = values . p. Tokens go to the rows of the first product such that a lane's 16 are those
 * of one block: its values are 16 bytes side by side.
 * Bound by unpacking: some 760 vector instructions a tile of 64 tokens at 128 channels, 1.4 us a tile and SIMD, about what the memory takes for it (72 % of the
 * vector units' time in all, where lengths differ and the longest sequences end alone; matrix cores 12 %). 64
 * sequences of 8192 tokens, 8 heads of 128: 124 us, 4.8 TB/s of packed bytes; the same of 1 to 8192 tokens 102 to 107 us, where the longest ones
 * end last. Short sequences: 7 to 9 us, of which 4.5 are a launch with its first load and last store, the rest loads that wait for each other
 * (length, table, codes).
 */
template <int J>
__global__ void __launch_bounds__(256, J <= 4 ? 3 : 2)
attend4_kernel(Attend4 a)
{
	constexpr uint32_t D = 32 * J, SCALES = 64 * J + 32; /* bytes of a block's scales in LDS: 8 banks on from one block to the next */
	__shared__ union {
		struct {
			__attribute__((aligned(16))) uint8_t scales[4][4][SCALES];
			uint64_t places[4][2][WAVE];
			int32_t from[4][2][WAVE];
		};
		f32x4 sums[2][2 * J][WAVE];
		float weights[MOST_PARTS][16]; /* of the parts of the rows */
	} lds;
	__shared__ f32x4 shares[256];
	__shared__ bool last;
	__shared__ float most[4][16], total[4][16];
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE, i16 = lane % 16, kg = lane / 16;
	/* first parts of all units before their second ones: the dies take work-groups in turn, and parts behind the end of a shorter sequence are empty */
	const uint32_t head = blockIdx.x, s = blockIdx.y, part = a.row_tiles == 1 ? blockIdx.z : blockIdx.z / a.row_tiles, row_tile = blockIdx.z - part * a.row_tiles;
	const uint32_t whole = (s * a.cache.heads + head) * a.row_tiles + row_tile; /* (counts work-groups: 31 bits) */
	const Sequence seq = sequence_of(a.batch, s, a.cache.page_shift);
	const uint32_t tiles = tiles_of(a, seq, row_tile);
	const uint32_t begin = part * a.tiles_per_split, end = min(tiles, begin + a.tiles_per_split);
	if (part > 0 && begin >= tiles) return;
	const uint32_t parts = tiles > a.tiles_per_split ? (tiles + a.tiles_per_split - 1) / a.tiles_per_split : 1;
	const Row4 row = row_of(a, seq, row_tile, i16);
	if (seq.queries == 0) return; /* no rows */

	/* queries: 8 channels a lane for each j; on their way while the first tile's pages are looked up, put to use while that tile is on its way */
	u32x4 raw[J];
	{
		const uint16_t* p = (const uint16_t*)a.q + (size_t)(seq.first + (row.there ? row.token : 0)) * a.q_token + ((size_t)head * a.batch.group + (row.there ? row.head : 0)) * a.q_head + 8 * kg;
		load_pieces<J>(p, 32, a.vec, raw);
	}
	const int32_t sees = row.there ? (int32_t)visible_to(a.batch, seq, row.token) : 0;
	const Magnitudes mk = load_magnitudes(a.cache.levels, head, 0), mv = load_magnitudes(a.cache.levels, head, 1);
	const bool listed = a.chosen != nullptr;
	const int32_t* list = a.chosen + (listed ? ((size_t)(seq.first + last_query_of(a, seq, row_tile)) * a.cache.heads + head) * a.top : 0);
	const int32_t* table = a.batch.table + (size_t)s * a.batch.table_stride;
	const uint32_t sub_bits = a.cache.page_shift - 4, last_entry = (listed ? a.top : a.batch.table_stride) - 1;
	const uint32_t last_page = (seq.length - 1) >> a.cache.page_shift; /* (looked at where there is a token) places on pages behind it may not fit 32 bits */

	/*
	 * Where the blocks of the wavefront's tiles lie, 16 tiles at a time, one block a lane (4 n + b: block b of the n-th tile), and their places in
	 * the sequence (INT32_MAX: it is not there, and any block's address stands in its place). They are kept in LDS, in halves that take turns.
	 */
	auto find_places = [&](uint32_t first_tile, uint32_t half) {
		const uint32_t n = 4 * (first_tile + lane / 4 * 4) + lane % 4, entry = n >> sub_bits, sub = n & ((1u << sub_bits) - 1);
		uint32_t logical = min(entry, last_entry);
		if (listed) logical = (uint32_t)list[logical];
		const uint32_t page = (uint32_t)table[min(logical, a.batch.table_stride - 1)];
		const bool there = entry <= last_entry && logical <= last_page && page < a.cache.page_count;
		lds.places[wave][half][lane] = block_offset<J>(a.cache, there ? page : 0, head, sub);
		lds.from[wave][half][lane] = there ? (int32_t)((logical << a.cache.page_shift) + 16 * sub) : INT32_MAX;
	};
	struct Where { const uint8_t* keys; const uint8_t* values; int32_t from; };
	auto where = [&](uint32_t n) {
		const uint64_t* at = &lds.places[wave][n / 16 % 2][4 * (n % 16)];
		Where w;
		w.keys = a.cache.blocks + at[i16 / 4] + (i16 % 4) * (D / 2) + kg * 4 * J;
		w.values = a.cache.blocks + at[kg] + 8 * D + i16 * 16;
		w.from = lds.from[wave][n / 16 % 2][4 * (n % 16) + kg];
		return w;
	};
	auto fetch_keys = [&](Tile4<J>& t, const Where& w) {
#pragma unroll
		for (int u = 0; u < 4; ++u) load_words<J>(w.keys + u * (2 * D), t.kc[u]);
	};
	auto fetch_values = [&](Tile4<J>& t, const Where& w) {
#pragma unroll
		for (int j = 0; j < J; ++j) t.vc[j] = *(const u32x4*)(w.values + 256 * j);
	};
	auto fetch_scales = [&](Tile4<J>& t, const Where& w) {
#pragma unroll
		for (int n = 0; n < (J + 3) / 4; ++n)
			if (4 * J - 16 * n >= 16 || (int)i16 < 4 * J - 16 * n) t.sc[n] = *(const u32x4*)(w.values + 8 * D + 256 * n);
	};

	float m = -__builtin_inff(), l = 0.0f; /* of the lane's row: the maximum of all its lanes, the sum of the lane's own tokens */
	bool any_far = false; /* rows of the wavefront with scores far from zero */
	f32x4 o[2 * J];
#pragma unroll
	for (int c = 0; c < 2 * J; ++c) o[c] = f32x4{ 0.0f, 0.0f, 0.0f, 0.0f };

	half8v q[J];
	float row_scale = 1.0f;
	auto take_queries = [&]() {
		float x[J][8], largest = 0.0f;
		floats_of<J>(raw, a.bf16, x);
#pragma unroll
		for (int j = 0; j < J; ++j)
			for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(x[j][e]));
		largest = fmaxf(largest, __shfl_xor(largest, 16));
		largest = fmaxf(largest, __shfl_xor(largest, 32));
		const float by = query_scale(a.scale, largest, &row_scale);
#pragma unroll
		for (int j = 0; j < J; ++j)
			for (int e = 0; e < 8; ++e) q[j][e] = (_Float16)(x[j][e] * by);
	};

	auto work = [&](Tile4<J>& t, int32_t from, const Where& next) { /* ... and leaves the next tile's loads under way */
		const int32_t limit = from == INT32_MAX ? 0 : sees - from; /* tokens of the lane's block that its row sees */
		uint8_t* const scales = lds.scales[wave][0]; /* (a wavefront's own: LDS takes its accesses in their order) */
		/* what lies behind the last token may hold anything: the scales of its values become zeros */
		const int32_t written = from == INT32_MAX ? 0 : (int32_t)seq.length - from;
		const bool cut = __any(written < 16);
#pragma unroll
		for (int n = 0; n < (J + 3) / 4; ++n)
			if (4 * J - 16 * n >= 16 || (int)i16 < 4 * J - 16 * n) {
				if (cut && (int)i16 + 16 * n >= 2 * J) { /* scales of values: 8 tokens */
#pragma unroll
					for (int d = 0; d < 4; ++d) {
						const int first = 8 * ((int)i16 & 1) + 2 * d;
						t.sc[n][d] &= written >= first + 2 ? 0xFFFFFFFFu : written == first + 1 ? 0xFFFFu : 0u;
					}
				}
				*(u32x4*)(scales + kg * SCALES + 256 * n + 16 * i16) = t.sc[n];
			}
		wave_sync();
		fetch_scales(t, next);
		float sc[16];
#pragma unroll
		for (int u = 0; u < 4; ++u) {
			uint32_t ks[(J + 1) / 2];
			load_halves<J>(scales + (i16 / 4) * SCALES + (4 * u + i16 % 4) * 2 * J, ks);
			f32x4 acc{ 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
			for (int j = 0; j < J; ++j) {
				const uint32_t scale = twice(ks[j / 2], j % 2);
				u32x4 w;
				uint32_t p[4];
				unpack4<false>(t.kc[u][j], mk, p[0], p[1]);
				unpack4<true>(t.kc[u][j], mk, p[2], p[3]);
				for (int e = 0; e < 4; ++e) w[e] = times(p[e], scale);
				acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, w), q[j], acc, 0, 0, 0);
			}
			for (int r = 0; r < 4; ++r) sc[4 * u + r] = acc[r];
		}
		fetch_keys(t, next);
		if (__any(limit < 16)) {
#pragma unroll
			for (int e = 0; e < 16; ++e) sc[e] = e < limit ? sc[e] : -__builtin_inff();
		}
		float top = sc[0];
#pragma unroll
		for (int e = 1; e < 16; ++e) top = fmaxf(top, sc[e]);
		top = fmaxf(top, __shfl_xor(top, 16));
		top = fmaxf(top, __shfl_xor(top, 32));
		const float now = fmaxf(m, top);
		if (__any(now > m)) {
			const float less = m == now ? 1.0f : exp2_((m - now) * row_scale); /* (both -inf: nothing seen yet) */
			l *= less;
#pragma unroll
			for (int c = 0; c < 2 * J; ++c) o[c] *= less;
			m = now;
			any_far = __any(far_score(m, row_scale));
		}
		const float base = below_most(m, row_scale, any_far, [&](float most) {
#pragma unroll
			for (int e = 0; e < 16; ++e) sc[e] -= most;
		});
		half8v p[2];
#pragma unroll
		for (int e = 0; e < 16; ++e) {
			const float v = exp2_(fmaf(sc[e], row_scale, base));
			l += v;
			p[e / 8][e % 8] = (_Float16)v; /* (the sum is that of the floats: see RAISE) */
		}
#pragma unroll
		for (int j = 0; j < J; ++j) {
#pragma unroll
			for (int half = 0; half < 2; ++half) { /* tokens 0 to 7 of the lane's block, then 8 to 15 */
				const u32x4 vs = *(const u32x4*)(scales + kg * SCALES + 32 * J + 32 * j + 16 * half);
				u32x4 low, high;
				for (int d = 0; d < 2; ++d) {
					uint32_t x, y;
					const uint32_t code = t.vc[j][2 * half + d];
					unpack4<false>(code, mv, x, y);
					low[2 * d] = times(x, vs[2 * d]);
					low[2 * d + 1] = times(y, vs[2 * d + 1]);
					unpack4<true>(code, mv, x, y);
					high[2 * d] = times(x, vs[2 * d]);
					high[2 * d + 1] = times(y, vs[2 * d + 1]);
				}
				o[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, low), p[half], o[2 * j], 0, 0, 0);
				o[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, high), p[half], o[2 * j + 1], 0, 0, 0);
			}
		}
		fetch_values(t, next);
	};

	const uint32_t count = end > begin + wave ? (end - begin - wave + 3) / 4 : 0; /* tiles of this wavefront */
	if (count) {
		Tile4<J> t;
		const uint32_t tile0 = begin + wave;
		find_places(tile0, 0);
		wave_sync();
		Where w = where(0);
		fetch_scales(t, w);
		fetch_keys(t, w);
		fetch_values(t, w);
		take_queries();
		for (uint32_t n = 0; n < count; ++n) {
			const int32_t from = w.from;
			if (n % 16 == 7 && n + 9 < count) find_places(tile0 + 4 * (n + 9), (n + 9) / 16 % 2);
			wave_sync();
			w = where(min(n + 1, count - 1)); /* (the last tile is fetched twice: a fetch under a condition would make the compiler wait for everything) */
			work(t, from, w);
		}
	}

	/* the four wavefronts' parts */
	l += __shfl_xor(l, 16);
	l += __shfl_xor(l, 32);
	if (kg == 0) { most[wave][i16] = m; total[wave][i16] = l; }
	__syncthreads(); /* (from here on LDS holds sums) */
	float all = most[0][i16];
	for (int w = 1; w < 4; ++w) all = fmaxf(all, most[w][i16]);
	const float base = all == -__builtin_inff() ? 0.0f : all;
	const float mine = exp2_((m - base) * row_scale);
	float sum = 0.0f;
	for (int w = 0; w < 4; ++w) sum += total[w][i16] * exp2_((most[w][i16] - base) * row_scale);
#pragma unroll
	for (int c = 0; c < 2 * J; ++c) o[c] *= mine;
	if (wave >= 2)
#pragma unroll
		for (int c = 0; c < 2 * J; ++c) lds.sums[wave - 2][c][lane] = o[c];
	__syncthreads();
	if (wave < 2)
#pragma unroll
		for (int c = 0; c < 2 * J; ++c) o[c] += lds.sums[wave][c][lane];
	__syncthreads();
	if (wave == 1)
#pragma unroll
		for (int c = 0; c < 2 * J; ++c) lds.sums[0][c][lane] = o[c];
	__syncthreads();
	if (wave == 0) {
#pragma unroll
		for (int c = 0; c < 2 * J; ++c) o[c] += lds.sums[0][c][lane];
	}
	if (parts == 1) {
		if (wave != 0 || !row.there) return;
		const float by = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum; /* a row that sees nothing is zero; NaN stays */
		const size_t token = seq.first + row.token, query_head = (size_t)head * a.batch.group + row.head;
		char* to = (char*)a.out + 2 * (token * a.out_token + query_head * a.out_head);
#pragma unroll
		for (int c = 0; c < 2 * J; ++c) {
			float v[4];
			for (int r = 0; r < 4; ++r) v[r] = o[c][r] * by;
			store_out4(a, to, 16 * c + 4 * kg, v);
		}
		if (kg == 0 && a.lse) a.lse[token * a.batch.query_heads + query_head] = sum == 0.0f ? -__builtin_inff() : (all * row_scale + log2f(sum * LOWERED)) * 0.693147180559945309f;
		return;
	}

	/*
	 * The parts of the rows: each work-group leaves its sums, and the last one to do so joins them, in their order. Stores of device scope pass
	 * the L2 of the die by, so a part is there for everybody once they have completed.
	 */
	uint64_t* const all_parts = (uint64_t*)a.partial + (size_t)whole * a.splits * (16 * (D / 2 + 1)); /* [part]: [16][D / 2] pairs, [16] of maximum and sum */
	const uint32_t rows = rows_of(a, seq, row_tile);
	if (wave == 0 && row.there) {
		uint64_t* to = all_parts + (size_t)part * (16 * (D / 2 + 1));
#pragma unroll
		for (int c = 0; c < 2 * J; ++c)
			for (int h = 0; h < 2; ++h)
				__hip_atomic_store(to + i16 * (D / 2) + 8 * c + 2 * kg + h, pair_of(o[c][2 * h], o[c][2 * h + 1]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
		if (kg == 0) __hip_atomic_store(to + 16 * (D / 2) + i16, pair_of(all * row_scale, sum), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
	}
	asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
	__syncthreads();
	const uint32_t tid = threadIdx.x;
	if (tid == 0) last = atomicAdd(&tickets[whole], 1u) == parts - 1;
	__syncthreads();
	if (!last) return;
	__builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent"); /* (nothing below is read ahead of the ticket, nor from a cache that was filled before it) */
	if (tid == 0) __hip_atomic_store(&tickets[whole], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); /* for the next call */
	const float* const left = (const float*)all_parts;
	constexpr size_t PART = 2 * 16 * (D / 2 + 1);
	{ /* weights: 16 lanes a row, all their parts under way at once */
		constexpr uint32_t EACH = MOST_PARTS / 16;
		const uint32_t r = tid / 16, from = tid % 16;
		float2 v[EACH];
		float top = -__builtin_inff(), s1 = 0.0f;
#pragma unroll
		for (uint32_t u = 0; u < EACH; ++u) {
			v[u] = float2{ -__builtin_inff(), 0.0f };
			if (from + 16 * u < parts && r < rows) v[u] = *(const float2*)(left + (from + 16 * u) * PART + 16 * D + 2 * r);
		}
#pragma unroll
		for (uint32_t u = 0; u < EACH; ++u) top = fmaxf(top, v[u].x);
		for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
		const float lowest = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
		for (uint32_t u = 0; u < EACH; ++u) {
			const float weight = exp2_(v[u].x - lowest);
			lds.weights[from + 16 * u][r] = weight;
			s1 += v[u].y * weight;
		}
		for (int d = 1; d < 16; d *= 2) s1 += __shfl_xor(s1, d);
		if (from == 0) { most[0][r] = top; total[0][r] = s1; }
	}
	__syncthreads();
	const uint32_t quads = rows * (D / 4), across = min(quads, 256u), groups = 256 / across, group = tid / across;
	for (uint32_t e0 = 0; e0 < quads; e0 += across) {
		const uint32_t e = e0 + tid % across, r = min(e, quads - 1) / (D / 4);
		f32x4 mine{ 0.0f, 0.0f, 0.0f, 0.0f };
		auto add = [&](auto batch) { /* the group's parts, so many under way */
			constexpr uint32_t BATCH = decltype(batch)::value;
			for (uint32_t p = group; p < parts; p += BATCH * groups) {
				f32x4 v[BATCH];
#pragma unroll
				for (uint32_t u = 0; u < BATCH; ++u) v[u] = *(const f32x4*)(left + min(p + u * groups, parts - 1) * PART + 4 * e);
#pragma unroll
				for (uint32_t u = 0; u < BATCH; ++u)
					if (p + u * groups < parts) mine += v[u] * lds.weights[p + u * groups][r];
			}
		};
		if (group < groups && e < quads) {
			if (parts > 4 * groups) add(std::integral_constant<uint32_t, 16>{});
			else add(std::integral_constant<uint32_t, 4>{});
		}
		if (groups > 1) { /* (then this loop has one turn) */
			shares[tid] = mine;
			__syncthreads();
			if (group == 0)
				for (uint32_t g = 1; g < groups; ++g) mine += shares[g * across + tid];
		}
		if (group != 0 || e >= quads) continue;
		const float s1 = total[0][r], by = s1 > 0.0f ? 1.0f / s1 : s1 == s1 ? 0.0f : s1;
		const Row4 to_row = row_of(a, seq, row_tile, r);
		const size_t token = seq.first + to_row.token, query_head = (size_t)head * a.batch.group + to_row.head;
		float v[4];
		for (int i = 0; i < 4; ++i) v[i] = mine[i] * by;
		store_out4(a, (char*)a.out + 2 * (token * a.out_token + query_head * a.out_head), 4 * (e % (D / 4)), v);
		if (e % (D / 4) == 0 && a.lse) a.lse[token * a.batch.query_heads + query_head] = s1 == 0.0f ? -__builtin_inff() : (most[0][r] + log2f(s1 * LOWERED)) * 0.693147180559945309f;
	}
}

/* ---------------------------------------------------------------- many rows ---------------------- */

typedef float f32x16 __attribute__((ext_vector_type(16)));

/* tiles of 64 tokens that 256 rows of a sequence look at; 0: no such rows, and at least 1 (of nothing) where there are. (Rows, and tiles of all units,
 * are counted in 31 bits where a call is divided in shares.) */
__device__ __forceinline__ uint32_t many_tiles(const Attend4& a, uint32_t s, uint32_t row_tile)
{
	const Sequence seq = sequence_of(a.batch, s, a.cache.page_shift);
	const uint64_t all_rows = (uint64_t)seq.queries * a.batch.group, first_row = (uint64_t)row_tile * 256;
	if (first_row >= all_rows) return 0;
	const uint64_t last = min(first_row + 255, all_rows - 1);
	const uint32_t query = !a.batch.causal ? 0 : a.joined ? (uint32_t)last / a.batch.group : (uint32_t)(last / a.batch.group);
	return max(1u, (visible_to(a.batch, seq, query) + 63) / 64);
}

__device__ __forceinline__ uint32_t scan4(uint32_t v) /* sums up to and with each lane */
{
	for (uint32_t d = 1; d < WAVE; d *= 2) {
		const uint32_t below = (uint32_t)__shfl_up((int)v, d);
		if (threadIdx.x % WAVE >= d) v += below;
	}
	return v;
}

/* What a work-group of the many-rows kernel takes: the tiles [from, to) of all units (a unit is a head of an entry, an entry 256 rows of a
 * sequence; entries in order, their heads side by side), which begin in a place of unit (entry, head); or whole units. Each wavefront finds it. */
struct Share4 { uint32_t from, to, entry, head, at, shares, total; };
__device__ __forceinline__ uint32_t share_begin(uint32_t total, uint32_t g, uint32_t shares)
{
	const uint32_t each = total / shares, more = total - each * shares; /* the first ones take one more */
	return each * g + min(g, more);
}
__device__ __forceinline__ uint32_t share_with(uint32_t total, uint32_t tile, uint32_t shares)
{
	const uint32_t each = total / shares, more = total - each * shares, large = more * (each + 1);
	return tile < large ? tile / (each + 1) : more + (tile - large) / each;
}
__device__ __forceinline__ Share4 share_of(const Attend4& a, uint32_t g)
{
	const uint32_t lane = threadIdx.x % WAVE, entries = a.batch.sequences * a.row_tiles, heads = a.cache.heads;
	Share4 share{};
	uint32_t total = 0, most = 0, units = 0, w = 0, upto = 0;
	for (uint32_t base = 0; base < entries; base += WAVE) {
		const uint32_t e = base + lane;
		w = e < entries ? many_tiles(a, e / a.row_tiles, e % a.row_tiles) : 0;
		upto = scan4(w);
		total += (uint32_t)__builtin_amdgcn_readlane((int)upto, WAVE - 1);
		units += (uint32_t)__popcll(__ballot(w != 0));
		uint32_t largest = w;
		for (int d = 1; d < WAVE; d *= 2) largest = max(largest, (uint32_t)__shfl_xor((int)largest, d));
		most = max(most, (uint32_t)__builtin_amdgcn_readfirstlane((int)largest));
	}
	total *= heads;
	units *= heads;
	share.total = total;
	if (total == 0) return share;
	share.shares = min(a.splits, max(total / MANY_LEAST, units));
	/* whole units, a round of them at a time, where that takes no longer than equal shares and what joining them costs */
	if ((uint64_t)((entries * heads + a.splits - 1) / a.splits) * most <= total / share.shares + MANY_COST) {
		share.shares = 0;
		return share;
	}
	if (g >= share.shares) return share;
	share.from = share_begin(total, g, share.shares);
	share.to = share_begin(total, g + 1, share.shares);
	uint32_t before = 0;
	for (uint32_t base = 0; base < entries; base += WAVE) {
		if (entries > WAVE) {
			const uint32_t e = base + lane;
			w = e < entries ? many_tiles(a, e / a.row_tiles, e % a.row_tiles) : 0;
			upto = scan4(w);
		}
		const uint64_t behind = __ballot(before + upto * heads > share.from);
		if (behind) {
			const int e = __ffsll((unsigned long long)behind) - 1;
			const uint32_t tiles = (uint32_t)__builtin_amdgcn_readlane((int)w, e);
			const uint32_t into = share.from - (before + ((uint32_t)__builtin_amdgcn_readlane((int)upto, e) - tiles) * heads);
			share.entry = base + (uint32_t)e;
			share.head = into / tiles;
			share.at = into - share.head * tiles;
			break;
		}
		before += (uint32_t)__builtin_amdgcn_readlane((int)upto, WAVE - 1) * heads;
	}
	return share;
}

/*
 * Many rows (pieces of prompts): a work-group of eight wavefronts takes 256 rows of one head, 32 a wavefront, and a part of the tokens. Tiles of 64
 * tokens become half-precision numbers once for all of them: wavefront w < 4 unpacks the keys of block w, wavefront 4 + w its values, into LDS,
 * into one of two buffers while everybody works on the other. Scores are [token][row] as above (v_mfma_f32_32x32x16_f16, 16 tokens a lane and
 * half of the tile), so that probabilities stay in their registers: the values' tokens lie in LDS in the order in which a lane has them. Rows of
 * LDS are 16 bytes longer than their contents: 8 lanes one below the other read 8 different groups of banks.
 * Bound by the sum of its phases: 2 x 1024 queries, 32 heads on 8 of 128, 16384 and fewer tokens take 530 us (570 on another card), 764 TFLOP/s of the 1150 that a large matrix
 * product reaches; one sequence of 16384, in two parts, 328, 812. Matrix cores are busy 34 % of that time, vector units 49 % (265 instructions a wavefront and
 * tile, 36 %, and 32 exponentials among them that take four times as long), LDS some 40 %: all wavefronts pass one barrier a tile and are in the same phase
 * at the same time. A work-group takes a part of a unit (256 rows of a head), or its share of all units' tiles, from inside of one to inside of another. Heads of
 * 32 and 64 channels have two work-groups on a compute unit (376 and 405 us with one, 321 and 375 with two, before the shares), for which 64 channels keep 4 to 12
 * registers in memory. So do wide heads, whose sums and queries are more than the registers hold: 192 channels 2, 224 19 to 33, 256 50 to 72 (1277 us, 635 TFLOP/s).
 */
template <int J>
__device__ __forceinline__ void many_unit(const Attend4& a, uint8_t* many, uint32_t (*blocks_there)[4], uint32_t entry, uint32_t head, uint32_t begin, uint32_t until,
                                          bool whole, uint32_t parts, uint32_t slot)
{
	constexpr uint32_t D = 32 * J, KROW = 2 * D + 16, VROW = 144, TILE = 64 * KROW + D * VROW;
	constexpr int STEP = (J <= 5 ? 2 : 1); /* times 32 tokens of a tile: scores held at a time */
	/* scores always give the maximum up themselves (see below_most) where registers go to memory anyway, and a branch costs more of them (2 x 1024 queries, 256
	 * channels: 1328 us, 1475 with the branch; 224: 947 and 954; 192: 762 and 747, 128: 550 and 540) */
	constexpr bool EXACT = J > 6;
	uint32_t thread = threadIdx.x;
	asm volatile("" : "+v"(thread)); /* addresses that follow from it are made anew for each unit, not kept from one to the next */
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(thread / WAVE)), lane = thread % WAVE, n32 = lane % 32, h = lane / 32;
	const uint32_t s = entry / a.row_tiles;
	const Sequence seq = sequence_of(a.batch, s, a.cache.page_shift);
	const uint64_t all_rows = (uint64_t)seq.queries * a.batch.group, first_row = (uint64_t)(entry % a.row_tiles) * 256;
	const uint32_t rows = (uint32_t)min((uint64_t)256, all_rows - first_row);
	const uint32_t end = min(until, (visible_to(a.batch, seq, (uint32_t)((first_row + rows - 1) / a.batch.group)) + 63) / 64);

	/* the lane's row, and what the rows of its wavefront see at least and at most */
	const uint32_t wave_rows = rows > 32 * wave ? min(32u, rows - 32 * wave) : 0;
	const bool there = n32 < wave_rows;
	const uint64_t x_row = first_row + 32 * wave + (there ? n32 : 0);
	const uint32_t token = there ? (uint32_t)(x_row / a.batch.group) : 0, query_head = (uint32_t)(head * a.batch.group + (there ? x_row % a.batch.group : 0));
	const int32_t sees = there ? (int32_t)visible_to(a.batch, seq, token) : 0;
	const int32_t least = wave_rows ? (int32_t)visible_to(a.batch, seq, (uint32_t)((first_row + 32 * wave) / a.batch.group)) : 0;
	const int32_t seen = wave_rows ? (int32_t)visible_to(a.batch, seq, (uint32_t)((first_row + 32 * wave + wave_rows - 1) / a.batch.group)) : 0;

	half8v q[2 * J]; /* channels 16 c + 8 h .. + 7 */
	float row_scale;
	{
		float x[2 * J][8];
		u32x4 raw[2 * J];
		load_pieces<2 * J>((const uint16_t*)a.q + (size_t)(seq.first + token) * a.q_token + (size_t)query_head * a.q_head + 8 * h, 16, a.vec, raw);
		floats_of<2 * J>(raw, a.bf16, x);
		float largest = 0.0f;
#pragma unroll
		for (int c = 0; c < 2 * J; ++c)
			for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(x[c][e]));
		largest = fmaxf(largest, __shfl_xor(largest, 32));
		const float by = query_scale(a.scale, largest, &row_scale);
#pragma unroll
		for (int c = 0; c < 2 * J; ++c)
			for (int e = 0; e < 8; ++e) q[c][e] = (_Float16)(x[c][e] * by);
	}

	const uint32_t b = wave % 4, sub_bits = a.cache.page_shift - 4; /* the block of a tile that this wavefront unpacks */
	const bool values = wave >= 4;
	const Magnitudes mag = load_magnitudes(a.cache.levels, head, values ? 1 : 0);
	const Constant4 table = constant4(a.batch.table) + (size_t)s * a.batch.table_stride;
	constexpr int VITEMS = (16 * J + WAVE - 1) / WAVE; /* pairs of channels a lane */
	struct { uint32_t codes[values_words<J>()]; u32x4 scales[VITEMS][2]; uint32_t key_scales[(J + 1) / 2]; } in;
	int32_t written = 0; /* tokens of the block that are there */
	bool known = false;  /* it lies on a page of the cache */
	auto fetch = [&](uint32_t tile) {
		const uint32_t n = 4 * tile + b, entry = n >> sub_bits, sub = n & ((1u << sub_bits) - 1);
		const uint32_t page = (uint32_t)table[min(entry, a.batch.table_stride - 1)];
		known = entry < a.batch.table_stride && page < a.cache.page_count;
		written = known ? (int32_t)seq.length - (int32_t)(16 * n) : 0;
		const uint8_t* block = a.cache.blocks + block_offset<J>(a.cache, known ? page : 0, head, sub);
		if (!values) {
			load_words<J>(block + lane * 4 * J, in.codes); /* lane = 4 token + kg */
			load_halves<J>(block + 16 * D + lane / 4 * 2 * J, in.key_scales);
		} else {
#pragma unroll
			for (int i = 0; i < VITEMS; ++i) {
				const uint32_t pair = min(lane + WAVE * i, 16u * J - 1);
				const u32x4 w = *(const u32x4*)(block + 8 * D + 16 * pair);
				for (int e = 0; e < 4; ++e) in.codes[4 * i + e] = w[e];
				in.scales[i][0] = *(const u32x4*)(block + 17 * D + 32 * (pair / 16));
				in.scales[i][1] = *(const u32x4*)(block + 17 * D + 32 * (pair / 16) + 16);
			}
		}
	};
	auto unpack = [&](uint32_t buffer) {
		uint8_t* const tile = many + buffer * TILE;
		if (!values) {
			if (lane == 0) blocks_there[buffer][b] = known ? 1 : 0;
			uint8_t* row = tile + (16 * b + lane / 4) * KROW + 16 * (lane % 4);
#pragma unroll
			for (int j = 0; j < J; ++j) {
				uint32_t w[4];
				unpack4<false>(in.codes[j], mag, w[0], w[1]);
				unpack4<true>(in.codes[j], mag, w[2], w[3]);
				const uint32_t scale = twice(in.key_scales[j / 2], j % 2);
				*(u32x4*)(row + 64 * j) = u32x4{ times(w[0], scale), times(w[1], scale), times(w[2], scale), times(w[3], scale) };
			}
		} else {
#pragma unroll
			for (int i = 0; i < VITEMS; ++i) {
				if (written < 16) { /* what lies behind the last token may hold anything: scales of zero */
#pragma unroll
					for (int d = 0; d < 8; ++d) in.scales[i][d / 4][d % 4] &= written >= 2 * d + 2 ? 0xFFFFFFFFu : written == 2 * d + 1 ? 0xFFFFu : 0u;
				}
				const uint32_t pair = lane + WAVE * i;
				if (16 * J % WAVE && pair >= 16 * J) continue;
				uint32_t low[8], high[8];
#pragma unroll
				for (int d = 0; d < 4; ++d) {
					unpack4<false>(in.codes[4 * i + d], mag, low[2 * d], low[2 * d + 1]);
					unpack4<true>(in.codes[4 * i + d], mag, high[2 * d], high[2 * d + 1]);
					for (int e = 0; e < 2; ++e) {
						const uint32_t scale = in.scales[i][d / 2][2 * (d % 2) + e];
						low[2 * d + e] = times(low[2 * d + e], scale);
						high[2 * d + e] = times(high[2 * d + e], scale);
					}
				}
				/* tokens 0 to 3 and 8 to 11 are those of the lanes with h = 0, the others of h = 1 */
				uint8_t* row = tile + 64 * KROW + (32 * (pair / 16) + pair % 16) * VROW + 32 * b;
				*(u32x4*)row = u32x4{ low[0], low[1], low[4], low[5] };
				*(u32x4*)(row + 16) = u32x4{ low[2], low[3], low[6], low[7] };
				*(u32x4*)(row + 16 * VROW) = u32x4{ high[0], high[1], high[4], high[5] };
				*(u32x4*)(row + 16 * VROW + 16) = u32x4{ high[2], high[3], high[6], high[7] };
			}
		}
	};

	float m = -__builtin_inff(), l = 0.0f, base = RAISE;
	bool any_far = false; /* rows of the wavefront with scores far from zero */
	f32x16 o[J];
#pragma unroll
	for (int j = 0; j < J; ++j)
		for (int e = 0; e < 16; ++e) o[j][e] = 0.0f;

	auto work = [&](uint32_t buffer, int32_t from) {
		const uint8_t* const tile = many + buffer * TILE;
		uint32_t blocks = 0;
		for (int n = 0; n < 4; ++n) blocks |= blocks_there[buffer][n] << n;
		blocks = (uint32_t)__builtin_amdgcn_readfirstlane((int)blocks);
#pragma unroll
		for (int t0 = 0; t0 < 2; t0 += STEP) {
			f32x16 sc[STEP];
#pragma unroll
			for (int t = 0; t < STEP; ++t) {
				for (int e = 0; e < 16; ++e) sc[t][e] = 0.0f;
#pragma unroll
				for (int c = 0; c < 2 * J; ++c)
					sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const half8v*)(tile + (32 * (t0 + t) + n32) * KROW + 32 * c + 16 * h), q[c], sc[t], 0, 0, 0);
			}
			if (least - from < 64 || blocks != 15) { /* (neither is negative: no sum that may pass 31 bits) */
#pragma unroll
				for (int e = 0; e < 16 * STEP; ++e) {
					const int32_t place = from + 32 * (t0 + e / 16) + 8 * (e % 16 / 4) + 4 * (int32_t)h + e % 4;
					sc[e / 16][e % 16] = place < sees && (blocks >> (2 * t0 + e / 8) & 1) ? sc[e / 16][e % 16] : -__builtin_inff();
				}
			}
			float top = sc[0][0];
#pragma unroll
			for (int e = 1; e < 16 * STEP; ++e) top = fmaxf(top, sc[e / 16][e % 16]);
			top = fmaxf(top, __shfl_xor(top, 32));
			const float now = fmaxf(m, top);
			if (any_far || __any(now > m)) {
				const float less = m == now ? 1.0f : exp2_((m - now) * row_scale);
				l *= less;
#pragma unroll
				for (int j = 0; j < J; ++j) o[j] *= less;
				m = now;
				if constexpr (!EXACT) {
					any_far = __any(far_score(m, row_scale));
					base = below_most(m, row_scale, any_far, [&](float most) {
#pragma unroll
						for (int t = 0; t < STEP; ++t) sc[t] -= most;
					});
				}
			}
			if constexpr (EXACT) {
				const float most = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
				for (int t = 0; t < STEP; ++t) sc[t] -= most;
			}
			half8v p[2 * STEP];
#pragma unroll
			for (int e = 0; e < 16 * STEP; ++e) {
				const float v = exp2_(fmaf(sc[e / 16][e % 16], row_scale, base));
				l += v;
				p[e / 8][e % 8] = (_Float16)v;
			}
#pragma unroll
			for (int j = 0; j < J; ++j)
#pragma unroll
				for (int c = 0; c < 2 * STEP; ++c)
					o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const half8v*)(tile + 64 * KROW + (32 * j + n32) * VROW + 32 * (2 * t0 + c) + 16 * h), p[c], o[j], 0, 0, 0);
		}
	};

	if (begin < end) {
		fetch(begin);
		unpack(0);
		fetch(min(begin + 1, end - 1));
		__syncthreads();
		for (uint32_t tile = begin; tile < end; ++tile) {
			const uint32_t now = (tile - begin) % 2;
			if (tile + 1 < end) unpack(1 - now);
			if (tile + 2 < end) fetch(tile + 2);
			if ((int32_t)(64 * tile) < seen) work(now, (int32_t)(64 * tile));
			__syncthreads();
		}
	}
	l += __shfl_xor(l, 32);

	if (a.joined && begin == 0 && threadIdx.x == 0) /* for the join: the unit's first share, and how many it lies in */
		((uint2*)(a.partial + (size_t)(a.tiles_per_split ? 1 : 2) * a.splits * (256 * (D + 2))))[entry * a.cache.heads + head] = uint2{ blockIdx.x, parts };
	if (!there) return;
	if (whole) {
		const float by = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
		char* to = (char*)a.out + 2 * ((size_t)(seq.first + token) * a.out_token + (size_t)query_head * a.out_head);
#pragma unroll
		for (int j = 0; j < J; ++j)
			for (int e = 0; e < 4; ++e) {
				float v[4];
				for (int r = 0; r < 4; ++r) v[r] = o[j][4 * e + r] * by;
				store_out4(a, to, 32 * j + 8 * e + 4 * h, v);
			}
		if (h == 0 && a.lse) a.lse[(size_t)(seq.first + token) * a.batch.query_heads + query_head] = l == 0.0f ? -__builtin_inff() : (m * row_scale + log2f(l * LOWERED)) * 0.693147180559945309f;
		return;
	}

	/* a part of the tokens: [256][D] sums, then [256] pairs of maximum and sum, for join4_kernel */
	float* const to = a.partial + (size_t)slot * (256 * (D + 2));
	const uint32_t r = 32 * wave + n32;
#pragma unroll
	for (int j = 0; j < J; ++j)
		for (int e = 0; e < 4; ++e) *(f32x4*)(to + (size_t)r * D + 32 * j + 8 * e + 4 * h) = f32x4{ o[j][4 * e], o[j][4 * e + 1], o[j][4 * e + 2], o[j][4 * e + 3] };
	if (h == 0) *(float2*)(to + 256 * D + 2 * r) = float2{ m * row_scale, l };
}

template <int J, bool SHARES>
__global__ void __launch_bounds__(512, J <= 2 ? 4 : 2)
attend4_many_kernel(Attend4 a)
{
	extern __shared__ __attribute__((aligned(16))) uint8_t many[]; /* two tiles: keys [token][channel], values [channel][token] */
	__shared__ uint32_t blocks_there[2][4];
	const uint32_t heads = a.cache.heads, entries = a.batch.sequences * a.row_tiles;
	if constexpr (!SHARES) {
		const uint32_t units = entries * heads, part = blockIdx.x / units, unit = blockIdx.x % units, entry = unit / heads;
		const uint32_t weight = many_tiles(a, entry / a.row_tiles, entry % a.row_tiles), begin = part * a.tiles_per_split;
		if (begin >= weight) return;
		const uint32_t parts = (weight + a.tiles_per_split - 1) / a.tiles_per_split;
		many_unit<J>(a, many, blocks_there, entry, unit % heads, begin, min(weight, begin + a.tiles_per_split), parts == 1, parts, blockIdx.x);
	} else {
		__shared__ Share4 share; /* (in registers it would be there through all the work) */
		const Share4 mine = share_of(a, blockIdx.x);
		if (mine.total == 0 || (mine.shares && blockIdx.x >= mine.shares)) return;
		if (threadIdx.x == 0) share = mine;
		__syncthreads();
		const bool shared = __builtin_amdgcn_readfirstlane((int)mine.shares) != 0;
		uint32_t entry = (uint32_t)__builtin_amdgcn_readfirstlane((int)(shared ? mine.entry : blockIdx.x / heads));
		uint32_t head = (uint32_t)__builtin_amdgcn_readfirstlane((int)(shared ? mine.head : blockIdx.x % heads));
		uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)mine.at);
		uint32_t left = (uint32_t)__builtin_amdgcn_readfirstlane((int)(mine.to - mine.from)); /* tiles of the share */
		while (entry < entries) { /* a unit, or a part of one, after the other */
			const uint32_t weight = many_tiles(a, entry / a.row_tiles, entry % a.row_tiles);
			const uint32_t begin = at, until = shared ? min(weight, at + left) : weight;
			const bool whole = begin == 0 && until == weight;
			uint32_t parts = 1;
			if (!whole && begin == 0) parts = share_with(share.total, share.to - left + weight - 1, share.shares) - blockIdx.x + 1;
			if (weight) many_unit<J>(a, many, blocks_there, entry, head, begin, until, whole, parts, 2 * blockIdx.x + (begin == 0));
			if (!shared) {
				const uint32_t next = entry * heads + head + gridDim.x;
				entry = next / heads;
				head = next % heads;
				continue;
			}
			left -= until - begin;
			if (left == 0) return;
			at = 0;
			if (++head == heads || weight == 0) {
				head = 0;
				++entry;
			}
		}
	}
}

/* Joins the parts of many rows: 256 rows of sums are more than one work-group should read alone, so they have a kernel. A wavefront takes a row, 8 J
 * lanes 4 channels each of every (64 / 8 J)-th part. */
constexpr uint32_t JOIN_GROUPS = 64; /* work-groups a unit */
template <int J>
__global__ void __launch_bounds__(256)
join4_kernel(Attend4 a)
{
	constexpr uint32_t D = 32 * J, LANES = 8 * J, GROUPS = WAVE / LANES;
	constexpr size_t PART = 256 * (D + 2);
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE;
	const uint32_t unit = blockIdx.x / JOIN_GROUPS, entry = unit / a.cache.heads, head = unit % a.cache.heads;
	const Sequence seq = sequence_of(a.batch, entry / a.row_tiles, a.cache.page_shift);
	const uint64_t all_rows = (uint64_t)seq.queries * a.batch.group, first_row = (uint64_t)(entry % a.row_tiles) * 256;
	if (first_row >= all_rows) return;
	const uint32_t rows = (uint32_t)min((uint64_t)256, all_rows - first_row);
	const uint32_t each = a.tiles_per_split ? 1 : 2; /* slots a work-group */
	const uint2 record = ((const uint2*)(a.partial + each * (size_t)a.splits * PART))[unit];
	const uint32_t parts = record.y, group = lane / LANES, at = lane % LANES;
	if (parts <= 1) return; /* written where it belongs */
	/* of shares the first part is the second one of its work-group, the others are first ones */
	const float* left = a.partial + each * (size_t)record.x * PART;
	const size_t first = (each - 1) * PART, step = (a.tiles_per_split ? (size_t)a.batch.sequences * a.row_tiles * a.cache.heads : 2) * PART; /* from a part's work-group to the next one's */
	for (uint32_t r = blockIdx.x % JOIN_GROUPS * 4 + wave; r < rows; r += 4 * JOIN_GROUPS) {
		float top = -__builtin_inff();
		for (uint32_t p = lane; p < parts; p += WAVE) top = fmaxf(top, left[(p ? p * step : first) + 256 * D + 2 * r]);
		for (int d = 1; d < WAVE; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
		const float lowest = top == -__builtin_inff() ? 0.0f : top;
		float sum = 0.0f;
		f32x4 mine{ 0.0f, 0.0f, 0.0f, 0.0f };
		if (group < GROUPS)
#pragma unroll 4
			for (uint32_t p = group; p < parts; p += GROUPS) {
				const float* part = left + (p ? p * step : first);
				const float2 ml = *(const float2*)(part + 256 * D + 2 * r);
				const float weight = exp2_(ml.x - lowest);
				sum += ml.y * weight;
				mine += *(const f32x4*)(part + (size_t)r * D + 4 * at) * weight;
			}
		for (uint32_t g = 1; g < GROUPS; ++g) { /* the groups' sums, in their order */
			const int other = (int)(at + g * LANES);
			const f32x4 more{ __shfl(mine[0], other), __shfl(mine[1], other), __shfl(mine[2], other), __shfl(mine[3], other) };
			const float more_sum = __shfl(sum, other);
			if (group == 0) { mine += more; sum += more_sum; }
		}
		if (group != 0) continue;
		const float by = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;
		const uint64_t x = first_row + r;
		const size_t to_token = seq.first + x / a.batch.group, to_head = (size_t)head * a.batch.group + x % a.batch.group;
		float v[4];
		for (int e = 0; e < 4; ++e) v[e] = mine[e] * by;
		store_out4(a, (char*)a.out + 2 * (to_token * a.out_token + to_head * a.out_head), 4 * at, v);
		if (at == 0 && a.lse) a.lse[to_token * a.batch.query_heads + to_head] = sum == 0.0f ? -__builtin_inff() : (top + log2f(sum * LOWERED)) * 0.693147180559945309f;
	}
}

template <int J>
int launch_attend4(Attend4 a, const Plan4& plan)
{
	a.row_tiles = plan.row_tiles;
	a.splits = plan.splits;
	a.tiles_per_split = plan.tiles_per_split;
	a.joined = plan.joined;
	if (plan.many) {
		constexpr uint32_t bytes = 2 * (64 * (64 * J + 16) + 32 * J * 144);
		if (bytes > 65536) { /* more LDS than a launch may ask for unannounced, on this device */
			static int allowed = -1;
			const DeviceInfo* dev = nullptr;
			const int rc = device_info(&dev);
			if (rc) return rc;
			if (allowed != dev->device) {
				KMX_HIP(hipFuncSetAttribute((const void*)attend4_many_kernel<J, false>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
				KMX_HIP(hipFuncSetAttribute((const void*)attend4_many_kernel<J, true>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
				allowed = dev->device;
			}
		}
		if (a.tiles_per_split == 0) KMX_LAUNCH_KERNEL((attend4_many_kernel<J, true>), dim3(a.splits), dim3(512), bytes, stream(), a);
		else KMX_LAUNCH_KERNEL((attend4_many_kernel<J, false>), dim3(a.splits), dim3(512), bytes, stream(), a);
		KMX_LAUNCH_CHECK("attend4_many_kernel");
		if (a.joined) {
			KMX_LAUNCH_KERNEL((join4_kernel<J>), dim3((unsigned)(plan.units * JOIN_GROUPS)), dim3(256), 0, stream(), a);
			KMX_LAUNCH_CHECK("join4_kernel");
		}
		return KMX_OK;
	}
	if (a.batch.sequences > 65535 || (uint64_t)a.row_tiles * a.splits > 65535)
		return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_attend: %u sequences of %u queries are too many for one call", a.batch.sequences, a.batch.max_queries);
	KMX_LAUNCH_KERNEL((attend4_kernel<J>), dim3(a.cache.heads, a.batch.sequences, a.row_tiles * a.splits), dim3(256), 0, stream(), a);
	KMX_LAUNCH_CHECK("attend4_kernel");
	return KMX_OK;
}

} // namespace kmx

#endif
