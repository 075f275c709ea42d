/*
 * Attention over prompts (kmx_prompt_attend of include/kmx.h), kernels for J groups of 32 channels (one object per J: prompt_attend_inst.hip).
 *
 * For a row r (a query head of a query) that sees the tokens t < vis: o_r = sum_t p_rt v_t / l_r, p_rt = 2^(c s_rt - m_r), s_rt = +- q_r . k_t, c = |scale| log2(e),
 * l_r = sum_t p_rt; lse_r = ln 2 (m_r + log2 l_r). m_r is any number near the largest c s_rt: it is raised when one passes it by more than 2^RISE, and what
 * was added up before is lowered by as much. Exponents are c s + base, base = LIFT - m; where c s is far from zero that difference of two roundings is no small number any more, and they
 * are c (s - shift) + LIFT, shift the score itself.
 */
#ifndef KMX_PROMPT_ATTEND_IMPL_H
#define KMX_PROMPT_ATTEND_IMPL_H

#include "prompt_attend.h"

#include <type_traits>

namespace kmx {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

/*
 * Probabilities are rounded to the type of the values for their product with them, sums are those of the floats. They are taken times 2^LIFT, and may pass the
 * reference by 2^RISE: half precision holds them up to 2^15, with 11 bits down to 2^-21 of the reference and none below 2^-32; bfloat16 has 8 bits of all of them.
 */
constexpr float LIFT = 7.0f, MOST_SUM = 0x1p15f; /* 2^(LIFT + RISE), RISE = 8 */
constexpr float FAR = 0x1p20f;           /* exponents of 2 from here on: below it the base has two roundings of 2^-5 at most, the same for all tokens of a row */
constexpr float NOTHING = 3.4028235e38f; /* the base of rows that have no token with a weight so far: the first score that is a number comes to an infinity, and raises */

__device__ __forceinline__ f32x16 product(const u32x4& a, const u32x4& b, const f32x16& c, __bf16)
{
	return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 product(const u32x4& a, const u32x4& b, const f32x16& c, _Float16)
{
	return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8v, a), __builtin_bit_cast(half8v, b), c, 0, 0, 0);
}
/* two numbers that are no NaN, or both whatever they are, rounded to the nearest */
__device__ __forceinline__ uint32_t rounded_pair(float x, float y, __bf16)
{
	typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
	return __builtin_bit_cast(uint32_t, bf16x2{ (__bf16)x, (__bf16)y });
}
__device__ __forceinline__ uint32_t rounded_pair(float x, float y, _Float16)
{
	return __builtin_bit_cast(uint32_t, half2v{ (_Float16)x, (_Float16)y });
}
/* the larger one of a lane's and of that 32 lanes on (of the two results of the exchange the compiler would drop the second: it is hidden from it that they are) */
__device__ __forceinline__ float both_halves_most(float v)
{
	const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
	uint32_t low = r[0], high = r[1];
	asm volatile("" : "+v"(low), "+v"(high));
	return fmaxf(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high));
}
/* 4 rows (tokens) x 16 columns of LDS: the lanes of each group of 16 hand in 8 bytes of a row, 4 lanes a row, and get 4 tokens of their column */
__device__ __forceinline__ u32x2 read_turned(const uint8_t* p)
{
	return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p)));
}

/* whether one of the 8 numbers is an infinity or NaN; those as zeros */
template <typename T>
__device__ __forceinline__ bool without_strange(u32x4& w)
{
	constexpr uint32_t EXPONENT = __is_same(T, __bf16) ? 0x7F80u : 0x7C00u;
	bool found = false;
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		const bool low = (w[i] & EXPONENT) == EXPONENT, high = (w[i] >> 16 & EXPONENT) == EXPONENT;
		w[i] &= (low ? 0u : 0xFFFFu) | (high ? 0u : 0xFFFF0000u);
		found = found || low || high;
	}
	return found;
}

/* an address that is the same in all lanes, in scalar registers */
__device__ __forceinline__ void* same_in_all(const void* p)
{
	const uint64_t u = (uint64_t)p;
	return (void*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)u));
}

struct Prompt4 { uint32_t query_first, queries, token_first, tokens; };
/* queries and tokens of sequence s, held to what there is */
__device__ __forceinline__ Prompt4 prompt_of(const PromptAttend& a, uint32_t s)
{
	const int32_t from = constant4(a.query_starts)[s], to = constant4(a.query_starts)[s + 1], begin = constant4(a.token_starts)[s], end = constant4(a.token_starts)[s + 1];
	Prompt4 p{ 0, 0, 0, 0 };
	if (from >= 0 && to > from && (uint32_t)to <= a.queries) {
		p.query_first = (uint32_t)from;
		p.queries = min((uint32_t)(to - from), a.max_queries);
	}
	if (begin >= 0 && end > begin && (uint32_t)end <= a.tokens) {
		p.token_first = (uint32_t)begin;
		p.tokens = min((uint32_t)(end - begin), a.max_tokens);
	}
	return p;
}
__device__ __forceinline__ int32_t sees_of(const PromptAttend& a, const Prompt4& p, uint32_t query)
{
	if (!a.causal) return (int32_t)p.tokens;
	const int64_t n = (int64_t)p.tokens - p.queries + query + 1;
	return n > 0 ? (int32_t)n : 0;
}

template <int J> constexpr uint32_t key_row() { return 64 * J + 16; }                       /* bytes: 8 tokens one below the other read 8 groups of banks */
template <int J> constexpr uint32_t value_row() { return 64 * J + (J % 2 ? 0 : 64); }       /* 64 or 192 bytes on in the banks: 4 tokens side by side */
template <int J, int W> constexpr int prompt_waves() { return J <= 6 ? 2 : 1; } /* wavefronts a SIMD: 256 registers each, or 512 */
template <int J, int W> constexpr int prompt_batch() { return J <= 6 ? 1 : J; }
template <int J> constexpr uint32_t prompt_lds() { return 3 * 32 * (key_row<J>() + value_row<J>()) + 1024; } /* (and a place for what wavefronts without pieces store) */

/*
 * Attention over prompts: out = sum_t exp(scale q . k_t) v_t / sum_t exp(scale q . k_t) in one pass, with a reference for the exponents that is raised where a row's weights come to
 * more than 2^15. A work-group of W wavefronts takes 32 W rows of one head of the keys (the query heads of a query side by side, then the next query's), 32 a wavefront, over all
 * tokens or a part of them. Tiles of 32 tokens pass through LDS as they are, three of keys and three of values, from registers that were loaded two tiles before. Both products have the
 * keys' and values' side as their first operand (v_mfma_f32_32x32x16): scores come out as [token][row], a lane has 16 scores of its row, and its probabilities are, as they stand, its
 * piece of the second operand of [channel][row] = values . p; the values' columns are turned on the way from LDS (ds_read_b64_tr_b16).
 * While the vector units make a tile's probabilities, the matrix cores have the scores of the next one and the sums of the one before: nothing of these three waits for another.
 *
 * 8192 tokens, 32 heads of 128 over 8 in bf16, causal: 525 us (cards differ, 515 to 537), 1.05 of the 1.33 PFLOP/s that a large product of matrices reaches here. The matrix cores are busy
 * 52 % of that time, the vector units 43 %; LDS hands each operand to one product only, 128 KiB a tile and work-group, which at 128 bytes a cycle takes as long as the products. At 64
 * channels no unit is full: 6 prompts of up to 4096 in half precision 206 us, matrix cores 25 %, vector units 40 %. A single query over 8192 tokens: 129 us by one work-group a head, 18 by
 * parts (its keys and values take 7). Steps on the way, at 8192 tokens on one card: scores, powers and sums one after the other 1191 us; side by side 733; operands two products ahead 606;
 * powers between the products 564; sums in place of the largest score 528; three places in LDS and buffer loads 521; eight wavefronts 513; scores far from zero, 1 more.
 */
template <typename T, int J, int W, bool VEC>
__global__ void __launch_bounds__(64 * W, (prompt_waves<J, W>()))
prompt_attend_kernel(PromptAttend a)
{
	constexpr uint32_t KROW = key_row<J>(), VROW = value_row<J>(), KTILE = 32 * KROW, PLACE = KTILE + 32 * VROW;
	constexpr uint32_t THREADS = 64 * W, ROWS = 32 * W;
	constexpr uint32_t TILE_PIECES = 4 * J * 32; /* of 16 bytes, of keys, and as many of values */
	constexpr int PIECES = (2 * TILE_PIECES + THREADS - 1) / THREADS; /* that a lane brings each step */
	extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
	__shared__ uint32_t strange; /* values that are no numbers, where not all rows see them */
	const uint32_t tid = threadIdx.x, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid / WAVE)), lane = tid % WAVE, n32 = lane % 32, h = lane / 32;
	/* heads take turns over the dies, and the rows that see the most come first */
	const uint32_t part = blockIdx.x / a.units, unit = blockIdx.x - part * a.units, head = unit % a.heads, rest = unit / a.heads, s = rest % a.sequences, row_tile = a.row_tiles - 1 - rest / a.sequences;
	const Prompt4 p = prompt_of(a, s);
	const uint32_t all_rows = p.queries * a.group, first_row = row_tile * ROWS; /* (31 bits) */
	if (first_row >= all_rows) return;
	const uint32_t rows = min(ROWS, all_rows - first_row);
	const uint32_t all_tiles = ((uint32_t)sees_of(a, p, (first_row + rows - 1) / a.group) + 31) / 32, start = part * a.tiles_per_part;
	if (part && start >= all_tiles) return;
	const uint32_t end = min(all_tiles - start, a.tiles_per_part); /* tiles, from the part's first one on */
	const int32_t limit = (int32_t)min(32 * (start + end), 0x7FFFFFFFu); /* tokens behind are another part's */
	const int32_t all_see = min(sees_of(a, p, first_row / a.group), limit);

	/* the rows of the lane, what those of its wavefront see at least, and the tiles they look at */
	const uint32_t wave_first = 32 * wave, wave_rows = rows > wave_first ? min(32u, rows - wave_first) : 0;
	const bool there = n32 < wave_rows;
	const uint32_t x = first_row + (there ? wave_first + n32 : 0), query = x / a.group, query_head = head * a.group + (x - query * a.group);
	const int32_t sees = there ? min(sees_of(a, p, query), limit) : 0;
	const int32_t least = wave_rows ? min(sees_of(a, p, (first_row + wave_first) / a.group), limit) : 0;
	const uint32_t seen = wave_rows ? ((uint32_t)min(sees_of(a, p, (first_row + wave_first + wave_rows - 1) / a.group), limit) + 31) / 32 : 0, mine = seen > start ? seen - start : 0;

	u32x4 q[2 * J]; /* channels 16 c + 8 h .. + 7 */
	const uint16_t* from = (const uint16_t*)a.q + (size_t)(p.query_first + query) * a.q_token + (size_t)query_head * a.q_head + 8 * h;
#pragma unroll
	for (int c = 0; c < 2 * J; ++c) {
		q[c] = load_raw8(from + 16 * c, VEC);
		for (int e = 0; e < 4; ++e) q[c][e] = (q[c][e] & a.q_keep) ^ a.q_turn; /* the sign of the scale; nothing of them where it is 0 */
		if constexpr (prompt_waves<J, W>() == 1) asm volatile("" : "+a"(q[c])); /* (the other half of the registers) */
	}

	/* what lies behind the last token is the last token again: no row sees it */
	const uint16_t* const key_rows = (const uint16_t*)a.k + (size_t)p.token_first * a.token_stride + (size_t)head * a.head_stride;
	const uint16_t* const value_rows = (const uint16_t*)a.v + (size_t)p.token_first * a.token_stride + (size_t)head * a.head_stride;
	/*
	 * Pieces of 16 bytes of a step: a tile's keys, then (another tile's) values, shared out over the lanes; whole wavefronts bring the one or the other. `at`: where they lie from the
	 * sequence's first token on, `to`: where they go in LDS, in the three places in turn. With whole pieces what lies behind the last token is zeros (the hardware's own check of
	 * offsets in a buffer), else the last token again: no row sees it.
	 */
	struct Staged { u32x4 w[PIECES]; };
	const uint32_t stride = (uint32_t)(2 * a.token_stride), size = p.tokens ? (p.tokens - 1) * stride + 64 * J : 0;
	const auto size_in_all = __builtin_amdgcn_readfirstlane((int)size);
	constexpr uint32_t AHEAD_KEYS = 3, AHEAD_VALUES = 1; /* tiles on */
	bool values[PIECES];
	void* rows_of[PIECES];
	uint32_t at[PIECES], to[PIECES], to0[PIECES], to1[PIECES], to2[PIECES];
#pragma unroll
	for (int i = 0; i < PIECES; ++i) {
		const uint32_t first = __builtin_amdgcn_readfirstlane((int)(WAVE * wave + THREADS * i)), piece = tid + THREADS * i;
		values[i] = first >= TILE_PIECES;
		rows_of[i] = same_in_all(values[i] ? value_rows : key_rows);
		const bool none = first >= 2 * TILE_PIECES; /* (those fetch nothing, and store to a place of their own) */
		const uint32_t n = none ? 0 : values[i] ? piece - TILE_PIECES : piece, token = n / (4 * J), part = 16 * (n % (4 * J));
		const uint32_t from = token + 32 * (start + (values[i] ? AHEAD_VALUES : AHEAD_KEYS));
		at[i] = VEC ? (none ? size : from * stride + part) : (none ? 0xFFFFFFFFu : from);
		to[i] = none ? 3 * PLACE + 16 * lane : values[i] ? KTILE + token * VROW + part : token * KROW + part; /* and in a place: */
		to0[i] = to[i] + (none ? 0 : values[i] ? PLACE : 0);
		to1[i] = to[i] + (none ? 0 : values[i] ? 2 * PLACE : PLACE);
		to2[i] = to[i] + (none ? 0 : values[i] ? 0 : 2 * PLACE);
	}
	auto load = [&](int i) { /* and on to the next tile */
		u32x4 w;
		if constexpr (VEC) {
			const auto buffer = __builtin_amdgcn_make_buffer_rsrc(rows_of[i], 0, size_in_all, 0x00020000);
			w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(buffer, (int)at[i], 0, 0));
			at[i] += 32 * stride;
			asm volatile("" : "+v"(at[i])); /* (one register, not one for each of six steps) */
		} else {
			w = load_raw8((const uint16_t*)rows_of[i] + (size_t)min(at[i], p.tokens - 1) * a.token_stride + 8 * ((tid + THREADS * i) % (4 * J)), false);
			at[i] = at[i] > 0xFFFFFFFFu - 32 ? at[i] : at[i] + 32;
		}
		return w;
	};
	auto check = [&](Staged& g, uint32_t tile) { /* of values: 0 times an infinity must not come into rows that do not see it */
		if ((int32_t)(32 * (start + tile) + 32) <= all_see) return;
		bool found = false;
#pragma unroll
		for (int i = 0; i < PIECES; ++i)
			if (values[i]) found = without_strange<T>(g.w[i]) || found;
		if (__any(found)) strange = 1;
	};

	float base = NOTHING, shift = 0.0f, l = 0.0f;
	float most_sum = MOST_SUM; /* no sum is small enough where rows of the wavefront have a shift */
	f32x16 o[J];
#pragma unroll
	for (int j = 0; j < J; ++j)
		for (int e = 0; e < 16; ++e) o[j][e] = 0.0f;

	struct Scores { f32x16 s; };
	struct Weights { u32x4 w[2]; };
	const uint8_t* const key_at = lds + n32 * KROW + 16 * h;
	const uint8_t* const value_at = lds + KTILE + (4 * h + lane % 16 / 4) * VROW + 32 * (lane / 16 % 2) + 8 * (lane % 4);
	auto key_operand = [&](uint32_t at, int i) { return *(const u32x4*)(key_at + at + 32 * i); };
	auto value_operand = [&](u32x4& w, uint32_t at, int i, int half) { /* tokens 0 to 3 of 8, or the others */
		const u32x2 v = read_turned(value_at + at + (16 * (i % 2) + 8 * half) * VROW + 64 * (i / 2));
		w[2 * half] = v[0];
		w[2 * half + 1] = v[1];
	};
	auto score = [&](Scores& sc, uint32_t at) {
		for (int e = 0; e < 16; ++e) sc.s[e] = 0.0f;
#pragma unroll
		for (int c = 0; c < 2 * J; ++c) {
			const u32x4 w = key_operand(at, c);
			sc.s = product(w, q[c], sc.s, T{});
		}
	};
	auto weigh = [&](Weights& p, float& sum, const Scores& sc) {
		sum = 0.0f;
#pragma unroll
		for (int e = 0; e < 16; e += 2) {
			const float x = __builtin_amdgcn_exp2f(fmaf(sc.s[e], a.factor, base)), y = __builtin_amdgcn_exp2f(fmaf(sc.s[e + 1], a.factor, base));
			sum += x + y;
			p.w[e / 8][e % 8 / 2] = rounded_pair(x, y, T{});
		}
	};
	/* the references of rows whose scores pass them (all rows of the wavefront: what has not passed stays), with what was added up so far */
	auto raise = [&](const Scores& sc) {
		float top = sc.s[0];
#pragma unroll
		for (int e = 1; e < 16; ++e) top = fmaxf(top, sc.s[e]);
		top = both_halves_most(top);
		const float most = top * a.factor, old_base = base, old_shift = shift;
		if (fmaf(top - shift, a.factor, base) > LIFT) {
			const bool away = !(fabsf(most) < FAR);
			shift = away ? top : 0.0f;
			base = away ? LIFT : LIFT - most;
		}
		const float less = __builtin_amdgcn_exp2f(fminf(fmaf(old_shift - shift, a.factor, base - old_base), 0.0f)); /* (1 where there was nothing, or an infinity) */
		most_sum = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, __any(shift != 0.0f) ? -1.0f : MOST_SUM)));
		l *= less;
#pragma unroll
		for (int j = 0; j < J; ++j) o[j] *= less;
	};
	auto lower = [&](Scores& sc) { /* scores that are not looked at again */
#pragma unroll
		for (int e = 0; e < 16; ++e) sc.s[e] -= shift;
	};
	auto hide = [&](Scores& sc, uint32_t tile) { /* tokens that a row does not see */
		const int32_t from = (int32_t)(32 * (start + tile));
		if (least - from >= 32) return;
		const int32_t some = sees - from - 4 * (int32_t)h; /* (compared with numbers that stand in the instructions) */
#pragma unroll
		for (int e = 0; e < 16; ++e) sc.s[e] = some > 8 * (e / 4) + e % 4 ? sc.s[e] : -__builtin_inff();
	};
	/* operands come in batches, one in use and one on its way */
	constexpr int STEPS = 2 * J, BATCH = prompt_batch<J, W>(), SLOTS = 2 * STEPS, BATCH_SLOTS = 2 * BATCH;
	u32x4 kop[2][BATCH], vop[2][BATCH];
	Staged g0, g1; /* keys three tiles on and values one; then those of the next tile */
	Scores s0, s1;
	Weights w0, w1;
	/*
	 * A step: the scores of the tile behind, the sums of the tile before, the tile's own weights; the keys of three tiles on and the values of the next one go to LDS and those of
	 * two tiles later are loaded. All in this order and no other (the compiler would have all products first): between two products, of 32 cycles each, one or two probabilities,
	 * each in three turns -- its exponent, the power, where it goes --, operands for later products, a piece of what goes to LDS. One wavefront a SIMD issues an instruction in four
	 * cycles: places in LDS are known when this is compiled (N is the tile's number modulo 6: three places, two sets of registers).
	 */
	auto work = [&](auto number, uint32_t tile) {
		constexpr uint32_t N = decltype(number)::value, HERE = N % 3 * PLACE, ON1 = (N + 1) % 3 * PLACE, ON2 = (N + 2) % 3 * PLACE;
		Staged& g = N % 2 ? g1 : g0;
		Scores &now = N % 2 ? s1 : s0, &next = N % 2 ? s0 : s1;
		Weights &before = N % 2 ? w0 : w1, &weights = N % 2 ? w1 : w0;
		hide(now, tile);
		for (int e = 0; e < 16; ++e) next.s[e] = 0.0f;
		float sum, exponent[2], power[2], before_last = 0.0f;
		auto turn = [&](int n) { /* (the empty statements keep what they name here: left alone all of it goes to where it is used) */
			const int e2 = n - 2;
			if (n >= 2) {
				sum = e2 ? sum + power[n % 2] : power[n % 2];
				asm volatile("" : "+v"(sum));
				if (e2 % 2) {
					uint32_t w = rounded_pair(before_last, power[n % 2], T{});
					asm volatile("" : "+v"(w));
					weights.w[e2 / 8][e2 % 8 / 2] = w;
				}
				before_last = power[n % 2];
			}
			if (n >= 1 && n <= 16) {
				power[(n - 1) % 2] = __builtin_amdgcn_exp2f(exponent[(n - 1) % 2]);
				asm volatile("" : "+v"(power[(n - 1) % 2]));
			}
			if (n < 16) {
				exponent[n % 2] = fmaf(now.s[n], a.factor, base);
				asm volatile("" : "+v"(exponent[n % 2]));
			}
		};
		constexpr int TURNS = 16 + 2, BATCHES = STEPS / BATCH, READS = 3 * BATCH, MOVES = (2 * PIECES + BATCHES - 1) / BATCHES, ITEMS = READS + MOVES;
		auto slot = [&](int t) {
#pragma unroll
			for (int n = TURNS * t / SLOTS; n < TURNS * (t + 1) / SLOTS; ++n) turn(n);
			/* one of a batch's reads of operands for the next, or of its moves -- first those to LDS, then those from memory --, evenly over its slots: all wavefronts
			 * are about here, and LDS takes a read of theirs in 5 cycles and a write in 13 */
			const int batch = t / BATCH_SLOTS, in = t % BATCH_SLOTS, first = (batch + 1) * BATCH, at = (batch + 1) % 2;
#pragma unroll
			for (int p = ITEMS * in / BATCH_SLOTS; p < ITEMS * (in + 1) / BATCH_SLOTS; ++p) {
				const int move = MOVES * p / ITEMS, read = p - move;
				if (MOVES * (p + 1) / ITEMS > move) {
					const int m = batch * MOVES + move, i = m % PIECES;
					if (m < PIECES) *(u32x4*)(lds + (N % 3 == 0 ? to0[i] : N % 3 == 1 ? to1[i] : to2[i])) = g.w[i];
					else if (m < 2 * PIECES) g.w[i] = load(i);
				} else {
					const int n = read / 3, i = first < STEPS ? first + n : n;
					if (read % 3 == 0) kop[at][n] = key_operand(first < STEPS ? ON1 : ON2, i);
					else value_operand(vop[at][n], first < STEPS ? ON2 : HERE, i, read % 3 - 1);
				}
			}
			__builtin_amdgcn_sched_barrier(0);
		};
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (int i = 0; i < STEPS; ++i) {
			const int batch = i / BATCH, n = i % BATCH;
			next.s = product(kop[batch % 2][n], q[i], next.s, T{});
			slot(2 * i);
			o[i / 2] = product(vop[batch % 2][n], before.w[i % 2], o[i / 2], T{});
			slot(2 * i + 1);
		}
		/* a sum that is no more than 2^(LIFT + RISE) has no weight above it: no need to look for the largest score. (Weights of scores far from zero are made here only.) */
		if (__any(!(sum <= most_sum))) {
			raise(now);
			lower(now);
			weigh(weights, sum, now);
		}
		l += sum;
	};

	if (wave == 0) strange = 0;
	__syncthreads();
	if (end) {
		for (int c = 0; c < 2; ++c) w1.w[c] = u32x4{ 0, 0, 0, 0 };
		/* the first tiles: three of keys, one of values. (Whole wavefronts take part or do not: where lanes leave a loop one by one the compiler has put copies of registers behind it, to the
		 * other half of the file, before the lanes are back.) */
		auto bring_tile = [&](const uint16_t* rows, uint32_t tile, uint32_t place, uint32_t row, bool checked) {
			for (uint32_t first = WAVE * wave; first < TILE_PIECES; first += THREADS) {
				const uint32_t piece = first + lane, token = piece / (4 * J), at_row = piece % (4 * J);
				u32x4 w = load_raw8(rows + (size_t)min(32 * (start + tile) + token, p.tokens - 1) * a.token_stride + 8 * at_row, VEC);
				if (checked && (int32_t)(32 * (start + tile) + 32) > all_see && __any(without_strange<T>(w))) strange = 1;
				*(u32x4*)(lds + place + token * row + 16 * at_row) = w;
			}
		};
		for (uint32_t n = 0; n < 3; ++n) bring_tile(key_rows, n, n * PLACE, KROW, false);
		bring_tile(value_rows, 0, KTILE, VROW, true);
		for (uint32_t first = WAVE * wave; first < TILE_PIECES; first += THREADS) { /* (nothing before the first tile) */
			const uint32_t piece = first + lane;
			*(u32x4*)(lds + 2 * PLACE + KTILE + piece / (4 * J) * VROW + 16 * (piece % (4 * J))) = u32x4{ 0, 0, 0, 0 };
		}
		auto fetch = [&](Staged& g) {
#pragma unroll
			for (int i = 0; i < PIECES; ++i) g.w[i] = load(i);
		};
		fetch(g0);
		fetch(g1);
		__syncthreads();
		/* the last step of a wavefront adds up its last tile (and sees no tokens itself); those with fewer tiles only bring theirs */
		const uint32_t steps = end + 1, my_steps = mine ? mine + 1 : 0;
		if (mine) {
			score(s0, 0);
			hide(s0, 0);
			raise(s0);
#pragma unroll
			for (int n = 0; n < BATCH; ++n) {
				kop[0][n] = key_operand(PLACE, n);
				for (int half = 0; half < 2; ++half) value_operand(vop[0][n], 2 * PLACE, n, half);
			}
		}
		__syncthreads();
		uint32_t tile = 0;
		auto step = [&](auto number) {
			check(decltype(number)::value % 2 ? g1 : g0, tile + 1);
			work(number, tile);
			/* what was stored to LDS is there: of what LDS was asked for since, the last batch's reads are for the next step and need not be back */
			constexpr int LATE = 3 * BATCH < 14 ? 3 * BATCH : 14;
			asm volatile("s_waitcnt lgkmcnt(%0)\n\ts_barrier" :: "n"(LATE) : "memory");
			return ++tile < my_steps;
		};
		while (tile < my_steps)
			if (!step(std::integral_constant<uint32_t, 0>{}) || !step(std::integral_constant<uint32_t, 1>{}) || !step(std::integral_constant<uint32_t, 2>{}) ||
			    !step(std::integral_constant<uint32_t, 3>{}) || !step(std::integral_constant<uint32_t, 4>{}) || !step(std::integral_constant<uint32_t, 5>{}))
				break;
		auto bring = [&](Staged& g) {
			check(g, tile + 1);
#pragma unroll
			for (int i = 0; i < PIECES; ++i) {
				const uint32_t place = (tile + (values[i] ? AHEAD_VALUES : 0)) % 3;
				*(u32x4*)(lds + to[i] + (WAVE * wave + THREADS * i < 2 * TILE_PIECES ? place * PLACE : 0)) = g.w[i];
			}
			fetch(g);
			__syncthreads();
		};
		for (; tile < steps; ++tile) {
			if (tile % 2) bring(g1);
			else bring(g0);
		}
	}

	if (strange) { /* infinities and NaN come to the rows that see them (their weights are above 0, however small) */
#pragma unroll 1
		for (uint32_t t = max((uint32_t)all_see / 32, start) * 32; t < p.tokens && t < (uint32_t)limit; ++t) {
			const uint16_t* from = value_rows + (size_t)t * a.token_stride;
#pragma unroll
			for (int j = 0; j < J; ++j)
#pragma unroll
				for (int e = 0; e < 16; ++e) {
					const float x = raw_element(from[32 * j + 8 * (e / 4) + 4 * h + e % 4], false, __is_same(T, __bf16));
					const bool number = fabsf(x) <= 3.4028235e38f;
					o[j][e] += !number && (int32_t)t < sees ? x : 0.0f;
				}
		}
	}

	/* what the end needs is read and worked out here, and takes up no registers in the loop */
	auto last = (const __attribute__((address_space(4))) PromptAttend*)__builtin_amdgcn_kernarg_segment_ptr();
	asm volatile("" : "+s"(last));
	const uint32_t id = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), n = id % 32, half = id / 32, r = wave_first + n;
	l += __shfl_xor(l, 32);
	if (r >= rows) return;
	const float reference = fminf(fmaf(shift, last->factor, LIFT - base), NOTHING); /* (of a row without a weight the lowest number) */
	if (last->parts > 1) { /* [unit][part]: [ROWS][channel] sums, [ROWS] of reference and sum of weights, for prompt_join_kernel */
		float* const to = last->partial + ((size_t)unit * last->parts + part) * (ROWS * (32 * J + 2));
#pragma unroll
		for (int j = 0; j < J; ++j)
			for (int e = 0; e < 4; ++e)
				*(f32x4*)(to + (size_t)r * (32 * J) + 32 * j + 8 * e + 4 * half) = f32x4{ o[j][4 * e], o[j][4 * e + 1], o[j][4 * e + 2], o[j][4 * e + 3] };
		if (half == 0) *(float2*)(to + ROWS * (32 * J) + 2 * r) = float2{ reference, l };
		return;
	}
	const float by = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l; /* a row that sees nothing is zero; NaN stays */
	const uint32_t in = (first_row + r) / last->group, out_head = head * last->group + (first_row + r - in * last->group);
	uint16_t* const row = (uint16_t*)last->out + (size_t)(p.query_first + in) * last->out_token + (size_t)out_head * last->out_head;
#pragma unroll
	for (int j = 0; j < J; ++j)
		for (int e = 0; e < 4; ++e) {
			const uint32_t low = rounded_pair(o[j][4 * e] * by, o[j][4 * e + 1] * by, T{}), high = rounded_pair(o[j][4 * e + 2] * by, o[j][4 * e + 3] * by, T{});
			uint16_t* at = row + 32 * j + 8 * e + 4 * half;
			if constexpr (VEC) *(u32x2*)at = u32x2{ low, high };
			else {
				at[0] = (uint16_t)low;
				at[1] = (uint16_t)(low >> 16);
				at[2] = (uint16_t)high;
				at[3] = (uint16_t)(high >> 16);
			}
		}
	if (half == 0 && last->lse)
		last->lse[(size_t)(p.query_first + in) * last->query_heads + out_head] = l == 0.0f ? -__builtin_inff() : (reference + log2f(l) - LIFT) * 0.693147180559945309f;
}

/* The parts of 32 W rows: a wavefront a row, 8 J lanes 4 channels each of every (64 / 8 J)-th part. */
template <typename T, int J, int W>
__global__ void __launch_bounds__(256)
prompt_join_kernel(PromptAttend a)
{
	constexpr uint32_t D = 32 * J, ROWS = 32 * W, LANES = 8 * J, GROUPS = WAVE / LANES;
	constexpr size_t PART = ROWS * (D + 2);
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE;
	const uint32_t unit = blockIdx.x / (ROWS / 4), r = blockIdx.x % (ROWS / 4) * 4 + wave;
	const uint32_t head = unit % a.heads, rest = unit / a.heads, s = rest % a.sequences, row_tile = a.row_tiles - 1 - rest / a.sequences;
	const Prompt4 p = prompt_of(a, s);
	const uint32_t all_rows = p.queries * a.group, first_row = row_tile * ROWS;
	if (first_row + r >= all_rows) return;
	const uint32_t rows = min(ROWS, all_rows - first_row), tiles = ((uint32_t)sees_of(a, p, (first_row + rows - 1) / a.group) + 31) / 32;
	const uint32_t parts = tiles ? (tiles + a.tiles_per_part - 1) / a.tiles_per_part : 1, group = lane / LANES, at = lane % LANES;
	const float* const left = a.partial + (size_t)unit * a.parts * PART;
	float top = -__builtin_inff();
	for (uint32_t n = lane; n < parts; n += WAVE) top = fmaxf(top, left[n * PART + ROWS * D + 2 * r]);
	for (int d = 1; d < WAVE; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
	float sum = 0.0f;
	f32x4 mine{ 0.0f, 0.0f, 0.0f, 0.0f };
	if (group < GROUPS)
#pragma unroll 4
		for (uint32_t n = group; n < parts; n += GROUPS) {
			const float* from = left + n * PART;
			const float2 ml = *(const float2*)(from + ROWS * D + 2 * r);
			const float weight = __builtin_amdgcn_exp2f(ml.x - top);
			sum += ml.y * weight;
			mine += *(const f32x4*)(from + (size_t)r * D + 4 * at) * weight;
		}
	for (uint32_t g = 1; g < GROUPS; ++g) { /* the groups' sums, in their order */
		const int other = (int)(at + g * LANES);
		const f32x4 more{ __shfl(mine[0], other), __shfl(mine[1], other), __shfl(mine[2], other), __shfl(mine[3], other) };
		const float more_sum = __shfl(sum, other);
		if (group == 0) { mine += more; sum += more_sum; }
	}
	if (group != 0) return;
	const float by = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;
	const uint32_t query = (first_row + r) / a.group, query_head = head * a.group + (first_row + r - query * a.group);
	uint16_t* to = (uint16_t*)a.out + (size_t)(p.query_first + query) * a.out_token + (size_t)query_head * a.out_head + 4 * at;
	const uint32_t low = rounded_pair(mine[0] * by, mine[1] * by, T{}), high = rounded_pair(mine[2] * by, mine[3] * by, T{});
	to[0] = (uint16_t)low;
	to[1] = (uint16_t)(low >> 16);
	to[2] = (uint16_t)high;
	to[3] = (uint16_t)(high >> 16);
	if (at == 0 && a.lse) a.lse[(size_t)(p.query_first + query) * a.query_heads + query_head] = sum == 0.0f ? -__builtin_inff() : (top + log2f(sum) - LIFT) * 0.693147180559945309f;
}

template <typename T, int J, int W, bool VEC>
static int launch_prompt_kernel(const PromptAttend& a, uint32_t units)
{
	constexpr uint32_t bytes = prompt_lds<J>();
	if (bytes > 65536 - 64) { /* more LDS than a launch may ask for unannounced, on this device */
		static int allowed = -1;
		const DeviceInfo* dev = nullptr;
		const int rc = device_info(&dev);
		if (rc) return rc;
		if (allowed != dev->device) {
			KMX_HIP(hipFuncSetAttribute((const void*)prompt_attend_kernel<T, J, W, VEC>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
			allowed = dev->device;
		}
	}
	KMX_LAUNCH_KERNEL((prompt_attend_kernel<T, J, W, VEC>), dim3(units), dim3(64 * W), bytes, stream(), a);
	KMX_LAUNCH_CHECK("prompt_attend_kernel");
	return KMX_OK;
}

template <typename T, int J, int W>
static int launch_prompt_rows(PromptAttend a, const PromptPlan& plan)
{
	a.row_tiles = plan.row_tiles;
	a.units = plan.units;
	a.parts = plan.parts;
	a.tiles_per_part = plan.tiles_per_part;
	const int rc = a.vec ? launch_prompt_kernel<T, J, W, true>(a, plan.units * plan.parts) : launch_prompt_kernel<T, J, W, false>(a, plan.units * plan.parts);
	if (rc || plan.parts == 1) return rc;
	KMX_LAUNCH_KERNEL((prompt_join_kernel<T, J, W>), dim3(plan.units * (32 * W / 4)), dim3(256), 0, stream(), a);
	KMX_LAUNCH_CHECK("prompt_join_kernel");
	return KMX_OK;
}

template <typename T, int J>
static int launch_prompt_of(const PromptAttend& a, const PromptPlan& plan)
{
	if constexpr (J == 5 || J == 6) return launch_prompt_rows<T, J, 8>(a, plan);
	else {
		if constexpr (J == 3 || J == 4)
			if (plan.wide) return launch_prompt_rows<T, J, 8>(a, plan);
		return launch_prompt_rows<T, J, 4>(a, plan);
	}
}

template <int J>
int launch_prompt_attend(const PromptAttend& a, bool bf16, const PromptPlan& plan)
{
	return bf16 ? launch_prompt_of<__bf16, J>(a, plan) : launch_prompt_of<_Float16, J>(a, plan);
}

} // namespace kmx

#endif
