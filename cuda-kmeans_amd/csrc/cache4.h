/*
 * The 4-bit cache on the device (kmx_cache4_* of include/kmx.h): where a block keeps what, and how codes become numbers.
 *
 * A block is 16 tokens of one head, 18 dim bytes (J = dim / 32 groups of 32 channels):
 *   [0, 8 dim)        codes of the keys, token by token: dim / 2 bytes, word J g + j holds channels 32 j + 8 g .. + 7 (byte b: channel b in the
 *                     low nibble, b + 4 in the high one). A lane of a matrix instruction wants 8 channels of one token for each j: its J
 *                     words lie side by side.
 *   [8 dim, 16 dim)   codes of the values, pair by pair: pair 16 j + i holds channels 32 j + i (low) and 32 j + 16 + i (high), one byte a
 *                     token. A lane of the second product wants tokens of one channel, and a token that is written touches no byte of another.
 *   [16 dim, 17 dim)  scales of the keys, half precision, [token][j];  [17 dim, 18 dim) scales of the values, [j][token]
 * A scale has 5 significant bits and a magnitude 6, so that their product is a number of half precision from 2^-14 on: the matrix cores take the very
 * values that the cache stands for, smaller ones to the nearest multiple of 2^-24.
 */
#ifndef KMX_CACHE4_H
#define KMX_CACHE4_H

#include "kmx_internal.h"
#include "cache4_plan.h"

namespace kmx {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

struct Cache4 {
	uint8_t* blocks;
	int8_t* bounds;         /* [page][head][2 dim], may be null */
	float* bound_scales;    /* [page][head] */
	const uint16_t* levels; /* [head][keys, values][8], half precision */
	uint32_t heads, page_count, page_shift; /* log2 of the tokens of a page */
};

template <int J>
__device__ __forceinline__ size_t block_offset(const Cache4& c, uint32_t page, uint32_t head, uint32_t sub)
{
	return ((((size_t)page * c.heads + head) << (c.page_shift - 4)) + sub) * (576u * J);
}

/* The 8 magnitudes of a head as two tables of bytes that v_perm_b32 looks up */
struct Magnitudes { uint32_t lo0, lo1, hi0, hi1; };

__device__ __forceinline__ Magnitudes load_magnitudes(const uint16_t* levels, uint32_t head, uint32_t which)
{
	const u32x4 w = *(const u32x4*)(levels + ((size_t)head * 2 + which) * 8);
	return { __builtin_amdgcn_perm(w[1], w[0], 0x06040200u), __builtin_amdgcn_perm(w[3], w[2], 0x06040200u),
	         __builtin_amdgcn_perm(w[1], w[0], 0x07050301u), __builtin_amdgcn_perm(w[3], w[2], 0x07050301u) };
}

/* The four codes in the low nibbles of w (high = false), or in the high ones, as two pairs of halves. 7 instructions for 4 numbers: mask, two
 * look-ups of a byte each, the sign bit, and two that put the bytes side by side. */
template <bool HIGH>
__device__ __forceinline__ void unpack4(uint32_t w, const Magnitudes& m, uint32_t& first, uint32_t& second)
{
	const uint32_t index = (HIGH ? w >> 4 : w) & 0x07070707u;
	const uint32_t lo = __builtin_amdgcn_perm(m.lo1, m.lo0, index);
	const uint32_t hi = __builtin_amdgcn_perm(m.hi1, m.hi0, index) | (HIGH ? w & 0x80808080u : (w & 0x08080808u) << 4);
	first = __builtin_amdgcn_perm(hi, lo, 0x05010400u);
	second = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
}

__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b)
{
	return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, a) * __builtin_bit_cast(half2v, b));
}

__device__ __forceinline__ uint32_t twice(uint32_t half_word, bool upper) /* one half of a word in both */
{
	return __builtin_amdgcn_perm(half_word, half_word, upper ? 0x07060706u : 0x05040504u);
}

/* between what lanes of a wavefront write to LDS and what others of it read there (LDS takes a wavefront's accesses in their order; this keeps
 * the compiler to it) */
__device__ __forceinline__ void wave_sync()
{
	__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
	__builtin_amdgcn_wave_barrier();
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v)
{
	return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v)
{
	return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, false);
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E; /* inside groups of 4 lanes */

/* 8 elements of a caller's row of 16 bits each as they are, two a word; vec: 16-byte aligned */
__device__ __forceinline__ u32x4 load_raw8(const uint16_t* p, bool vec)
{
	if (vec) return *(const u32x4*)p;
	u32x4 w;
	for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
	return w;
}
__device__ __forceinline__ float raw_element(uint32_t w, bool upper, bool bf16)
{
	if (bf16) return __builtin_bit_cast(float, upper ? w & 0xFFFF0000u : w << 16);
	return (float)__builtin_bit_cast(_Float16, (uint16_t)(upper ? w >> 16 : w));
}

/* rounded to the nearest, ties to even; NaN stays NaN */
__device__ __forceinline__ uint32_t bf16_bits(float v)
{
	const uint32_t u = __builtin_bit_cast(uint32_t, v);
	if (v != v) return (u >> 16) | 0x40u;
	return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
template <typename T>
__device__ __forceinline__ uint32_t bits16(float v)
{
	if constexpr (__is_same(T, __bf16)) return bf16_bits(v);
	else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float x[8])
{
	if constexpr (sizeof(T) == 4) {
		if (vec) {
			__builtin_nontemporal_store(f32x4{ x[0], x[1], x[2], x[3] }, (f32x4*)p);
			__builtin_nontemporal_store(f32x4{ x[4], x[5], x[6], x[7] }, (f32x4*)(p + 4));
		} else
			for (int i = 0; i < 8; ++i) p[i] = x[i];
	} else {
		uint32_t b[8];
		for (int i = 0; i < 8; ++i) b[i] = bits16<T>(x[i]);
		if (vec) __builtin_nontemporal_store(u32x4{ b[0] | b[1] << 16, b[2] | b[3] << 16, b[4] | b[5] << 16, b[6] | b[7] << 16 }, (u32x4*)p);
		else
			for (int i = 0; i < 8; ++i) ((uint16_t*)p)[i] = (uint16_t)b[i];
	}
}

/* What a batch of queries sees of the cache */
struct Batch4 {
	const int32_t* starts;  /* sequences + 1 */
	const int32_t* lengths; /* sequences */
	const int32_t* table;   /* sequences x table_stride */
	uint32_t sequences, tokens, max_queries, table_stride, max_length;
	uint32_t group, query_heads; /* query heads per head of the cache */
	bool causal;
};

/* queries and cached tokens of sequence b, held to what the buffers have room for */
struct Sequence { uint32_t first, queries, length; };
/* numbers that no kernel writes while another reads them: scalar loads also behind stores, where an index is the same in all lanes */
typedef const __attribute__((address_space(4))) int32_t* Constant4;
__device__ __forceinline__ Constant4 constant4(const int32_t* p) { return (Constant4)(uint64_t)p; }

__device__ __forceinline__ Sequence sequence_of(const Batch4& b, uint32_t s, uint32_t page_shift)
{
	const int32_t from = constant4(b.starts)[s], to = constant4(b.starts)[s + 1], length = constant4(b.lengths)[s];
	Sequence q{ 0, 0, 0 };
	if (from >= 0 && to > from && (uint32_t)to <= b.tokens) {
		q.first = (uint32_t)from;
		q.queries = (uint32_t)(to - from);
		if (q.queries > b.max_queries) q.queries = b.max_queries;
	}
	if (length > 0) {
		const uint64_t room = min((uint64_t)b.table_stride << page_shift, (uint64_t)b.max_length);
		q.length = (uint64_t)length < room ? (uint32_t)length : (uint32_t)room;
	}
	return q;
}
/* tokens that query i of the sequence sees */
__device__ __forceinline__ uint32_t visible_to(const Batch4& b, const Sequence& q, uint32_t i)
{
	if (!b.causal) return q.length;
	const int64_t n = (int64_t)q.length - q.queries + i + 1;
	return n > 0 ? (uint32_t)n : 0;
}

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

/* cache4.hip: the checks of the entry points, and the work space of a call */
int check_cache4(const char* who, const kmx_cache4* cache, Cache4* out);
int check_batch4(const char* who, const kmx_cache4* cache, const kmx_cache4_batch* batch, int causal, Batch4* out);
int check_type(const char* who, int type, bool floats);
bool aligned_rows(const void* p, size_t token_stride, size_t head_stride, size_t size);
int place_cache4(const char* who, size_t floats, float** partials, const char* reserve = "kmx_cache4_reserve");

/* cache4_attend_impl.h, one object per J: see there */
struct Attend4 {
	Cache4 cache;
	Batch4 batch;
	const void* q; size_t q_token, q_head;
	void* out; size_t out_token, out_head;
	float* lse;
	const int32_t* chosen; uint32_t top; /* pages chosen for each token and head, or null */
	float scale;
	bool bf16, vec;
	uint32_t row_tiles, splits, tiles_per_split; /* (filled in by the launcher) */
	bool joined; /* parts of many rows are left to the kernel that joins them */
	float* partial; /* sums of parts, where there are any */
	/* prefixes that sequences share: what their attention leaves (no prefix_starts), and what that of the sequences' own tokens is joined with */
	float* rows; float* row_sums; /* [token][query head][channel], and of each row the largest score (to the base of 2) and the sum; null: no prefix */
	const int32_t* prefix_starts; uint32_t prefixes, prefix_queries;
};
template <int J> int launch_attend4(Attend4 a, const Plan4& plan);

} // namespace kmx

#endif
