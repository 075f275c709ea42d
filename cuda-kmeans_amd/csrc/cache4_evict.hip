/*
 * What of the 4-bit cache is kept (kmx_cache4_weigh, kmx_cache4_evict of include/kmx.h): attention weights added up token by token, and the choice and the moves by
 * which a sequence gets back to its budget.
 */
#include "cache4.h"

#include <cmath>

namespace kmx {

/* ---------------------------------------------------------------- weights ------------------------ */

struct Weigh4 {
	Cache4 cache;
	Batch4 batch;
	const void* q; size_t q_token, q_head;
	const float* lse;
	float* weights; /* [page][head][token of the page] */
	float scale;
	bool bf16, vec;
};

constexpr uint32_t WEIGH_TOKENS = 256; /* of a work-group, 64 a wavefront */

/*
 * A work-group takes 256 tokens of one head of a sequence, whose keys its wavefronts unpack once and keep, four blocks each; the rows (query heads of the head, of all queries)
 * come by 64 at a time through LDS, a tile of 16 from each wavefront. The keys are the second operand (v_mfma_f32_16x16x32_f16): scores come out as [row][token], so that
 * the weights of a token, 2^(c s - log2(e) lse), are added up in the lane that has it, and four lanes at the end. Rows are asked for before the keys are unpacked.
 * Bound by the chain length - table - codes - products of its work-groups, three rounds of them, at 32 sequences of up to 2048 tokens (13.8 us; the packed keys alone take 5); 32 queries over
 * 32768 tokens 18.8 us, vector units busy 42 % of it (powers 13 %), matrix cores 13 %: each work-group makes halves of the same rows of queries, 64 between two barriers. 128 tokens a work-group instead of 256: 16.9 for 15.6 and 141 for 116 (64 x 8192); 256 after 256 by the same work-groups: 17.5 for 15.6.
 */
template <int J>
__global__ void __launch_bounds__(256)
weigh4_kernel(Weigh4 a)
{
	constexpr uint32_t D = 32 * J;
	__shared__ half8v queries[4][J][WAVE];
	__shared__ float factors[4][16], sums[4][16];
	__shared__ int32_t looks[4][16];
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE, i16 = lane % 16, kg = lane / 16;
	const uint32_t head = blockIdx.x, s = blockIdx.y, from = blockIdx.z * WEIGH_TOKENS;
	const Sequence seq = sequence_of(a.batch, s, a.cache.page_shift);
	if (seq.queries == 0 || from >= visible_to(a.batch, seq, seq.queries - 1)) return;
	const int32_t least = (int32_t)visible_to(a.batch, seq, 0);

	/* a row of 16 for the wavefront, of those from `first` on: asked for before what is to be done in the meantime */
	const uint64_t rows = (uint64_t)seq.queries * a.batch.group;
	u32x4 raw[J];
	float lse = 0.0f;
	int32_t look = 0;
	bool there = false;
	auto fetch = [&](uint64_t first) {
		if (first + 16 * wave >= rows) return;
		const uint64_t row = first + 16 * wave + i16;
		there = row < rows;
		const uint32_t token = there ? (uint32_t)row / a.batch.group : 0, query_head = head * a.batch.group + (there ? (uint32_t)row - token * a.batch.group : 0);
		const uint16_t* p = (const uint16_t*)a.q + (size_t)(seq.first + token) * a.q_token + (size_t)query_head * a.q_head + 8 * kg;
		lse = a.lse[(size_t)(seq.first + token) * a.batch.query_heads + query_head];
		if (a.vec) {
#pragma unroll
			for (int j = 0; j < J; ++j) raw[j] = load_raw8(p + 32 * j, true);
		} else {
#pragma unroll
			for (int j = 0; j < J; ++j) raw[j] = load_raw8(p + 32 * j, false);
		}
		look = there ? (int32_t)visible_to(a.batch, seq, token) : 0;
	};
	fetch(0);

	/* the wavefront's blocks */
	const Constant4 table = constant4(a.batch.table) + (size_t)s * a.batch.table_stride;
	const uint32_t sub_bits = a.cache.page_shift - 4, begin = from + 64 * wave;
	const Magnitudes mag = load_magnitudes(a.cache.levels, head, 0);
	half8v keys[4][J];
	bool known[4];
	size_t to[4];
	const bool some = begin < seq.length;
	if (some) {
		uint32_t pages[4];
#pragma unroll
		for (int b = 0; b < 4; ++b) pages[b] = (uint32_t)table[min((begin / 16 + b) >> sub_bits, a.batch.table_stride - 1)];
#pragma unroll
		for (int b = 0; b < 4; ++b) {
			const uint32_t n = begin / 16 + b, entry = n >> sub_bits, sub = n & ((1u << sub_bits) - 1), page = pages[b];
			known[b] = 16 * n < seq.length && entry < a.batch.table_stride && page < a.cache.page_count;
			const uint8_t* block = a.cache.blocks + block_offset<J>(a.cache, known[b] ? page : 0, head, known[b] ? sub : 0);
			to[b] = (((size_t)(known[b] ? page : 0) * a.cache.heads + head) << a.cache.page_shift) + 16 * sub;
			uint32_t codes[J];
			if constexpr (J % 4 == 0) {
				for (int i = 0; i < J / 4; ++i) { const u32x4 v = ((const u32x4*)(block + i16 * (D / 2) + kg * 4 * J))[i]; for (int e = 0; e < 4; ++e) codes[4 * i + e] = v[e]; }
			} else {
				for (int j = 0; j < J; ++j) codes[j] = ((const uint32_t*)(block + i16 * (D / 2) + kg * 4 * J))[j];
			}
			const uint16_t* scales = (const uint16_t*)(block + 16 * D) + i16 * J;
#pragma unroll
			for (int j = 0; j < J; ++j) {
				uint32_t p[4];
				unpack4<false>(codes[j], mag, p[0], p[1]);
				unpack4<true>(codes[j], mag, p[2], p[3]);
				const uint32_t scale = scales[j] | (uint32_t)scales[j] << 16;
				keys[b][j] = __builtin_bit_cast(half8v, u32x4{ times(p[0], scale), times(p[1], scale), times(p[2], scale), times(p[3], scale) });
			}
		}
	}
	float w[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
	const bool cut = (int32_t)(begin + 64) > least; /* not all queries see all of the wavefront's tokens */
	for (uint64_t first = 0; first < rows; first += 64) {
		__syncthreads(); /* (the rows before are done with) */
		if (first + 16 * wave < rows) {
			float x[J][8], largest = 0.0f;
			auto take = [&](bool bf16) { /* (one question for all of them) */
#pragma unroll
				for (int j = 0; j < J; ++j)
					for (int e = 0; e < 8; ++e) x[j][e] = raw_element(there ? raw[j][e / 2] : 0u, e % 2, bf16);
			};
			if (a.bf16) take(true);
			else take(false);
#pragma unroll
			for (int j = 0; j < J; ++j)
				for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(x[j][e]));
			largest = fmaxf(largest, __shfl_xor(largest, 16));
			largest = fmaxf(largest, __shfl_xor(largest, 32));
			float factor;
			const float by = query_scale(a.scale, largest, &factor);
#pragma unroll
			for (int j = 0; j < J; ++j) {
				half8v v;
				for (int e = 0; e < 8; ++e) v[e] = (_Float16)(x[j][e] * by);
				queries[wave][j][lane] = v;
			}
			if (kg == 0) {
				factors[wave][i16] = factor;
				sums[wave][i16] = there ? -1.44269504088896341f * lse : -__builtin_inff(); /* no such row: no weight */
				looks[wave][i16] = look;
			}
			fetch(first + 64);
		}
		__syncthreads();
		if (!some) continue;
		const uint32_t tiles = (uint32_t)min((uint64_t)4, (rows - first + 15) / 16);
		for (uint32_t n = 0; n < tiles; ++n) {
			f32x4 sc[4];
#pragma unroll
			for (int b = 0; b < 4; ++b) sc[b] = f32x4{ 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
			for (int j = 0; j < J; ++j) {
				const half8v v = queries[n][j][lane];
#pragma unroll
				for (int b = 0; b < 4; ++b) sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, keys[b][j], sc[b], 0, 0, 0);
			}
			const f32x4 factor = *(const f32x4*)&factors[n][4 * kg], less = *(const f32x4*)&sums[n][4 * kg];
			if (cut) {
				const i32x4 look = *(const i32x4*)&looks[n][4 * kg];
#pragma unroll
				for (int b = 0; b < 4; ++b)
					for (int r = 0; r < 4; ++r) {
						const float p = __builtin_amdgcn_exp2f(fmaf(sc[b][r], factor[r], less[r]));
						w[b] += (int32_t)(begin + 16 * b + i16) < look[r] ? p : 0.0f;
					}
			} else {
#pragma unroll
				for (int b = 0; b < 4; ++b)
					for (int r = 0; r < 4; ++r) w[b] += __builtin_amdgcn_exp2f(fmaf(sc[b][r], factor[r], less[r]));
			}
		}
	}
	if (!some) return;
	float mine = 0.0f;
	size_t at = 0;
	bool store = false;
#pragma unroll
	for (int b = 0; b < 4; ++b) {
		w[b] += __shfl_xor(w[b], 16);
		w[b] += __shfl_xor(w[b], 32);
		if ((int)kg == b) { mine = w[b]; at = to[b]; store = known[b] && begin + 16 * b + i16 < seq.length; }
	}
	/* one addition to a token of a sequence; of a page that several sequences have, each adds its own */
	if (store) unsafeAtomicAdd(a.weights + at + i16, mine);
}

/* ---------------------------------------------------------------- choice ------------------------- */

struct Evict4 {
	Cache4 cache;
	const int32_t* lengths;
	const int32_t* table;
	float* weights;
	int32_t* kept; /* [sequence][head][keep] */
	int32_t* left; /* [sequence] */
	uint32_t sequences, table_stride, max_length, keep, first, recent;
	uint32_t words, cached; /* LDS: words of 64 places, weights */
};

constexpr uint32_t EVICT_THREADS = 1024, EVICT_WAVES = EVICT_THREADS / WAVE, EVICT_BINS = 2048;
constexpr uint32_t EVICT_CACHED = 24576;   /* weights of a sequence that LDS holds: 96 KB, and 24 KB for which of them move */
constexpr uint32_t EVICT_TOKENS = 1 << 18; /* of a sequence */
constexpr uint32_t EVICT_WORD = 24;        /* bytes for 64 places: those that stay, those at the threshold, free and moving ones before */
constexpr uint32_t evict_bytes(uint32_t words, uint32_t cached) { return EVICT_WORD * words + 4 * cached + 2 * ((cached / 2 + 1) / 2 * 2); }
constexpr uint32_t MOST_EVICT_BYTES = EVICT_TOKENS / 64 * EVICT_WORD > evict_bytes(EVICT_CACHED / 64, EVICT_CACHED) ? EVICT_TOKENS / 64 * EVICT_WORD : evict_bytes(EVICT_CACHED / 64, EVICT_CACHED);

__device__ __forceinline__ uint32_t evict_length(const Evict4& e, uint32_t s)
{
	const int32_t n = constant4(e.lengths)[s];
	const uint64_t room = min((uint64_t)e.table_stride << e.cache.page_shift, (uint64_t)e.max_length);
	return n > 0 ? (uint32_t)min((uint64_t)n, room) : 0;
}
/* where place t of a sequence's tokens has its weight; false: its page is not there */
__device__ __forceinline__ bool weight_of(const Evict4& e, const int32_t* table, uint32_t head, uint32_t t, size_t* at)
{
	const uint32_t page = (uint32_t)table[t >> e.cache.page_shift];
	*at = (((size_t)page * e.cache.heads + head) << e.cache.page_shift) + (t & ((1u << e.cache.page_shift) - 1));
	return page < e.cache.page_count;
}
/* whole numbers in the order of the weights; NaN, and pages that are not there: the lowest */
__device__ __forceinline__ uint32_t key_of(float w)
{
	const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f); /* (one zero) */
	return w != w ? 0 : u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint32_t sum_below(const uint32_t* counts, uint32_t wave)
{
	uint32_t sum = 0;
#pragma unroll
	for (uint32_t w = 0; w < EVICT_WAVES; ++w) sum += w < wave ? counts[w] : 0; /* (all are read at once) */
	return sum;
}
__device__ __forceinline__ uint64_t lanes_below(uint32_t lane) { return ((uint64_t)1 << lane) - 1; }

/* sums of what the threads before have; EVICT_WAVES counts */
__device__ __forceinline__ uint32_t sum_before(uint32_t mine, uint32_t* counts, uint32_t wave, uint32_t lane)
{
	int v = (int)mine; /* within rows of 16 lanes, then from row to row */
	v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
	v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
	v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
	v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
	v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
	v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
	const uint32_t upto = (uint32_t)v;
	if (lane == WAVE - 1) counts[wave] = upto;
	__syncthreads();
	return sum_below(counts, wave) + upto - mine;
}

/*
 * One work-group a sequence and head. The threshold of the weights by counting them in 2048 equal shares of the range of their keys, then of the share that it lies in:
 * three rounds at most. Then, for 64 places a word: which stay (of those at the threshold the first ones), how many places below the edge become free before them and how many
 * tokens from the edge on have to move. The n-th moving one goes to the n-th free place. Up to 24576 weights stay in LDS, with the list of those that move; else the list is the begin of
 * `kept`, from where it goes to the free places, the highest first: none of them lies below where it is listed.
 * Bound by latency (one work-group a compute unit, few of them): weights come eight at a time, all that is written depends on LDS alone.
 * 16384 tokens to 4096, 32 work-groups: 24 us (weights 4, the threshold 10 in three rounds, words 4, places and lists 3, what is written 3); 1025 to 1024: 10 (5 of them the threshold).
 */
__global__ void __launch_bounds__(EVICT_THREADS)
evict4_choose_kernel(Evict4 e)
{
	extern __shared__ __attribute__((aligned(16))) uint32_t lds[]; /* words of 64 places, weights, a list of tokens */
	__shared__ uint32_t bins[EVICT_BINS], counts[4][EVICT_WAVES], found[3];
	const uint32_t tid = threadIdx.x, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid / WAVE)), lane = tid % WAVE;
	const uint32_t head = blockIdx.x, s = blockIdx.y, n = evict_length(e, s);
	int32_t* const kept = e.kept + ((size_t)s * e.cache.heads + head) * e.keep;
	if (head == 0 && tid == 0) e.left[s] = (int32_t)min(n, e.keep);
	if (n <= e.keep) {
		for (uint32_t i = tid; i < e.keep; i += EVICT_THREADS) kept[i] = i < n ? (int32_t)i : -1;
		return;
	}
	const int32_t* table = e.table + (size_t)s * e.table_stride;
	const uint32_t edge = e.keep - e.recent, places = edge - e.first, rest = n - e.first - e.recent; /* `places` of the `rest` tokens stay: fewer */
	const uint32_t words = (rest + 63) / 64;
	uint64_t *const bits = (uint64_t*)lds, *const level = bits + e.words;
	uint32_t *const freed = (uint32_t*)(level + e.words), *const moved = freed + e.words;
	float* const cache = (float*)(moved + e.words);
	uint16_t* const list = (uint16_t*)(cache + e.cached);
	const bool cached = rest <= e.cached;
	auto weight_at = [&](uint32_t t) {
		size_t at;
		return weight_of(e, table, head, t, &at) ? e.weights[at] : __builtin_nanf("");
	};

	/* one more in a share. Many weights are alike (tokens that nothing has looked at yet have 0): those of the first lane's share are counted before they are added, since LDS adds to one
	 * address one after the other */
	auto count = [&](bool mine, uint32_t share) {
		const uint64_t some = __ballot(mine);
		if (!some) return;
		const int first = __ffsll((unsigned long long)some) - 1;
		const bool same = mine & (share == (uint32_t)__builtin_amdgcn_readlane((int)share, first));
		const uint32_t many = (uint32_t)__popcll(__ballot(same));
		if (mine & (!same | ((int)lane == first))) atomicAdd(&bins[share], same ? many : 1u);
	};
	constexpr int KEYS = 4; /* that a thread has at a time */
	auto keys_at = [&](uint32_t (&k)[KEYS], uint32_t x0) {
		float w[KEYS];
		if (cached) {
#pragma unroll
			for (int i = 0; i < KEYS; ++i) w[i] = cache[min(x0 + i * EVICT_THREADS + tid, rest - 1)];
		} else {
#pragma unroll
			for (int i = 0; i < KEYS; ++i) w[i] = weight_at(e.first + min(x0 + i * EVICT_THREADS + tid, rest - 1));
		}
#pragma unroll
		for (int i = 0; i < KEYS; ++i) k[i] = key_of(w[i]);
	};

	/* the weights, and the range of their keys */
	const float recent = tid < e.recent ? weight_at(n - e.recent + tid) : 0.0f; /* (the first of them) */
	if (tid < 2) found[tid] = tid ? 0u : ~0u;
	for (uint32_t i = tid; i < EVICT_BINS; i += EVICT_THREADS) bins[i] = 0;
	__syncthreads();
	uint32_t low = ~0u, high = 0;
	constexpr int AT_ONCE = 8;
	for (uint32_t x = tid; x < rest; x += AT_ONCE * EVICT_THREADS) {
		uint32_t page[AT_ONCE];
		float w[AT_ONCE];
#pragma unroll
		for (int i = 0; i < AT_ONCE; ++i) page[i] = (uint32_t)table[(e.first + min(x + i * EVICT_THREADS, rest - 1)) >> e.cache.page_shift];
#pragma unroll
		for (int i = 0; i < AT_ONCE; ++i) {
			const uint32_t t = e.first + min(x + i * EVICT_THREADS, rest - 1);
			const size_t at = (((size_t)(page[i] < e.cache.page_count ? page[i] : 0) * e.cache.heads + head) << e.cache.page_shift) + (t & ((1u << e.cache.page_shift) - 1));
			w[i] = e.weights[at];
		}
#pragma unroll
		for (int i = 0; i < AT_ONCE; ++i) {
			const float mine = page[i] < e.cache.page_count ? w[i] : __builtin_nanf("");
			const uint32_t k = key_of(mine), at = x + i * EVICT_THREADS;
			if (cached && at < rest) cache[at] = mine;
			low = min(low, k); /* (the last one counts again) */
			high = max(high, k);
		}
	}
	for (int d = 1; d < WAVE; d *= 2) {
		low = min(low, (uint32_t)__shfl_xor((int)low, d));
		high = max(high, (uint32_t)__shfl_xor((int)high, d));
	}
	if (lane == 0) {
		atomicMin(&found[0], low);
		atomicMax(&found[1], high);
	}
	__syncthreads();
	low = found[0];
	high = found[1];
	uint32_t need = places; /* of the tokens between low and high */
	while (need && low != high) { /* (the shares are zero here) */
		uint32_t shift = 0;
		while ((high - low) >> shift >= EVICT_BINS) ++shift;
		for (uint32_t x0 = 0; x0 < rest; x0 += KEYS * EVICT_THREADS) {
			uint32_t k[KEYS];
			keys_at(k, x0);
#pragma unroll
			for (int i = 0; i < KEYS; ++i) count((x0 + i * EVICT_THREADS + tid < rest) & (k[i] >= low) & (k[i] <= high), (k[i] - low) >> shift);
		}
		__syncthreads();
		/* the share that holds the need-th largest: thread t has shares 2047 - 2 t and the one below */
		const uint32_t upper = bins[EVICT_BINS - 1 - 2 * tid], lower = bins[EVICT_BINS - 2 - 2 * tid];
		bins[EVICT_BINS - 1 - 2 * tid] = bins[EVICT_BINS - 2 - 2 * tid] = 0;
		const uint32_t above = sum_before(upper + lower, counts[0], wave, lane);
		if (above < need && above + upper + lower >= need) {
			const bool first = above + upper >= need;
			found[0] = EVICT_BINS - (first ? 1 : 2) - 2 * tid;
			found[1] = need - above - (first ? 0 : upper);
		}
		__syncthreads();
		low += found[0] << shift;
		high = min(high, low + ((1u << shift) - 1));
		need = found[1];
	}
	const uint32_t threshold = need ? low : ~0u; /* above it all stay, at it the first `need` (without places: none) */

	for (uint32_t x0 = 0; x0 < rest; x0 += KEYS * EVICT_THREADS) {
		uint32_t k[KEYS];
		keys_at(k, x0);
#pragma unroll
		for (int i = 0; i < KEYS; ++i) {
			const uint32_t x = x0 + i * EVICT_THREADS + tid;
			const uint64_t above = __ballot((x < rest) & (k[i] > threshold)), at = __ballot((x < rest) & (k[i] == threshold));
			if (lane == 0 && x < rest) {
				bits[x / 64] = above;
				level[x / 64] = at;
			}
		}
	}
	__syncthreads();
	/* threads have words side by side, four at most */
	const uint32_t each = (words + EVICT_THREADS - 1) / EVICT_THREADS, word = tid * each, word_end = min(words, word + each);
	auto below_edge = [&](uint32_t w) { return 64 * w >= places ? (uint64_t)0 : places - 64 * w >= 64 ? ~(uint64_t)0 : lanes_below(places - 64 * w); };
	uint32_t mine = 0;
	for (uint32_t w = word; w < word_end; ++w) mine += (uint32_t)__popcll(level[w]);
	uint32_t before = sum_before(mine, counts[1], wave, lane), free_here = 0, move_here = 0;
	for (uint32_t w = word; w < word_end; ++w) {
		uint64_t at = level[w];
		const uint32_t count = (uint32_t)__popcll(at);
		for (uint32_t more = before >= need ? count : before + count > need ? before + count - need : 0; more; --more) at &= ~((uint64_t)1 << (63 - __clzll((long long)at))); /* the last ones go */
		before += count;
		const uint64_t bit = bits[w] | at, below = below_edge(w);
		bits[w] = bit;
		free_here += (uint32_t)__popcll(~bit & below);
		move_here += (uint32_t)__popcll(bit & ~below);
	}
	uint32_t free_before = sum_before(free_here, counts[2], wave, lane), move_before = sum_before(move_here, counts[3], wave, lane);
	for (uint32_t w = word; w < word_end; ++w) {
		const uint64_t bit = bits[w], below = below_edge(w);
		freed[w] = free_before;
		moved[w] = move_before;
		free_before += (uint32_t)__popcll(~bit & below);
		move_before += (uint32_t)__popcll(bit & ~below);
	}
	__syncthreads();
	for (uint32_t x = places / EVICT_THREADS * EVICT_THREADS + tid; x < rest; x += EVICT_THREADS) {
		const uint64_t beyond = bits[x / 64] & ~below_edge(x / 64);
		if (!(beyond >> lane & 1)) continue;
		const uint32_t to = moved[x / 64] + (uint32_t)__popcll(beyond & lanes_below(lane));
		if (cached) list[to] = (uint16_t)x;
		else kept[e.first + to] = (int32_t)(e.first + x);
	}
	__syncthreads();
	auto put = [&](uint32_t t, float w) {
		size_t at;
		if (weight_of(e, table, head, t, &at)) e.weights[at] = w;
	};
	if (cached) {
#pragma unroll 4
		for (uint32_t x = tid; x < places; x += EVICT_THREADS) {
			const uint64_t bit = bits[x / 64];
			uint32_t from = x;
			if (!(bit >> lane & 1)) {
				from = list[freed[x / 64] + (uint32_t)__popcll(~bit & lanes_below(lane))];
				size_t at;
				put(e.first + x, weight_of(e, table, head, e.first + from, &at) ? cache[from] : 0.0f);
			}
			kept[e.first + x] = (int32_t)(e.first + from);
		}
	} else {
		for (uint32_t top = (places + EVICT_THREADS - 1) / EVICT_THREADS; top-- > 0;) {
			const uint32_t x = top * EVICT_THREADS + tid;
			int32_t from = (int32_t)(e.first + x);
			bool free = false;
			if (x < places) {
				free = !(bits[x / 64] >> lane & 1);
				if (free) from = kept[e.first + freed[x / 64] + (uint32_t)__popcll(~bits[x / 64] & lanes_below(lane))];
			}
			__syncthreads();
			if (x < places) {
				kept[e.first + x] = from;
				size_t at;
				if (free) put(e.first + x, weight_of(e, table, head, (uint32_t)from, &at) ? e.weights[at] : 0.0f);
			}
		}
		__syncthreads(); /* (what moved from where the recent ones go) */
	}
	for (uint32_t i = tid; i < e.first; i += EVICT_THREADS) kept[i] = (int32_t)i;
	for (uint32_t i = tid; i < e.recent; i += EVICT_THREADS) kept[edge + i] = (int32_t)(n - e.recent + i);
	/* the recent ones move down in their order, later ones from places that earlier ones do not go to */
	for (uint32_t i0 = 0; i0 < e.recent; i0 += EVICT_THREADS) {
		const uint32_t i = i0 + tid;
		float w = recent;
		size_t at;
		if (i0 && i < e.recent) w = weight_at(n - e.recent + i);
		__syncthreads();
		if (i < e.recent) put(edge + i, weight_of(e, table, head, n - e.recent + i, &at) ? w : 0.0f);
	}
	__syncthreads();
#pragma unroll 4
	for (uint32_t t = e.keep + tid; t < n; t += EVICT_THREADS) put(t, 0.0f);
}

/* ---------------------------------------------------------------- moves -------------------------- */

/* what a lane holds of a row: a word of the keys' codes, a byte of one or two pairs of the values' channels, half a word of the scales */
template <int J> struct Row16 { uint32_t key; uint8_t value[J > 4 ? 2 : 1]; uint16_t scale; };

template <int J>
__device__ __forceinline__ Row16<J> take_row(const uint8_t* block, uint32_t t, uint32_t lane)
{
	constexpr uint32_t D = 32 * J;
	Row16<J> r{};
	if (lane < 4 * J) r.key = *(const uint32_t*)(block + t * (D / 2) + 4 * lane);
#pragma unroll
	for (int i = 0; i < (J > 4 ? 2 : 1); ++i)
		if (lane + WAVE * i < 16 * J) r.value[i] = block[8 * D + 16 * (lane + WAVE * i) + t];
	if (lane < 2 * J) r.scale = ((const uint16_t*)(block + 16 * D))[lane < J ? t * J + lane : 16 * J + 16 * (lane - J) + t];
	return r;
}
template <int J>
__device__ __forceinline__ void put_row(uint8_t* block, uint32_t t, uint32_t lane, const Row16<J>& r)
{
	constexpr uint32_t D = 32 * J;
	if (lane < 4 * J) *(uint32_t*)(block + t * (D / 2) + 4 * lane) = r.key;
#pragma unroll
	for (int i = 0; i < (J > 4 ? 2 : 1); ++i)
		if (lane + WAVE * i < 16 * J) block[8 * D + 16 * (lane + WAVE * i) + t] = r.value[i];
	if (lane < 2 * J) ((uint16_t*)(block + 16 * D))[lane < J ? t * J + lane : 16 * J + 16 * (lane - J) + t] = r.scale;
}

/*
 * Rows to their new places, a wavefront a row, eight rows on their way at a time. Of a sequence and head the first work-group moves those that come from the places which the recent ones
 * are about to take (the lowest places have them), and then these, in their order; the others share the rest, which come from behind all new places, by runs of 16 places.
 * Bound by the chain kept - table - row - place of each run: 4096 of 16384 tokens, 4 sequences, 8 heads of 128: 11 us.
 */
template <int J>
__global__ void __launch_bounds__(256)
evict4_move_kernel(Evict4 e)
{
	const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / WAVE)), lane = threadIdx.x % WAVE;
	const uint32_t head = blockIdx.x, s = blockIdx.y, n = evict_length(e, s);
	if (n <= e.keep) return;
	const int32_t* table = e.table + (size_t)s * e.table_stride;
	const int32_t* kept = e.kept + ((size_t)s * e.cache.heads + head) * e.keep;
	const uint32_t edge = e.keep - e.recent, page_mask = (1u << e.cache.page_shift) - 1;
	auto page_of = [&](uint32_t t) { return (uint32_t)table[t >> e.cache.page_shift]; };
	auto block_of = [&](uint32_t page, uint32_t t) { return e.cache.blocks + block_offset<J>(e.cache, page, head, (t & page_mask) / 16); };
	constexpr int AT_ONCE = 8;
	const bool begins = blockIdx.z == 0;
	const uint32_t waves = begins ? 4 : 4 * (gridDim.z - 1), number = begins ? wave : 4 * (blockIdx.z - 1) + wave;
	const uint32_t run = begins ? 64 : 16; /* places of a wavefront at a time */
	for (uint32_t i0 = e.first + run * number; i0 < edge; i0 += run * waves) {
		const uint32_t i = i0 + lane, from = lane < run && i < edge ? (uint32_t)kept[i] : i;
		const bool mine = begins ? from >= edge && from < e.keep : from >= e.keep;
		const bool moving = lane < run && i < edge && mine;
		const uint32_t source = moving ? page_of(from) : ~0u, target = moving ? page_of(i) : ~0u;
		uint64_t moves = __ballot(source < e.cache.page_count && target < e.cache.page_count);
		while (moves) {
			Row16<J> row[AT_ONCE];
			int bit[AT_ONCE];
#pragma unroll
			for (int k = 0; k < AT_ONCE; ++k) {
				bit[k] = moves ? __ffsll((unsigned long long)moves) - 1 : -1;
				if (bit[k] < 0) continue;
				moves &= moves - 1;
				const uint32_t t = (uint32_t)__builtin_amdgcn_readlane((int)from, bit[k]);
				row[k] = take_row<J>(block_of((uint32_t)__builtin_amdgcn_readlane((int)source, bit[k]), t), t % 16, lane);
			}
#pragma unroll
			for (int k = 0; k < AT_ONCE; ++k) {
				if (bit[k] < 0) continue;
				const uint32_t t = i0 + (uint32_t)bit[k];
				put_row<J>(block_of((uint32_t)__builtin_amdgcn_readlane((int)target, bit[k]), t), t % 16, lane, row[k]);
			}
		}
		if (begins && __any(from >= e.keep)) break; /* the lowest places have what came from the lowest: no more of its own behind */
	}
	if (!begins) return;
	for (uint32_t i0 = 0; i0 < e.recent; i0 += 4 * AT_ONCE) {
		const uint32_t first = i0 + AT_ONCE * wave, i = first + lane % AT_ONCE;
		const uint32_t source = i < e.recent ? page_of(n - e.recent + i) : ~0u, target = i < e.recent ? page_of(edge + i) : ~0u;
		const bool good = source < e.cache.page_count && target < e.cache.page_count;
		const uint32_t moves = (uint32_t)__ballot(good) & ((1u << AT_ONCE) - 1);
		__syncthreads(); /* what lay there has been read */
		Row16<J> row[AT_ONCE];
#pragma unroll
		for (int k = 0; k < AT_ONCE; ++k) {
			if (!(moves >> k & 1)) continue;
			const uint32_t t = n - e.recent + first + k;
			row[k] = take_row<J>(block_of((uint32_t)__builtin_amdgcn_readlane((int)source, k), t), t % 16, lane);
		}
		__syncthreads();
#pragma unroll
		for (int k = 0; k < AT_ONCE; ++k) {
			if (!(moves >> k & 1)) continue;
			const uint32_t t = edge + first + k;
			put_row<J>(block_of((uint32_t)__builtin_amdgcn_readlane((int)target, k), t), t % 16, lane, row[k]);
		}
	}
}

} // namespace kmx

using namespace kmx;

extern "C" {

int kmx_cache4_weigh(const kmx_cache4* cache, const kmx_cache4_batch* batch, int type, const void* q, size_t q_token_stride, size_t q_head_stride,
                     const float* lse, float scale, int causal, float* weights)
{
	clear_error();
	Weigh4 a{};
	int rc = check_cache4("kmx_cache4_weigh", cache, &a.cache);
	if (rc) return rc;
	rc = check_batch4("kmx_cache4_weigh", cache, batch, causal, &a.batch);
	if (rc) return rc;
	rc = check_type("kmx_cache4_weigh", type, false);
	if (rc) return rc;
	if (!(std::fabs(scale) <= 3.4e38f)) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_weigh: the scale is not finite");
	const uint64_t most = (uint64_t)a.batch.table_stride * cache->page_tokens;
	const uint32_t longest = a.batch.max_length < most ? a.batch.max_length : (uint32_t)most;
	if (batch->sequences == 0 || batch->tokens == 0 || batch->max_queries == 0 || longest == 0) return KMX_OK;
	if (!q || !lse || !weights) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_weigh: null device pointer");
	if ((uint64_t)(batch->max_queries < batch->tokens ? batch->max_queries : batch->tokens) * a.batch.group > 0x7FFFFFFFu) return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_weigh: rows of a head are counted in 31 bits");
	if ((uintptr_t)q % 2 || (uintptr_t)lse % 4 || (uintptr_t)weights % 4) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_weigh: rows start at multiples of their element's size");
	a.q = q;
	a.q_token = q_token_stride;
	a.q_head = q_head_stride;
	a.lse = lse;
	a.weights = weights;
	a.scale = scale;
	a.bf16 = type == KMX_BF16;
	a.vec = aligned_rows(q, q_token_stride, q_head_stride, 2);
	const uint32_t chunks = (longest - 1) / WEIGH_TOKENS + 1;
	if (batch->sequences > 65535 || chunks > 65535) return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_weigh: %u sequences of up to %u tokens are too many for one call", batch->sequences, longest);
	switch (cache->dim / 32) {
#define KMX_CASE(N) case N: KMX_LAUNCH_KERNEL((weigh4_kernel<N>), dim3(cache->heads, batch->sequences, chunks), dim3(256), 0, stream(), a); break;
		KMX_CASE(1) KMX_CASE(2) KMX_CASE(3) KMX_CASE(4) KMX_CASE(5) KMX_CASE(6) KMX_CASE(7) KMX_CASE(8)
#undef KMX_CASE
	}
	KMX_LAUNCH_CHECK("weigh4_kernel");
	return KMX_OK;
}

int kmx_cache4_evict(const kmx_cache4* cache, const kmx_cache4_batch* batch, float* weights, uint32_t keep, uint32_t first, uint32_t recent, int32_t* kept, int32_t* left)
{
	clear_error();
	Evict4 e{};
	int rc = check_cache4("kmx_cache4_evict", cache, &e.cache);
	if (rc) return rc;
	if (!batch) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_evict: null batch");
	if ((uint64_t)first + recent > keep) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_evict: %u tokens have no room for the %u first and %u recent ones", keep, first, recent);
	if (batch->max_length > EVICT_TOKENS) return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_evict: sequences of up to %u tokens, at most %u", batch->max_length, EVICT_TOKENS);
	if (batch->sequences == 0) return KMX_OK;
	if (!batch->lengths || (batch->table_stride && !batch->table) || !weights || (keep && !kept) || !left) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_evict: null device pointer");
	if ((uintptr_t)weights % 4 || (uintptr_t)kept % 4 || (uintptr_t)left % 4) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_evict: arrays start at multiples of their element's size");
	if (left == batch->lengths) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_cache4_evict: lengths and what is left of them are two arrays");
	if (batch->sequences > 65535) return fail(KMX_ERR_UNSUPPORTED, "kmx_cache4_evict: %u sequences are too many for one call", batch->sequences);
	const uint32_t table_stride = cache->page_count ? batch->table_stride : 0;
	const uint64_t most = (uint64_t)table_stride * cache->page_tokens;
	const uint32_t longest = batch->max_length < most ? batch->max_length : (uint32_t)most;
	e.lengths = batch->lengths;
	e.table = batch->table;
	e.weights = weights;
	e.kept = kept;
	e.left = left;
	e.sequences = batch->sequences;
	e.table_stride = table_stride;
	e.max_length = batch->max_length;
	e.keep = keep;
	e.first = first;
	e.recent = recent;
	const uint32_t places = keep < longest ? keep - recent - first : 0, rest = keep < longest ? longest - recent - first : 0;
	e.words = (rest + 63) / 64;
	const uint32_t room = (MOST_EVICT_BYTES - EVICT_WORD * e.words) / 6; /* beside the words: of 262144 tokens, for 5632 weights */
	e.cached = rest < EVICT_CACHED ? rest : EVICT_CACHED;
	if (e.cached > room) e.cached = room;
	const uint32_t bytes = evict_bytes(e.words, e.cached);
	static int allowed = -1;
	const DeviceInfo* dev = nullptr;
	rc = device_info(&dev);
	if (rc) return rc;
	if (bytes > 32768 && allowed != dev->device) { /* more LDS than a launch may ask for unannounced, on this device */
		KMX_HIP(hipFuncSetAttribute((const void*)evict4_choose_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)MOST_EVICT_BYTES));
		allowed = dev->device;
	}
	KMX_LAUNCH_KERNEL(evict4_choose_kernel, dim3(cache->heads, batch->sequences), dim3(EVICT_THREADS), bytes, stream(), e);
	KMX_LAUNCH_CHECK("evict4_choose_kernel");
	if (longest <= keep) return KMX_OK; /* nothing moves */
	/* work-groups for the moves of a head: about 16 rows each, and two that do all where they are many anyway */
	uint64_t parts = 1 + (places < longest - keep ? places : longest - keep) / 16;
	const uint64_t units = (uint64_t)cache->heads * batch->sequences, enough = 8 * (uint64_t)dev->compute_units / units + 1;
	if (parts > enough) parts = enough;
	if (parts > 65534) parts = 65534;
	switch (cache->dim / 32) {
#define KMX_CASE(N) case N: KMX_LAUNCH_KERNEL((evict4_move_kernel<N>), dim3(cache->heads, batch->sequences, (unsigned)parts + 1), dim3(256), 0, stream(), e); break;
		KMX_CASE(1) KMX_CASE(2) KMX_CASE(3) KMX_CASE(4) KMX_CASE(5) KMX_CASE(6) KMX_CASE(7) KMX_CASE(8)
#undef KMX_CASE
	}
	KMX_LAUNCH_CHECK("evict4_move_kernel");
	return KMX_OK;
}

} // extern "C"
