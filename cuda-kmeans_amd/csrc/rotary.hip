/*
 * Rotary positions (kmx_rotary of include/kmx.h): the pairs (a, b) of channels of a row at position p become gain (a cos x - b sin x, a sin x + b cos x),
 * x = 2 pi p f_i, f_i turns a position of pair i.
 *
 * Frequencies are kept as 64-bit fractions of a turn, so that p f_i without its whole turns is a product of whole numbers modulo 2^64: what a float or a table
 * would lose at far positions (2^-24 of 131072 radians is a hundredth of one) is never there. Its upper 32 bits -- 2^-32 of a turn, 1.5e-9 radians -- are taken to
 * the nearest quarter turn, and sine and cosine of the rest, within +- pi / 4, are the Taylor series up to x^9 and x^8 (the next terms are below 2^-25).
 */
#include "cache4.h"

#include <cmath>

namespace kmx {

constexpr uint32_t ROTARY_SETS = 4; /* of rows, in one call */

struct RotarySet { const void* in; void* out; size_t in_token, in_head, out_token, out_head; uint32_t until; }; /* heads of this set and those before it */
struct Rotary {
	RotarySet sets[ROTARY_SETS];
	const int32_t* positions;
	const uint64_t* turns;
	uint32_t tokens, heads;  /* heads of all sets */
	uint32_t half, dim;      /* pairs of a row that are rotated, channels of a row */
	uint32_t items, lanes;   /* pieces of a row, lanes that share a token's heads */
	float gain;
	bool inverse;
};

/* cosine and sine of p turns */
__device__ __forceinline__ float2 turned(int32_t position, uint64_t turns)
{
	const uint32_t low = (uint32_t)turns, high = (uint32_t)(turns >> 32);
	uint32_t part = __umulhi((uint32_t)position, low) + (uint32_t)position * high;
	if (position < 0) part -= low;
	const uint32_t quarter = (part + 0x20000000u) >> 30;
	const float x = (float)(int32_t)(part - (quarter << 30)) * (float)(6.28318530717958647692 / 4294967296.0), y = x * x;
	const float s = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f), 1.0f / 120.0f), -1.0f / 6.0f), x);
	const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 40320.0f, -1.0f / 720.0f), 1.0f / 24.0f), -0.5f), 1.0f);
	const float u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
	return float2{ __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, u) ^ ((quarter + 1) << 30 & 0x80000000u)),
	               __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) ^ (quarter << 30 & 0x80000000u)) };
}

template <typename T, uint32_t N> struct Piece { T v[N]; } __attribute__((packed, aligned(sizeof(T) * N >= 16 ? 16 : sizeof(T) * N)));
template <typename T> __device__ __forceinline__ float float_of(T v)
{
	if constexpr (sizeof(T) == 4) return v;
	else if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(float, (uint32_t)__builtin_bit_cast(uint16_t, v) << 16);
	else return (float)v;
}
template <typename T> __device__ __forceinline__ T rounded(float v)
{
	if constexpr (sizeof(T) == 4) return v;
	else return __builtin_bit_cast(T, (uint16_t)bits16<T>(v));
}

/*
 * A lane takes one piece of a token's rows -- N channels and their N partners -- for every `lanes`-th head, so that sines and cosines are made once for them; pieces
 * behind the rotated channels are copied. N: 16 bytes where rows allow it, else one pair at a time. Bound by memory: 16384 tokens of 32 + 8 heads of 128 channels in bfloat16 71.6 us, 4.7 TB/s (a copy of
 * 1 GiB: 5.0); 5003 tokens of 15 heads of 96 in 32 bits, neighbours in pairs, 11.1 (they stay in the memory-side cache); 32 tokens 5.5 to 6.2, of which a launch is 4.5.
 */
template <typename T, uint32_t N, bool HALVES>
__global__ void __launch_bounds__(256)
rotary_kernel(Rotary a)
{
	const uint32_t at = blockIdx.x * 256 + threadIdx.x, row = at / a.items, item = at - row * a.items, token = row / a.lanes, lane = row - token * a.lanes;
	if (token >= a.tokens) return;
	/* the two runs of N channels: of halves one in each, of neighbours (2 i, 2 i + 1) side by side */
	const uint32_t first = item * N, rotated = a.half / N;
	const bool turns = item < rotated;
	const uint32_t p0 = turns && HALVES ? first : 2 * first, p1 = turns && HALVES ? first + a.half : 2 * first + N;
	const bool second = turns || p1 < a.dim; /* what is copied may end with one run */
	float c[N], s[N];
	if (turns) {
		const int32_t position = a.positions[token];
		const uint64_t* f = a.turns + first;
#pragma unroll
		for (uint32_t i = 0; i < N; ++i) {
			const float2 cs = turned(position, f[i]);
			c[i] = cs.x * a.gain;
			s[i] = a.inverse ? -cs.y * a.gain : cs.y * a.gain;
		}
	}
	using Run = Piece<T, N>;
#pragma unroll 4
	for (uint32_t head = lane; head < a.heads; head += a.lanes) {
		uint32_t n = 0;
		for (uint32_t i = 0; i + 1 < ROTARY_SETS; ++i) n += head >= a.sets[i].until;
		const RotarySet& set = a.sets[n];
		const uint32_t h = n ? head - a.sets[n - 1].until : head;
		const T* in = (const T*)set.in + (size_t)token * set.in_token + (size_t)h * set.in_head;
		T* out = (T*)set.out + (size_t)token * set.out_token + (size_t)h * set.out_head;
		Run x = *(const Run*)(in + p0), y;
		if (second) y = *(const Run*)(in + p1);
		if (turns) {
			if constexpr (HALVES) {
#pragma unroll
				for (uint32_t i = 0; i < N; ++i) {
					const float u = float_of(x.v[i]), v = float_of(y.v[i]);
					x.v[i] = rounded<T>(fmaf(u, c[i], -v * s[i]));
					y.v[i] = rounded<T>(fmaf(u, s[i], v * c[i]));
				}
			} else {
				T z[2 * N];
#pragma unroll
				for (uint32_t i = 0; i < 2 * N; ++i) z[i] = i < N ? x.v[i] : y.v[i - N];
#pragma unroll
				for (uint32_t i = 0; i < N; ++i) {
					const float u = float_of(z[2 * i]), v = float_of(z[2 * i + 1]);
					z[2 * i] = rounded<T>(fmaf(u, c[i], -v * s[i]));
					z[2 * i + 1] = rounded<T>(fmaf(u, s[i], v * c[i]));
				}
#pragma unroll
				for (uint32_t i = 0; i < 2 * N; ++i) (i < N ? x.v[i] : y.v[i - N]) = z[i];
			}
		}
		*(Run*)(out + p0) = x;
		if (second) *(Run*)(out + p1) = y;
	}
}

template <typename T, uint32_t N>
static int launch_rotary(Rotary a, bool halves, bool copies, const DeviceInfo& dev)
{
	a.items = a.half / N + (copies ? (a.dim - 2 * a.half + 2 * N - 1) / (2 * N) : 0);
	/* heads a lane: one until the chip is full, then up to 8 */
	const uint64_t all = (uint64_t)a.tokens * a.heads * a.items, full = (uint64_t)dev.compute_units * 1024;
	const uint32_t each = all >= 8 * full ? 8 : all <= full ? 1 : (uint32_t)(all / full);
	a.lanes = (a.heads + each - 1) / each;
	const uint64_t groups = ((uint64_t)a.tokens * a.lanes * a.items + 255) / 256;
	if (groups > 0xFFFFFFu) return fail(KMX_ERR_UNSUPPORTED, "kmx_rotary: %u tokens of %u heads are too many for one call", a.tokens, a.heads);
	if (halves) KMX_LAUNCH_KERNEL((rotary_kernel<T, N, true>), dim3((unsigned)groups), dim3(256), 0, stream(), a);
	else KMX_LAUNCH_KERNEL((rotary_kernel<T, N, false>), dim3((unsigned)groups), dim3(256), 0, stream(), a);
	KMX_LAUNCH_CHECK("rotary_kernel");
	return KMX_OK;
}

template <typename T>
static int launch_rotary_of(const Rotary& a, bool halves, bool vec, bool copies, const DeviceInfo& dev)
{
	return vec ? launch_rotary<T, 16 / sizeof(T)>(a, halves, copies, dev) : launch_rotary<T, 1>(a, halves, copies, dev);
}

} // namespace kmx

using namespace kmx;

extern "C" {

int kmx_rotary_turns(uint32_t channels, double base, double stretch, double length, double slow, double fast, uint64_t* turns)
{
	clear_error();
	if (channels % 2) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary_turns: %u channels are no pairs", channels);
	if (!(base > 0.0 && std::isfinite(base)) || !(stretch > 0.0 && std::isfinite(stretch)))
		return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary_turns: base %g and stretch %g are above 0", base, stretch);
	if (!(length >= 0.0 && std::isfinite(length)) || !(slow >= 0.0 && std::isfinite(slow)) || !(fast >= slow && std::isfinite(fast)))
		return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary_turns: length %g, slow %g and fast %g: not negative, fast not below slow", length, slow, fast);
	if (channels && !turns) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary_turns: null pointer");
	const auto frequency = [&](uint32_t i) {
		const double f = std::pow(base, -2.0 * i / channels) / 6.283185307179586476925286766559; /* turns a position */
		const double made = length * f;
		double share = 0.0; /* of the frequency as it is */
		if (length > 0.0) share = made >= fast ? 1.0 : made <= slow ? 0.0 : (made - slow) / (fast - slow);
		return f * (share + (1.0 - share) / stretch);
	};
	for (uint32_t i = 0; i < channels / 2; ++i)
		if (!std::isfinite(frequency(i))) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary_turns: base %g and stretch %g: the frequency of pair %u is not finite", base, stretch, i);
	for (uint32_t i = 0; i < channels / 2; ++i) {
		const double g = frequency(i), part = g - std::floor(g); /* whole turns are none */
		const double scaled = std::nearbyint(std::ldexp(part, 64));
		turns[i] = scaled >= 18446744073709551616.0 ? 0 : (uint64_t)scaled;
	}
	return KMX_OK;
}

int kmx_rotary(int type, const kmx_rotary_rows* rows, uint32_t sets, uint32_t tokens, uint32_t dim, uint32_t channels, const uint64_t* turns, const int32_t* positions,
               int halves, int inverse, float gain)
{
	clear_error();
	if (type != KMX_F32 && type != KMX_F16 && type != KMX_BF16) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: unknown element type %d", type);
	if (channels % 2 || channels > dim) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: %u rotated channels of %u", channels, dim);
	if ((halves != 0 && halves != 1) || (inverse != 0 && inverse != 1)) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: halves and inverse are 0 or 1");
	if (!(std::fabs(gain) <= 3.4e38f)) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: the gain is not finite");
	if (sets > ROTARY_SETS) return fail(KMX_ERR_UNSUPPORTED, "kmx_rotary: %u sets of rows, at most %u", sets, ROTARY_SETS);
	if (sets && !rows) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: null rows");
	if (dim == 0 || tokens == 0 || sets == 0) return KMX_OK;
	const size_t size = type == KMX_F32 ? 4 : 2, run = 16 / size;
	Rotary a{};
	bool vec = (channels / 2) % run == 0 && dim % run == 0, copies = false;
	uint64_t heads = 0;
	for (uint32_t i = 0; i < ROTARY_SETS; ++i) {
		if (i < sets && rows[i].heads) {
			const kmx_rotary_rows& r = rows[i];
			if (!r.in || !r.out) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: null device pointer");
			if ((uintptr_t)r.in % size || (uintptr_t)r.out % size) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: rows start at multiples of their element's size");
			if (r.heads > 1 && r.out_head_stride < dim) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: head stride of the output %zu < dim %u", r.out_head_stride, dim);
			if (tokens > 1 && r.out_token_stride < dim) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: token stride of the output %zu < dim %u", r.out_token_stride, dim);
			const bool in_place = r.in == r.out;
			if (in_place && ((r.heads > 1 && r.in_head_stride != r.out_head_stride) || (tokens > 1 && r.in_token_stride != r.out_token_stride)))
				return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: rows that are rotated where they are have one set of strides");
			copies = copies || !in_place;
			vec = vec && (uintptr_t)r.in % 16 == 0 && (uintptr_t)r.out % 16 == 0 && r.in_token_stride * size % 16 == 0 && r.in_head_stride * size % 16 == 0 && r.out_token_stride * size % 16 == 0 && r.out_head_stride * size % 16 == 0;
			a.sets[i] = RotarySet{ r.in, r.out, r.in_token_stride, r.in_head_stride, r.out_token_stride, r.out_head_stride, 0 };
			heads += r.heads;
			if (heads > 0xFFFFFFu) return fail(KMX_ERR_UNSUPPORTED, "kmx_rotary: too many heads");
		}
		a.sets[i].until = (uint32_t)heads;
	}
	if (heads == 0 || (channels == 0 && !copies)) return KMX_OK;
	if (!positions || (channels && !turns)) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: null positions or turns");
	if ((uintptr_t)positions % 4 || (uintptr_t)turns % 8) return fail(KMX_ERR_INVALID_ARGUMENT, "kmx_rotary: positions start at multiples of 4 bytes, turns of 8");
	a.positions = positions;
	a.turns = turns;
	a.tokens = tokens;
	a.heads = (uint32_t)heads;
	a.half = channels / 2;
	a.dim = dim;
	a.gain = gain;
	a.inverse = inverse != 0;
	const DeviceInfo* dev = nullptr;
	const int rc = device_info(&dev);
	if (rc) return rc;
	if (type == KMX_F32) return launch_rotary_of<float>(a, halves, vec, copies && channels < dim, *dev);
	if (type == KMX_F16) return launch_rotary_of<_Float16>(a, halves, vec, copies && channels < dim, *dev);
	return launch_rotary_of<__bf16>(a, halves, vec, copies && channels < dim, *dev);
}

} // extern "C"
