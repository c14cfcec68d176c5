// The selective scan in chunks of 64 tokens on the matrix cores.  With L_t = sum_{s <= t} delta_s A inside a chunk and H the state in front of it:
//     y_t   = sum_{s <= t} (B_s . C_t) exp(L_t - L_s) delta_s x_s  +  exp(L_t) H C_t  +  D x_t
//     H_out = exp(L_64) H + sum_s exp(L_64 - L_s) delta_s x_s B_s^T
// so all that runs token by token is a sum of 64 steps; the rest are products of tiles.
//
// A block walks the chunks of one head (64 or 32 of its rows of the state) of one batch row, or of one segment of it: x is read once, y written once, B and C (shared
// by the heads of a group) come out of the L2.  Its waves have two trades, so that neither's chain of waits holds up the other:
//   * four (two for 32 rows) keep the state, 16 rows p each, in registers: H^T (rows n, columns p) += B (w x)^T, both operands with their tokens contiguous as they lie in
//     memory.  They also fetch the operands (requested two chunks ahead, written to the LDS one ahead; in float32 as many other waves do that, three ahead) and leave the state in the LDS for
//   * four others, which make the results of 16 tokens each: G = B C^T (rows s, columns t), the weights of the tokens s <= t as they sit in their lanes -
//     column t, four consecutive s a tile - which is the layout of a second operand, so Y^T = X^T W + H^T C^T needs no exchange between lanes.
// One barrier a chunk where the LDS holds two of them, two where it does not.
// The summation index of the results' products is a permuted one (slot 8 g + j of a lane group <-> 16 (j / 4) + 4 g + j % 4), the same in both operands.
//
// Half precision: x, B and C are exact.  The weights of the tokens and the state in front of a chunk are rounded to halves, 2^-11 of each term of y, which is
// what y itself is rounded to: the largest weight of a token and the largest element of a row of the state are brought to the top of a half's range by powers of
// two, so that this holds down to 2^-29 of them.  The weights of a token's own tile, which are mostly the largest, keep their remainders.  The state itself stays
// float32: w x enters as the sum of two halves, 22 bits.  Whether these lie where a half has its bits is looked at every time (a maximum and a few lane masks); where
// they do not, they are brought there in the same way, and the state goes along, as far as it remains a float.  That path is the slower one by a multiplication per
// value on either side: the state is kept 2^8 times what it is, which puts common steps outside of it.
// float32: every operand is the sum of two halves, 22 bits and a sign more than a half has, and a product is three (what is left out lies below 2^-22 of it).  The
// second halves are 2^11 times what they are and their products summed apart, so that they have their bits as far down as the first ones.  x, B
// and C are scaled by the powers of two that bring a chunk's largest element to the top of a half's range, the state and the weights likewise: all 22 bits down to
// 2^-29 of the largest, 2^-51 of the largest below that.  Sums are float32, and powers of two come out of them by exponents.  The fp32 matrix instruction does a
// sixteenth of what the one for halves does in its time (4 x 4096 tokens, 64 heads: 292 us with it in an early form of this kernel, 236 with halves then, 200 now).
// Steps are summed in 64 bits, and the distance of two tokens is put together from pieces of one sign - from a token to its tile's edge, tile by tile, and
// from an edge to a token - so that no difference of long sums is taken; inside a tile the sums are pairs of floats.
//
// Measured (heads of 64 rows, state 64; the bytes are x, B, C, dt, y and the states once): 4 x 4096 tokens, 64 heads, half precision 96 - 106 us = 2.6 - 2.9 TB/s, 16 x 1024 tokens 85,
// 16384 tokens, 128 heads 253 us = 2.2 TB/s, of which 80 are the first pass; float32 4 x 4096 tokens 200 us = 2.7 TB/s.  What bounds it, at one block of 8 waves on a
// CU as at two: the same loads and stores alone take 71 us (rows of 128 bytes, 8 KB apart), all the rest alone 89; the vector units issue 0.51 of the cycles
// (1570 instructions a chunk and block), the matrix units are busy 0.20 of them, with two blocks 0.61 and 0.24.  Two chunks ahead with the loads, one with the LDS, hides most of either behind the other.
#pragma once

#include "launch.hpp"
#include "selective_scan.hpp"

#include <type_traits>

namespace anygpu {

namespace scan {

constexpr int kChunk = 64;                  // tokens
constexpr float kUnit = 256.0f;             // half precision: the state and the weights into it are kept this many times what they are

// Where the sequences are shared out in segments: a first launch leaves the state behind every part of the segments but the last (taken from zeros, the first one's
// from the given state) and the decay across it, the second starts every segment from what the parts before it leave.
struct Plan
{
	int segments, segment_tokens, parts, rows, row_tiles, blocks;       // blocks: of one segment (batch rows x heads x tiles of R rows)
	float* states;                                        // [segments * parts][blocks][NT / 16][4 R] float4; the last slot: the given state
	float* decays;                                        // [segments * parts][blocks]
};

// R: rows of the state per block, 64 or 32.  STATES: the first launch, without results
template <typename T, int NT, int R, bool STATES>
struct Lds
{
	static constexpr bool kHalf = std::is_same_v<T, half_t>;
	static constexpr int kParts = kHalf ? 1 : 2;                            // halves of an operand
	// Bytes of a row: 160 has neither the 16-byte reads of B nor the transposing ones of B and C wait for a bank (144: four cycles more of eight, and two of
	// four), 144 not the 8-byte reads of X and H, which are more than X's two of 16 bytes (160: two more of four).
	static constexpr int kPitchX = kChunk * 2 + 16, kPitchB = kChunk * 2 + 32, kPitchH = NT * 2 + 16;
	static constexpr int kXLow = R * kPitchX, kBLow = NT * kPitchB, kHLow = R * kPitchH;       // from the first half to the second
	static constexpr int kX = 0, kB = kX + kParts * kXLow, kC = kB + kParts * kBLow, kStage = STATES ? kC : kC + kParts * kBLow;
	// a state in front of a chunk; the scales of four of its rows lie behind each of the first R / 4 rows, in what the pitch leaves there
	static constexpr int kScales = NT * 2, kFront = STATES ? 0 : kParts * kHLow;
	static constexpr int kTwoSteps = 2 * 7 * kChunk * 4 + 256;
	// two chunks' operands where that leaves room for as many blocks as the registers do (half precision: two, three without results) or does not matter
	static constexpr int kBlocks = kHalf && NT <= 64 ? (STATES ? 3 : 2) : 1;
	// float32, where fetching and splitting the operands is as much work as the state's: a trade of its own, where the registers leave room for its waves
	// (4 x 4096 tokens, 64 heads: 247 us without, 206 with; 3 x 1001 tokens, 32 heads, state 128, whose first pass only has it: 4 % less)
	static constexpr bool kMovers = !kHalf && (NT <= 64 || STATES);
	static constexpr int kThreads = 4 * R * (kMovers ? 2 : 1) + (STATES ? 0 : 256), kWaves = (kThreads / 64 * kBlocks + 3) / 4;        // (of a SIMD)
	static constexpr int kStages = kBlocks * (2 * kStage + 2 * kFront + kTwoSteps) <= 160 * 1024 ? 2 : 1;
	static constexpr int kFronts = kStages * kStage, kSteps = kFronts + kStages * kFront;      // the states, two sets of what a chunk's steps give
	// of a token: steps since its tile's start (pair), the same less log2(delta) (half precision, pair), from it to its tile's end (+ log2(delta) in half
	// precision), exp(L), weight into the state, delta (float32)
	static constexpr int kIn = 0, kInLow = 1, kOut = 2, kGain = 3, kWeight = 4, kFrom = 5, kFromLow = 6, kDelta = 5, kArrays = kHalf ? 7 : 6;
	// and: steps across the four tiles, the chunk's decay; float32: what the scales of x, B and C make of sums (see store_chunk; kBack: exponents)
	static constexpr int kDecay = 4, kScaleBC = 5, kSkip = 6, kBackX = 7, kBackC = 8, kBackBX = 9;
	static constexpr int kSet = kArrays * kChunk * 4 + 48;
	static constexpr int kMost = kSteps + 2 * kSet;                         // float32: the largest x, B and C of a chunk by wave, two sets
	static constexpr int kBytes = kMost + (kHalf ? 0 : 2 * 3 * 16);
};

// k of the 2^k with 2^14 <= v 2^k < 2^15, which brings v to the top of a half's range, between bounds whose products are floats
__device__ __forceinline__ int half_exponent(float v, int lowest, int highest)
{
	const int k = 141 - ((__builtin_bit_cast(int, v) >> 23) & 255);
	return k < lowest ? lowest : k > highest ? highest : k;
}

constexpr int kLowest = -113, kHighest = 116;       // of the largest float, and of what is a float 2^11 times as large

__device__ __forceinline__ float power_of_two(int k) { return __builtin_bit_cast(float, (127 + k) << 23); }

// a magnitude that a scale may be taken from: an infinity is beyond all of them, and its neighbours are to keep their bits
__device__ __forceinline__ float finite_or_zero(float v) { return v < INFINITY ? v : 0.0f; }

// a half times a float: the lower or upper half of two
template <int UPPER>
__device__ __forceinline__ float times_half(half2_t h, float v)
{
	float r;
	if constexpr (UPPER) asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(v));
	else asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(v));
	return r;
}

// a half times a float and a float added
template <int UPPER>
__device__ __forceinline__ float times_half_add(half2_t h, float v, float to)
{
	float r;
	if constexpr (UPPER) asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(v), "v"(to));
	else asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(v), "v"(to));
	return r;
}

// Every lane has the largest magnitude of its values; the four lanes l, l + 16, l + 32 and l + 48 share a row (or column).  True unless all values fit a half and
// every row that has any value but zero has one of `least` and more.
__device__ __forceinline__ bool rows_need_scale(float most, float least)
{
	const auto fold = [](unsigned long long m) {
		m |= m >> 32;
		return (unsigned)(m | (m >> 16)) & 0xFFFFu;
	};
	const unsigned long long over = __builtin_amdgcn_ballot_w64(!(most < 65504.0f)), some = __builtin_amdgcn_ballot_w64(most > 0.0f),
	                         enough = __builtin_amdgcn_ballot_w64(most >= least);
	return over != 0 || (fold(some) & ~fold(enough)) != 0;
}

// what a float keeps behind its rounding to a half: v - h, h the lower or upper half of two
template <int UPPER>
__device__ __forceinline__ float remainder_of(float v, half2_t h)
{
	float r;
	if constexpr (UPPER) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(v));
	else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(v));
	return r;
}

// four floats as halves, and their remainders as halves
__device__ __forceinline__ void split(float4_t v, half4_t& hi, half4_t& low)
{
	hi = __builtin_convertvector(v, half4_t);
	const half2_t h0 = {hi[0], hi[1]}, h1 = {hi[2], hi[3]};
	const float4_t rest = {remainder_of<0>(v[0], h0), remainder_of<1>(v[1], h0), remainder_of<0>(v[2], h1), remainder_of<1>(v[3], h1)};
	low = __builtin_convertvector(rest, half4_t);
}

// the value of the lane N below in the row of 16 lanes, 0 where there is none
template <int N>
__device__ __forceinline__ double row_shift(double v)
{
	typedef int Pair __attribute__((ext_vector_type(2)));
	Pair p = __builtin_bit_cast(Pair, v);
	p[0] = __builtin_amdgcn_update_dpp(0, p[0], 0x110 + N, 0xF, 0xF, true);
	p[1] = __builtin_amdgcn_update_dpp(0, p[1], 0x110 + N, 0xF, 0xF, true);
	return __builtin_bit_cast(double, p);
}

__device__ __forceinline__ double read_lane_f64(double v, int lane)
{
	typedef int Pair __attribute__((ext_vector_type(2)));
	Pair p = __builtin_bit_cast(Pair, v);
	p[0] = __builtin_amdgcn_readlane(p[0], lane);
	p[1] = __builtin_amdgcn_readlane(p[1], lane);
	return __builtin_bit_cast(double, p);
}

// The same with the remainders 2^11 times what they are: as far above the smallest half as the values themselves.  Products with them are summed apart.
constexpr float kLowUnit = 2048.0f;

__device__ __forceinline__ void split_wide(float4_t v, half4_t& hi, half4_t& low)
{
	hi = __builtin_convertvector(v, half4_t);
	const half2_t h0 = {hi[0], hi[1]}, h1 = {hi[2], hi[3]};
	const float4_t rest = {remainder_of<0>(v[0], h0), remainder_of<1>(v[1], h0), remainder_of<0>(v[2], h1), remainder_of<1>(v[3], h1)};
	low = __builtin_convertvector(rest * kLowUnit, half4_t);
}

__device__ __forceinline__ float4_t add_low(float4_t main, float4_t low)
{
	float4_t r;
#pragma unroll
	for (int i = 0; i < 4; ++i) r[i] = fmaf(low[i], 1.0f / kLowUnit, main[i]);
	return r;
}

typedef short short4_t __attribute__((ext_vector_type(4)));

// (lane i of a group of 16 gets element i of the 4-row band whose row i / 4, columns 4 (i % 4) .. + 3 its address points at)
__device__ __forceinline__ half4_t read_transposed(const char* lds)
{
	return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)lds));
}

__device__ __forceinline__ half8_t join(half4_t lo, half4_t hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

__device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

template <typename T, int NT, int R, bool STATES>
__global__ __launch_bounds__((Lds<T, NT, R, STATES>::kThreads), (Lds<T, NT, R, STATES>::kWaves)) void selective_scan_chunk_kernel(const ScanArgs a, const Plan plan)
{
	using L = Lds<T, NT, R, STATES>;
	constexpr int PT = R / 16, KT = 4 * R;                                  // tiles of rows, threads that keep the state
	constexpr bool HALF = L::kHalf;
	constexpr bool DOUBLE = L::kStages == 2;
	constexpr int EPV = 16 / (int)sizeof(T), VPR = kChunk / EPV;           // elements of a vector, vectors of a row
	constexpr int XV = R * VPR / KT, BV = NT * VPR / KT;                   // vectors of a thread
	// the widest states' B and C are too many registers to be requested ahead: they are fetched in parts where they are stored
	constexpr bool AHEAD = NT <= 128;
	constexpr int BA = AHEAD ? BV : 4, PARTS = BV / BA;
	constexpr int NB = NT / 16;
	typedef T Vec __attribute__((ext_vector_type(EPV)));
	typedef Vec LooseVec __attribute__((aligned(sizeof(T))));
	typedef T Quad __attribute__((ext_vector_type(4)));
	typedef Quad LooseQuad __attribute__((aligned(sizeof(T))));
	extern __shared__ __align__(16) char lds[];

	// the first four waves make the results, then come those that keep the state, then those that fetch, where they are others
	constexpr bool MOVERS = L::kMovers;
	static_assert(!MOVERS || DOUBLE, "those that fetch are a chunk ahead in the LDS");
	const int beyond = (int)threadIdx.x - (STATES ? 0 : 256);
	const int trade = __builtin_amdgcn_readfirstlane(beyond < 0 ? 0 : 1 + beyond / KT);
	const int tid = beyond < 0 ? threadIdx.x : beyond & (KT - 1), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);      // within the trade
	const bool moves = !MOVERS || trade == 2;
	const int l = lane & 15, g = lane >> 4;
	const int block = blockIdx.x % plan.blocks, segment = blockIdx.x / plan.blocks;
	const int bh = block / plan.row_tiles, p0 = (block - bh * plan.row_tiles) * R;
	const int batch = bh / a.heads, head = bh - batch * a.heads, group = head / (a.heads / a.groups);
	const int rows = a.head_dim - p0 < R ? a.head_dim - p0 : R, size = a.state_dim;
	const int length = __builtin_amdgcn_readfirstlane(scan_length(a.lengths, batch, a.seqlen));
	const int begin = segment * plan.segment_tokens;
	const int limit = a.seqlen - begin < plan.segment_tokens ? a.seqlen : begin + plan.segment_tokens;     // of the segment
	const int end = length < limit ? length : limit;

	const T* dt = static_cast<const T*>(a.dt) + batch * a.dt_batch + head * a.dt_head;
	const double rate = (double)a.a[head] * 1.4426950408889634;
	const float bias = a.bias ? a.bias[head] : 0.0f, skip = a.skip ? a.skip[head] : 0.0f;
	const auto load_step = [&](int t0) { return dt[(t0 + lane < end ? t0 + lane : end - 1) * a.dt_seq]; };
	// a chunk's sums of steps, a token per lane of one wave
	const auto make_steps = [&](int t0, float raw, int set) {
		float* out = reinterpret_cast<float*>(lds + L::kSteps + set * L::kSet);
		const bool live = t0 + lane < end;
		const float delta = live ? scan_delta(raw, bias, a.dt_min, a.dt_max) : 0.0f;
		// sums inside a tile of 16 tokens, which is a row of lanes
		double in = live ? (double)delta * rate : 0.0;
		if (in < -1024.0) in = -1024.0;                       // (2^-1024 is no float but 0, and the sums keep the bits of the steps behind a long one)
		in += row_shift<1>(in);
		in += row_shift<2>(in);
		in += row_shift<4>(in);
		in += row_shift<8>(in);
		const double t_0 = read_lane_f64(in, 15), t_1 = read_lane_f64(in, 31), t_2 = read_lane_f64(in, 47), t_3 = read_lane_f64(in, 63);
		const double before = (g > 0 ? t_0 : 0.0) + (g > 1 ? t_1 : 0.0) + (g > 2 ? t_2 : 0.0);
		const double behind = (g < 1 ? t_1 : 0.0) + (g < 2 ? t_2 : 0.0) + (g < 3 ? t_3 : 0.0);
		const double to_end = (g < 1 ? t_0 : g < 2 ? t_1 : g < 3 ? t_2 : t_3) - in, sum = before + in, rest = to_end + behind;
		const float in_hi = (float)in;
		out[L::kIn * kChunk + lane] = in_hi;
		out[L::kInLow * kChunk + lane] = (float)(in - (double)in_hi);
		if constexpr (HALF)
		{
			// exp(-L_s) delta_s as one exponential; a token without a step, and one whose step is no normal float (the logarithm takes it for none), has no weight
			const float log_delta = __builtin_amdgcn_logf(delta);
			const double from = in - (double)log_delta;
			const float from_hi = (float)from;
			out[L::kOut * kChunk + lane] = (float)(to_end + (double)log_delta);
			out[L::kFrom * kChunk + lane] = from_hi;
			out[L::kFromLow * kChunk + lane] = from_hi < INFINITY ? (float)(from - (double)from_hi) : 0.0f;
		}
		else
		{
			out[L::kOut * kChunk + lane] = (float)to_end;
			out[L::kDelta * kChunk + lane] = delta;
		}
		// 2^(hi + low) = 2^hi (1 + low ln 2)
		const auto power = [](double v) {
			const float hi = (float)v;
			return fast_exp2(hi) * fmaf((float)(v - (double)hi), 0.6931471805599453f, 1.0f);
		};
		const float past = power(sum);
		out[L::kGain * kChunk + lane] = past;
		out[L::kWeight * kChunk + lane] = power(rest) * (HALF ? delta * kUnit : delta);
		if ((lane & 15) == 15) out[L::kArrays * kChunk + g] = in_hi;
		if (lane == 63) out[L::kArrays * kChunk + 4] = past;
	};
	if (STATES || trade > 0)
	{
		const T* x = static_cast<const T*>(a.x) + batch * a.x_batch + ((int64_t)head * a.head_dim + p0) * a.x_row;
		const T* b = static_cast<const T*>(a.b) + batch * a.b_batch + (int64_t)group * a.state_row * a.b_row;
		const T* c = static_cast<const T*>(a.c) + batch * a.c_batch + (int64_t)group * a.state_row * a.c_row;
		// (without result waves one of these sums up the steps)
		const bool stepper = STATES && moves && wave == (int)(blockIdx.x & (PT - 1));

		// ---- the state: column p = 16 wave + l, rows n = 16 i + 4 g + r; half precision: kUnit times what it is ----
		float4_t h[NB];
		float decay = 1.0f;
		const int hp = 16 * wave + l;
		float* state = a.state + ((int64_t)bh * a.head_dim + p0 + hp) * a.state_row;
		const bool wide = size % 4 == 0 && a.state_row % 4 == 0 && (reinterpret_cast<uintptr_t>(a.state) & 15) == 0;
		const auto slot = [&](int s) { return reinterpret_cast<float4_t*>(plan.states) + ((int64_t)s * plan.blocks + block) * (NB * KT) + tid; };
#pragma unroll
		for (int i = 0; i < NB; ++i) h[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
		if (MOVERS && moves) {}
		else if (STATES || segment == 0)
		{
			if (segment == 0 && a.state != nullptr)
			{
				if (!STATES && plan.segments > 1)
				{
					// (the last segment's block may have written the new state already)
#pragma unroll
					for (int i = 0; i < NB; ++i) h[i] = slot(plan.segments * plan.parts - 1)[i * KT];
				}
				else if (hp < rows)
				{
#pragma unroll
					for (int i = 0; i < NB; ++i)
					{
						const int n = 16 * i + 4 * g;
						if (wide && n < size) h[i] = *reinterpret_cast<const float4_t*>(state + n);
						else if (n < size)
						{
#pragma unroll
							for (int r = 0; r < 4; ++r)
								if (n + r < size) h[i][r] = state[n + r];
						}
					}
				}
				if constexpr (STATES)
				{
#pragma unroll
					for (int i = 0; i < NB; ++i) slot(plan.segments - 1)[i * KT] = h[i];
				}
			}
		}
		else
		{
#pragma unroll
			for (int i = 0; i < NB; ++i) h[i] = slot(0)[i * KT];
			for (int s = 1; s < segment * plan.parts; ++s)
			{
				const float across = plan.decays[(int64_t)s * plan.blocks + block];
#pragma unroll
				for (int i = 0; i < NB; ++i) h[i] = h[i] * across + slot(s)[i * KT];
			}
		}

		// ---- operands: global -> registers -> LDS ----
		// Whole chunks go by way of registers.  Rows that do not exist repeat the last one: those of x end up in rows of y and of the state that nobody
		// stores, those of B are zeros in the LDS, so that what C has there meets zeros.
		struct Operands
		{
			Vec x[XV], b[BA], c[STATES ? 1 : BA];
		};
		unsigned xo[XV], bo[BA], co[STATES ? 1 : BA];                        // bytes from the first row's token (the launcher sees to it that they fit)
		const int vrow = tid / VPR, vcol = (tid % VPR) * EPV;
		constexpr int ROW_STEP = KT / VPR;
		const auto row_of = [&](int i, int live) { return vrow + i * ROW_STEP < live ? vrow + i * ROW_STEP : live - 1; };
		const auto offset = [&](int i, int live, int64_t stride) { return ((unsigned)row_of(i, live) * (unsigned)stride + vcol) * (unsigned)sizeof(T); };
#pragma unroll
		for (int i = 0; i < XV; ++i) xo[i] = offset(i, rows, a.x_row);
#pragma unroll
		for (int i = 0; i < BA; ++i)
		{
			bo[i] = offset(i, size, a.b_row);
			if constexpr (!STATES) co[i] = offset(i, size, a.c_row);
		}
		const auto fetch = [](const T* from, unsigned at) { return reinterpret_cast<const LooseVec*>(reinterpret_cast<const char*>(from) + at); };
		// The last chunk of a row that ends inside of it goes element by element: what does not exist repeats the last row and token and is replaced by zeros,
		// so that all loads go out before the first is waited for.
		const auto load_tail = [&](auto& v, const T* from, int64_t stride, int live, int tokens, int part) {
			constexpr int COUNT = sizeof(v) / sizeof(v[0]);
			// (nothing of this is to be kept ready in registers across the whole loop)
			live = __builtin_amdgcn_readfirstlane(live);
			tokens = __builtin_amdgcn_readfirstlane(tokens);
			asm volatile("" : "+s"(live), "+s"(tokens));
#pragma unroll
			for (int i = 0; i < COUNT; ++i)
			{
				const T* p = from + row_of(i + part * COUNT, live) * stride;
#pragma unroll
				for (int e = 0; e < EPV; ++e) v[i][e] = p[vcol + e < tokens ? vcol + e : tokens - 1];
			}
			typedef unsigned Words __attribute__((ext_vector_type(4)));
			constexpr int PER_WORD = EPV / 4;
#pragma unroll
			for (int i = 0; i < COUNT; ++i)
			{
				const int kept = vrow + (i + part * COUNT) * ROW_STEP < live ? tokens - vcol : 0;
				Words w = __builtin_bit_cast(Words, v[i]);
#pragma unroll
				for (int k = 0; k < 4; ++k) w[k] &= kept >= PER_WORD * (k + 1) ? ~0u : kept > PER_WORD * k ? 0xFFFFu : 0u;
				v[i] = __builtin_bit_cast(Vec, w);
			}
		};
		const auto load_chunk = [&](int t0, Operands& o, bool whole = false) {
			if (!whole && t0 >= end) return;
			if (!whole && t0 + kChunk > end)
			{
				load_tail(o.x, x + t0, a.x_row, rows, end - t0, 0);
				if constexpr (AHEAD)
				{
					load_tail(o.b, b + t0, a.b_row, size, end - t0, 0);
					if constexpr (!STATES) load_tail(o.c, c + t0, a.c_row, size, end - t0, 0);
				}
				return;
			}
			// (a scalar base and a lane's 32-bit offset, not six 64-bit pointers that are carried along in vector registers)
			asm volatile("" : "+s"(t0));
			// (plain loads also of x, which is read once or, by two passes, twice: non-temporal ones 72 us instead of 67 for 3 x 1001 tokens, state 128, float32, 29.1
			// and 27.2 for 500, and within 2 % of each other for what no cache holds)
#pragma unroll
			for (int i = 0; i < XV; ++i) o.x[i] = *fetch(x + t0, xo[i]);
			if constexpr (AHEAD)
			{
#pragma unroll
				for (int i = 0; i < BA; ++i) o.b[i] = *fetch(b + t0, bo[i]);
				if constexpr (!STATES)
				{
					// (float32 without waves that only fetch: 256 registers are all there are, and C's offsets are made afresh - 66.5 us, 68.2 with a spilled pair of them
					// for 3 x 1001 tokens, 32 heads, state 128)
					unsigned c_row = (unsigned)a.c_row;
					if constexpr (!HALF && !MOVERS) asm volatile("" : "+s"(c_row));
#pragma unroll
					for (int i = 0; i < BA; ++i) o.c[i] = *fetch(c + t0, HALF || MOVERS ? co[i] : offset(i, size, c_row));
				}
			}
		};
		// float32: the largest elements of what the registers hold
		const auto note_most = [&](int set, const Operands& o) {
			if constexpr (!HALF)
			{
				const auto most = [&](const auto& v, int which) {
					constexpr int COUNT = sizeof(v) / sizeof(v[0]);
					float m = 0.0f;
#pragma unroll
					for (int i = 0; i < COUNT; ++i)
#pragma unroll
						for (int e = 0; e < 4; ++e) m = fmaxf(m, __builtin_fabsf(v[i][e]));
					// Between 1 and 2^7 they are given as 2^6, a scale of 2^8: no reduction over the wave, and what two halves leave there is 2^-44
					float noted = 64.0f;
					if (__builtin_amdgcn_ballot_w64(!(m < 128.0f)) != 0 || __builtin_amdgcn_ballot_w64(m >= 1.0f) == 0)
					{
						m = 0.0f;
#pragma unroll
						for (int i = 0; i < COUNT; ++i)
#pragma unroll
							for (int e = 0; e < 4; ++e) m = fmaxf(m, finite_or_zero(__builtin_fabsf(v[i][e])));
						noted = wave_allreduce(m, MaxOp());
					}
					if (lane == 0) reinterpret_cast<float*>(lds + L::kMost)[12 * set + 4 * which + wave] = noted;
				};
				most(o.x, 0);
				most(o.b, 1);
				if constexpr (!STATES) most(o.c, 2);
			}
		};
		const auto store_rows = [&](const auto& v, int at, int pitch, int low, float up, int part) {
			constexpr int COUNT = sizeof(v) / sizeof(v[0]);
#pragma unroll
			for (int i = 0; i < COUNT; ++i)
			{
				char* const to = lds + at + (vrow + (i + part * COUNT) * ROW_STEP) * pitch + vcol * 2;
				if constexpr (HALF) *reinterpret_cast<Vec*>(to) = v[i];
				else
				{
					half4_t first, second;
					split_wide(v[i] * up, first, second);
					*reinterpret_cast<half4_t*>(to) = first;
					*reinterpret_cast<half4_t*>(to + low) = second;
				}
			}
		};
		const auto store_chunk = [&](int t0, int stage, int set, Operands& o) {
			const int at = stage * L::kStage;
			float up_x = 1.0f, up_b = 1.0f, up_c = 1.0f;
			if constexpr (!HALF)
			{
				const auto exponent = [&](int which, int highest) {
					const float* m = reinterpret_cast<const float*>(lds + L::kMost) + 12 * set + 4 * which;
					float most = m[0];
#pragma unroll
					for (int k = 1; k < PT; ++k) most = fmaxf(most, m[k]);
					return most > 0.0f ? half_exponent(most, kLowest, highest) : 0;
				};
				// (2^126 for B and C together: what their products become as weights is to be a float)
				const int k_x = exponent(0, kHighest);
				int k_b = exponent(1, kHighest), k_c = STATES ? 0 : exponent(2, kHighest);
				const int excess = k_b + k_c > 126 ? k_b + k_c - 126 : 0;
				k_b -= excess >> 1;
				k_c -= excess - (excess >> 1);
				up_x = power_of_two(k_x);
				up_b = power_of_two(k_b);
				up_c = power_of_two(k_c);
				if (tid == 0)
				{
					float* const out = reinterpret_cast<float*>(lds + L::kSteps + set * L::kSet) + L::kArrays * kChunk;
					int* const back = reinterpret_cast<int*>(out);
					// The products of B and C are up to 2^38; as weights they are 2^30 times less, and less than that where D would not be a float of their unit.
					const int skip_exponent = ((__builtin_bit_cast(int, skip) >> 23) & 255) - 126, room = 100 - (skip_exponent > 0 ? skip_exponent : 0);
					int unit = k_b + k_c - 30 < room ? k_b + k_c - 30 : room;
					unit = unit > k_b + k_c - 126 ? unit : k_b + k_c - 126;
					out[L::kScaleBC] = power_of_two(unit - k_b - k_c);                       // products of B and C -> weights, 2^unit times what they are
					out[L::kSkip] = __builtin_amdgcn_ldexpf(skip, unit);
					back[L::kBackX] = -(unit + k_x);                                         // products of x and weights -> results
					back[L::kBackC] = -k_c;                                                  // products of the state and C -> results
					back[L::kBackBX] = -(k_b + k_x);                                         // products of B and x -> the state
				}
			}
			store_rows(o.x, at + L::kX, L::kPitchX, L::kXLow, up_x, 0);
#pragma unroll 1
			for (int part = 0; part < PARTS; ++part)
			{
				if constexpr (!AHEAD)
				{
					if (t0 + kChunk <= end)
					{
#pragma unroll
						for (int i = 0; i < BA; ++i)
						{
							o.b[i] = *fetch(b + t0, offset(i + part * BA, size, a.b_row));
							if constexpr (!STATES) o.c[i] = *fetch(c + t0, offset(i + part * BA, size, a.c_row));
						}
					}
					else
					{
						load_tail(o.b, b + t0, a.b_row, size, end - t0, part);
						if constexpr (!STATES) load_tail(o.c, c + t0, a.c_row, size, end - t0, part);
					}
				}
				if (size < NT)
				{
#pragma unroll
					for (int i = 0; i < BA; ++i)
						if (vrow + (i + part * BA) * ROW_STEP >= size) o.b[i] = Vec{};
				}
				store_rows(o.b, at + L::kB, L::kPitchB, L::kBLow, up_b, part);
				if constexpr (!STATES) store_rows(o.c, at + L::kC, L::kPitchB, L::kBLow, up_c, part);
			}
		};
		// the state in front of a chunk, for the results
		const auto leave_state = [&](int front) {
			if constexpr (!STATES)
			{
				char* const to = lds + L::kFronts + front * L::kFront;
				char* const row = to + hp * L::kPitchH;
				float most = 0.0f;
#pragma unroll
				for (int i = 0; i < NB; ++i)
#pragma unroll
					for (int r = 0; r < 4; ++r) most = fmaxf(most, __builtin_fabsf(h[i][r]));
				// a scale for every row, which is a sequence of its own
				const int k = half_exponent(max_over_lane_rows(most), kLowest, HALF ? 112 : kHighest);
				const float up = power_of_two(k);
#pragma unroll
				for (int i = 0; i < NB; ++i)
				{
					char* const at = row + (16 * i + 4 * g) * 2;
					if constexpr (HALF) *reinterpret_cast<half4_t*>(at) = __builtin_convertvector(h[i] * up, half4_t);
					else
					{
						half4_t first, second;
						split_wide(h[i] * up, first, second);
						*reinterpret_cast<half4_t*>(at) = first;
						*reinterpret_cast<half4_t*>(at + L::kHLow) = second;
					}
				}
				// what a row's products are worth: a factor, in float32 an exponent
				if (g == 0) *reinterpret_cast<int*>(to + (hp >> 2) * L::kPitchH + L::kScales + (hp & 3) * 4) = HALF ? __builtin_bit_cast(int, power_of_two(-k) * (1.0f / kUnit)) : -k;
			}
		};
		if constexpr (HALF)
		{
#pragma unroll
			for (int i = 0; i < NB; ++i) h[i] = h[i] * kUnit;
		}
		// (the state is there from here on: without this the loop waits for its loads where it first uses it, behind loads of its own)
#pragma unroll
		for (int i = 0; i < NB; ++i) asm volatile("" : "+v"(h[i]));
		T raw = (T)0.0f;
		if (MOVERS && moves)
		{
			// Two chunks under way: a chunk's loads have the time of two until they are waited for, and nobody waits for them while another is split (4 x 4096 tokens,
			// 64 heads: 233 us with one, 198 with two, before the second halves had a scale of their own)
			Operands even, odd;
			if (begin < end)
			{
				load_chunk(begin, even);
				if (stepper) raw = load_step(begin);
				load_chunk(begin + kChunk, odd);
				note_most(0, even);
			}
			__syncthreads();
			if (begin < end)
			{
				store_chunk(begin, 0, 0, even);
				if (stepper)
				{
					make_steps(begin, (float)raw, 0);
					if (begin + kChunk < end) raw = load_step(begin + kChunk);
				}
				load_chunk(begin + 2 * kChunk, even);
				if (begin + kChunk < end) note_most(1, odd);
			}
			__syncthreads();
			// beside the work on the chunk at t0: the next one into the LDS, the scales of the one behind it
			const auto beside = [&](int t0, auto turn, auto whole, Operands& next, Operands& later) {
				constexpr int TURN = decltype(turn)::value;
				constexpr bool WHOLE = decltype(whole)::value;
				const bool more = WHOLE || t0 + kChunk < end;
				const T raw_next = raw;
				if (stepper && t0 + 2 * kChunk < end) raw = load_step(t0 + 2 * kChunk);
				if (more) store_chunk(t0 + kChunk, TURN ^ 1, TURN ^ 1, next);
				load_chunk(t0 + 3 * kChunk, next, WHOLE);
				if (more && stepper) make_steps(t0 + kChunk, (float)raw_next, TURN ^ 1);
				if (WHOLE || t0 + 2 * kChunk < end) note_most(TURN, later);
				__syncthreads();
			};
			const std::integral_constant<int, 0> first;
			const std::integral_constant<int, 1> second;
			int t0 = begin;
			// (as long as there are whole chunks to load, no way around a load: only then are the waits for the loads before it no waits for it)
			for (; end - t0 >= 5 * kChunk; t0 += 2 * kChunk)
			{
				beside(t0, first, std::true_type{}, odd, even);
				beside(t0 + kChunk, second, std::true_type{}, even, odd);
			}
			for (; t0 < end; t0 += 2 * kChunk)
			{
				beside(t0, first, std::false_type{}, odd, even);
				if (t0 + kChunk < end) beside(t0 + kChunk, second, std::false_type{}, even, odd);
			}
			return;
		}
		Operands next;
		if (begin < end)
		{
			if (!MOVERS) load_chunk(begin, next);
			if (stepper) raw = load_step(begin);
			leave_state(0);
			if (!MOVERS) note_most(0, next);
		}
		if constexpr (!HALF) __syncthreads();
		if (begin < end)
		{
			if (!MOVERS) store_chunk(begin, 0, 0, next);
			if (stepper)
			{
				make_steps(begin, (float)raw, 0);
				if (begin + kChunk < end) raw = load_step(begin + kChunk);
			}
			if constexpr (!MOVERS)
			{
				load_chunk(begin + kChunk, next);
				if (DOUBLE && begin + kChunk < end) note_most(1, next);
			}
		}
		__syncthreads();
		int turn = 0;
		for (int t0 = begin; t0 < end; t0 += kChunk, turn ^= 1)
		{
			const bool more = t0 + kChunk < end;
			const T raw_next = raw;
			if (stepper && t0 + 2 * kChunk < end) raw = load_step(t0 + 2 * kChunk);
			if constexpr (DOUBLE && !MOVERS)
			{
				if (more) store_chunk(t0 + kChunk, turn ^ 1, turn ^ 1, next);
				load_chunk(t0 + 2 * kChunk, next);
			}
			const char* const ops = lds + (DOUBLE ? turn * L::kStage : 0);
			const float* steps = reinterpret_cast<const float*>(lds + L::kSteps + turn * L::kSet);
			const float keep = steps[L::kArrays * kChunk + L::kDecay];
			decay *= keep;

			// w x, as two halves
			float4_t v[4];
			float most = 0.0f;
#pragma unroll
			for (int kk = 0; kk < 2; ++kk)
			{
				const char* const at = ops + L::kX + hp * L::kPitchX + (32 * kk + 8 * g) * 2;
				const half8_t xs = *reinterpret_cast<const half8_t*>(at);
				half8_t xl;
				if constexpr (!HALF) xl = *reinterpret_cast<const half8_t*>(at + L::kXLow);
#pragma unroll
				for (int q = 0; q < 2; ++q)
				{
					const float4_t w = *reinterpret_cast<const float4_t*>(steps + L::kWeight * kChunk + 32 * kk + 8 * g + 4 * q);
					const half2_t x0 = {xs[4 * q], xs[4 * q + 1]}, x1 = {xs[4 * q + 2], xs[4 * q + 3]};
					float4_t u = {times_half<0>(x0, w[0]), times_half<1>(x0, w[1]), times_half<0>(x1, w[2]), times_half<1>(x1, w[3])};
					if constexpr (!HALF)
					{
						const half2_t y0 = {xl[4 * q], xl[4 * q + 1]}, y1 = {xl[4 * q + 2], xl[4 * q + 3]};
						const float4_t w_low = w * (1.0f / kLowUnit);
						u = float4_t{times_half_add<0>(y0, w_low[0], u[0]), times_half_add<1>(y0, w_low[1], u[1]), times_half_add<0>(y1, w_low[2], u[2]), times_half_add<1>(y1, w_low[3], u[3])};
					}
					v[2 * kk + q] = u;
#pragma unroll
					for (int e = 0; e < 4; ++e) most = fmaxf(most, __builtin_fabsf(u[e]));
				}
			}
			float into = keep, down = 1.0f;
			bool scaled = false;
			int back = 0;                                         // float32: 2^back, products -> the state
			if constexpr (HALF)
			{
				// (below 2^-4 the second half of a value lies among the numbers whose last bit is worth 2^-24, which leaves 21 bits)
				scaled = rows_need_scale(most, 0.0625f);
				if (scaled)
				{
					// (the state goes along, as far as it remains a float)
					float largest = 0.0f;
#pragma unroll
					for (int i = 0; i < NB; ++i)
#pragma unroll
						for (int r = 0; r < 4; ++r) largest = fmaxf(largest, __builtin_fabsf(h[i][r]));
					const int k_most = half_exponent(max_over_lane_rows(most), kLowest, kHighest),
					          room = 252 - ((__builtin_bit_cast(int, max_over_lane_rows(largest)) >> 23) & 255), k = k_most < room ? k_most : room;
					const float up = power_of_two(k);
					into *= up;
					down = power_of_two(-k);
#pragma unroll
					for (int q = 0; q < 4; ++q) v[q] = v[q] * up;
				}
			}
			else
			{
				const int k = half_exponent(max_over_lane_rows(most), kLowest, kHighest);
				const float up = power_of_two(k);
				back = reinterpret_cast<const int*>(steps)[L::kArrays * kChunk + L::kBackBX] - k;
#pragma unroll
				for (int q = 0; q < 4; ++q) v[q] = v[q] * up;
			}
			half4_t hi[4], low[4];
#pragma unroll
			for (int q = 0; q < 4; ++q)
			{
				if constexpr (HALF) split(v[q], hi[q], low[q]);
				else split_wide(v[q], hi[q], low[q]);
			}
			if constexpr (HALF)
			{
#pragma unroll
				for (int i = 0; i < NB; ++i) h[i] = h[i] * into;
#pragma unroll
				for (int kk = 0; kk < 2; ++kk)
				{
					const half8_t v_low = join(low[2 * kk], low[2 * kk + 1]), v_hi = join(hi[2 * kk], hi[2 * kk + 1]);
					const char* const at = ops + L::kB + l * L::kPitchB + (32 * kk + 8 * g) * 2;
					half8_t bf[NB];
#pragma unroll
					for (int i = 0; i < NB; ++i) bf[i] = *reinterpret_cast<const half8_t*>(at + 16 * i * L::kPitchB);
#pragma unroll
					for (int i = 0; i < NB; ++i) h[i] = mfma(bf[i], v_low, h[i]);
#pragma unroll
					for (int i = 0; i < NB; ++i) h[i] = mfma(bf[i], v_hi, h[i]);
				}
				if (scaled)
				{
#pragma unroll
					for (int i = 0; i < NB; ++i) h[i] = h[i] * down;
				}
			}
			else
			{
				// sums of their own, two tiles at a time: the state may be far from what enters it, and keeps its range
				constexpr int TILES = 2;
#pragma unroll
				for (int i0 = 0; i0 < NB; i0 += TILES)
				{
					float4_t sum[TILES], low_sum[TILES];
#pragma unroll
					for (int i = 0; i < TILES; ++i) sum[i] = low_sum[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
					for (int kk = 0; kk < 2; ++kk)
					{
						const half8_t v_low = join(low[2 * kk], low[2 * kk + 1]), v_hi = join(hi[2 * kk], hi[2 * kk + 1]);
						const char* const at = ops + L::kB + (16 * i0 + l) * L::kPitchB + (32 * kk + 8 * g) * 2;
						half8_t bf[TILES];
#pragma unroll
						for (int i = 0; i < TILES; ++i) bf[i] = *reinterpret_cast<const half8_t*>(at + 16 * i * L::kPitchB + L::kBLow);
#pragma unroll
						for (int i = 0; i < TILES; ++i) low_sum[i] = mfma(bf[i], v_hi, low_sum[i]);
#pragma unroll
						for (int i = 0; i < TILES; ++i) bf[i] = *reinterpret_cast<const half8_t*>(at + 16 * i * L::kPitchB);
#pragma unroll
						for (int i = 0; i < TILES; ++i) low_sum[i] = mfma(bf[i], v_low, low_sum[i]);
#pragma unroll
						for (int i = 0; i < TILES; ++i) sum[i] = mfma(bf[i], v_hi, sum[i]);
					}
#pragma unroll
					for (int i = 0; i < TILES; ++i)
					{
						const float4_t both = add_low(sum[i], low_sum[i]);
#pragma unroll
						for (int r = 0; r < 4; ++r) h[i0 + i][r] = fmaf(h[i0 + i][r], keep, __builtin_amdgcn_ldexpf(both[r], back));
					}
				}
			}
			if (more && stepper) make_steps(t0 + kChunk, (float)raw_next, turn ^ 1);
			if constexpr (DOUBLE)
			{
				if (more) leave_state(turn ^ 1);
				if (!MOVERS && t0 + 2 * kChunk < end) note_most(turn, next);
				__syncthreads();
			}
			else
			{
				if (more) note_most(turn ^ 1, next);
				__syncthreads();
				if (more)
				{
					store_chunk(t0 + kChunk, 0, turn ^ 1, next);
					leave_state(0);
					load_chunk(t0 + 2 * kChunk, next);
					__syncthreads();
				}
			}
		}
		if constexpr (HALF)
		{
#pragma unroll
			for (int i = 0; i < NB; ++i) h[i] = h[i] * (1.0f / kUnit);
		}
		if constexpr (STATES)
		{
#pragma unroll
			for (int i = 0; i < NB; ++i) slot(segment)[i * KT] = h[i];
			if (tid == 0) plan.decays[(int64_t)segment * plan.blocks + block] = decay;
		}
		else if (segment == plan.segments - 1 && a.state != nullptr && hp < rows)
		{
#pragma unroll
			for (int i = 0; i < NB; ++i)
			{
				const int n = 16 * i + 4 * g;
				if (wide && n < size) *reinterpret_cast<float4_t*>(state + n) = h[i];
				else if (n < size)
				{
#pragma unroll
					for (int r = 0; r < 4; ++r)
						if (n + r < size) state[n + r] = h[i][r];
				}
			}
		}
		return;
	}

	if constexpr (!STATES)
	{
		T* y = static_cast<T*>(a.y) + ((int64_t)batch * a.seqlen * a.heads + head) * a.head_dim + p0;
		const int64_t y_token = (int64_t)a.heads * a.head_dim;
		// the waves of a block have one to four tiles of weights each; blocks deal them out differently, so that no SIMD has all the long ones
		const int tt = (wave + (int)blockIdx.x) & 3;
		T* to = y + (begin + 16 * tt + l) * y_token;
		// A lane's groups of four in its row of H and of X.  Two reads of 8 bytes take 2 cycles each, the one instruction that the compiler makes of two whose
		// distance it sees takes 16 (it goes 16 lanes at a time, which meet at a pitch of 144): it is not to see the distance.
		int h_at[NB], x_at[4];
#pragma unroll
		for (int k = 0; k < NB; ++k)
		{
			h_at[k] = l * L::kPitchH + (16 * k + 4 * g) * 2;
			asm volatile("" : "+v"(h_at[k]));
		}
#pragma unroll
		for (int k = 0; k < 4; ++k)
		{
			x_at[k] = l * L::kPitchX + (16 * k + 4 * g) * 2;
			asm volatile("" : "+v"(x_at[k]));
		}
		// in a token's own tile: D for itself (nothing of the tokens behind it, whatever they are)
		float4_t itself;
#pragma unroll
		for (int r = 0; r < 4; ++r) itself[r] = 4 * g + r == l ? (HALF ? skip : 1.0f) : 0.0f;
		const auto chunk = [&](auto which, int t0, int turn, auto before_stores) {
			constexpr int TT = decltype(which)::value;
			const char* const ops = lds + (DOUBLE ? turn * L::kStage : 0);
			const char* const front = lds + L::kFronts + (DOUBLE ? turn * L::kFront : 0);
			const float* steps = reinterpret_cast<const float*>(lds + L::kSteps + turn * L::kSet);
			const int t = 16 * TT + l;
			float4_t acc[PT];                                 // Y^T: rows p = 16 pt + 4 g + r, column t; first what the state in front gives
			float4_t gw[TT + 1];                             // G, then the weights: rows s = 16 j + 4 g + r, column t
#pragma unroll
			for (int pt = 0; pt < PT; ++pt) acc[pt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
			for (int j = 0; j <= TT; ++j) gw[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
			half8_t cf[NT / 32], cl[HALF ? 1 : NT / 32];
#pragma unroll
			for (int q = 0; q < NT / 32; ++q)
			{
				const char* src = ops + L::kC + (32 * q + 4 * g + (l >> 2)) * L::kPitchB + (16 * TT + 4 * (l & 3)) * 2;
				cf[q] = join(read_transposed(src), read_transposed(src + 16 * L::kPitchB));
				if constexpr (!HALF) cl[q] = join(read_transposed(src + L::kBLow), read_transposed(src + L::kBLow + 16 * L::kPitchB));
			}
#pragma unroll
			for (int j = 0; j <= TT; ++j)
			{
				float4_t low_sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
				for (int q = 0; q < NT / 32; ++q)
				{
					const char* src = ops + L::kB + (32 * q + 4 * g + (l >> 2)) * L::kPitchB + (16 * j + 4 * (l & 3)) * 2;
					const half8_t bf = join(read_transposed(src), read_transposed(src + 16 * L::kPitchB));
					if constexpr (!HALF)
					{
						const half8_t bl = join(read_transposed(src + L::kBLow), read_transposed(src + L::kBLow + 16 * L::kPitchB));
						low_sum = mfma(bl, cf[q], low_sum);
						low_sum = mfma(bf, cl[q], low_sum);
					}
					gw[j] = mfma(bf, cf[q], gw[j]);
				}
				if constexpr (!HALF) gw[j] = add_low(gw[j], low_sum);
			}
#pragma unroll
			for (int pt = 0; pt < PT; ++pt)
			{
				float4_t low_sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
				for (int q = 0; q < NT / 32; ++q)
				{
					const char* const row = front + 16 * pt * L::kPitchH;
					const half8_t hf = join(*reinterpret_cast<const half4_t*>(row + h_at[2 * q]), *reinterpret_cast<const half4_t*>(row + h_at[2 * q + 1]));
					if constexpr (!HALF)
					{
						const half8_t hl = join(*reinterpret_cast<const half4_t*>(row + L::kHLow + h_at[2 * q]), *reinterpret_cast<const half4_t*>(row + L::kHLow + h_at[2 * q + 1]));
						low_sum = mfma(hl, cf[q], low_sum);
						low_sum = mfma(hf, cl[q], low_sum);
					}
					acc[pt] = mfma(hf, cf[q], acc[pt]);
				}
				if constexpr (!HALF) acc[pt] = add_low(acc[pt], low_sum);
			}
			// ---- weights: G exp(L_t - L_s) delta_s, the skip term on the diagonal ----
			const float in = steps[L::kIn * kChunk + t], in_low = steps[L::kInLow * kChunk + t], gain = steps[L::kGain * kChunk + t];
			const float own = HALF ? 1.0f : steps[L::kArrays * kChunk + L::kSkip];
			// (float32 without waves that only fetch: compared anew in every chunk, for the masks would take eight scalar registers that there are not)
			int later = 4 * g;
			if constexpr (!HALF && !MOVERS) asm volatile("" : "+v"(later));
			float since = in;                                // from the end of the tile j to the token
			float most = 0.0f;
#pragma unroll
			for (int j = TT; j >= 0; --j)
			{
				const int s = 16 * j + 4 * g;
				if (j < TT - 1) since += steps[L::kArrays * kChunk + j + 1];
				float4_t e;
				if (j < TT)
				{
					const float4_t out = *reinterpret_cast<const float4_t*>(steps + L::kOut * kChunk + s);
#pragma unroll
					for (int r = 0; r < 4; ++r) e[r] = fast_exp2(since + out[r]);
				}
				else
				{
					const float4_t from = *reinterpret_cast<const float4_t*>(steps + (HALF ? L::kFrom : L::kIn) * kChunk + s);
					const float4_t low = *reinterpret_cast<const float4_t*>(steps + (HALF ? L::kFromLow : L::kInLow) * kChunk + s);
#pragma unroll
					for (int r = 0; r < 4; ++r) e[r] = fast_exp2((in - from[r]) + (in_low - low[r]));
				}
				if constexpr (!HALF)
				{
					// (the smallest and the largest steps last: their products with the scale alone may be no floats)
					gw[j] = gw[j] * (e * steps[L::kArrays * kChunk + L::kScaleBC]);
					e = *reinterpret_cast<const float4_t*>(steps + L::kDelta * kChunk + s);
				}
#pragma unroll
				for (int r = 0; r < 4; ++r)
				{
					if (j < TT) gw[j][r] = gw[j][r] * e[r];
					else gw[j][r] = later + r > l ? 0.0f : fmaf(gw[j][r], e[r], HALF ? itself[r] : itself[r] * own);
					most = fmaxf(most, __builtin_fabsf(gw[j][r]));
				}
			}
			// A column's largest weight, D among them, goes to the top of a half's range: those down to 2^-29 of it keep all their bits.  (Half precision: by 2^22 at
			// most.  What is lost of a weight then lies below 2^-47, of a result below 64 * 2^16 * 2^-47, half the last bit of the smallest halves; and the scale of a state, 2^105 at
			// most, remains a float with it.)
			const int k = half_exponent(max_over_lane_rows(most), kLowest, HALF ? 22 : kHighest);
			const float up = power_of_two(k), into = gain * up, down = power_of_two(-k);      // half precision: products with C -> those with the weights -> results
			int back_c = 0, back_w = 0;                                                       // float32: exponents of what either are worth
			if constexpr (!HALF)
			{
				const int* const back = reinterpret_cast<const int*>(steps) + L::kArrays * kChunk;
				back_c = back[L::kBackC];
				back_w = back[L::kBackX] - k;
			}
#pragma unroll
			for (int j = 0; j <= TT; ++j) gw[j] = gw[j] * up;
			const half4_t none = {};
			half4_t wf[TT + 1], wl[TT + 1];
#pragma unroll
			for (int j = 0; j <= TT; ++j)
			{
				// (half precision: the remainders of the own tile only)
				if (HALF && j < TT)
				{
					wf[j] = __builtin_convertvector(gw[j], half4_t);
					wl[j] = none;
				}
				else if constexpr (HALF) split(gw[j], wf[j], wl[j]);
				else split_wide(gw[j], wf[j], wl[j]);
			}
#pragma unroll
			for (int pt = 0; pt < PT; ++pt)
			{
				// float32: apart from the state's part, which has a scale of its own.  (In half precision a result that is far from its weights is no half.)
				float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f}, low_sum = sum;
				const char* const scales = front + (4 * pt + g) * L::kPitchH + L::kScales;
				if constexpr (HALF) sum = acc[pt] * (*reinterpret_cast<const float4_t*>(scales) * into);
#pragma unroll
				for (int kk = 0; 2 * kk <= TT; ++kk)
				{
					const char* const row = ops + L::kX + 16 * pt * L::kPitchX;
					const half8_t xf = join(*reinterpret_cast<const half4_t*>(row + x_at[2 * kk]), *reinterpret_cast<const half4_t*>(row + x_at[2 * kk + 1]));
					constexpr int LAST = TT;
					const bool pair = 2 * kk + 1 <= LAST;
					const half8_t w_hi = join(wf[2 * kk], pair ? wf[pair ? 2 * kk + 1 : 0] : none), w_low = join(wl[2 * kk], pair ? wl[pair ? 2 * kk + 1 : 0] : none);
					if constexpr (!HALF)
					{
						const half8_t xl = join(*reinterpret_cast<const half4_t*>(row + L::kXLow + x_at[2 * kk]), *reinterpret_cast<const half4_t*>(row + L::kXLow + x_at[2 * kk + 1]));
						low_sum = mfma(xl, w_hi, low_sum);
						low_sum = mfma(xf, w_low, low_sum);
					}
					else if (kk == TT / 2) sum = mfma(xf, w_low, sum);
					sum = mfma(xf, w_hi, sum);
				}
				if constexpr (HALF) acc[pt] = sum * down;
				else
				{
					typedef int Exponents __attribute__((ext_vector_type(4)));
					const Exponents back_h = *reinterpret_cast<const Exponents*>(scales);
					sum = add_low(sum, low_sum);
#pragma unroll
					for (int r = 0; r < 4; ++r)
						acc[pt][r] = __builtin_amdgcn_ldexpf(acc[pt][r] * gain, back_h[r] + back_c) + __builtin_amdgcn_ldexpf(sum[r], back_w);      // (decayed first: the products of a large state may be no floats)
				}
			}
			before_stores();
			if (t0 + t < end)
			{
				int live = rows;
				asm volatile("" : "+s"(live));
#pragma unroll
				for (int pair = 0; pair < PT / 2; ++pair)
				{
					if (HALF && 32 * pair + 32 <= live)
					{
						// Two tiles' groups of four change places between neighbouring rows of lanes, which leaves every lane eight consecutive results: stores of
						// 16 bytes, four lanes to 64 contiguous ones.
						unsigned d[2][2];
#pragma unroll
						for (int k = 0; k < 2; ++k)
						{
							const Quad q = __builtin_convertvector(acc[2 * pair + k], Quad);
							__builtin_memcpy(d[k], &q, 8);
						}
#pragma unroll
						for (int k = 0; k < 2; ++k) asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(d[0][k]), "+v"(d[1][k]));
						half8_t v;
						__builtin_memcpy(&v, d, 16);
						typedef half8_t LooseHalves __attribute__((aligned(2)));
						*reinterpret_cast<LooseHalves*>(to + 32 * pair + 16 * (g & 1) + 4 * (g & 2)) = v;
					}
					else
					{
#pragma unroll
						for (int k = 0; k < 2; ++k)
						{
							const int p = 32 * pair + 16 * k + 4 * g;
							float4_t v = acc[2 * pair + k];
							if (p + 3 < live)
							{
								if constexpr (!HALF)
									if (a.add) v = v + *reinterpret_cast<const LooseQuad*>(to + p);
								*reinterpret_cast<LooseQuad*>(to + p) = __builtin_convertvector(v, Quad);
							}
							else
							{
#pragma unroll
								for (int r = 0; r < 3; ++r)
									if (p + r < live) to[p + r] = (T)(!HALF && a.add ? v[r] + (float)to[p + r] : v[r]);
							}
						}
					}
				}
			}
		};
		const auto walk = [&](auto which) {
			// the waves with one tile of weights sum up the steps of the next chunk (first, so that they wait for none of their stores)
			constexpr bool STEPPER = decltype(which)::value == 0;
			T raw = (T)0.0f;
			if (STEPPER && begin < end)
			{
				make_steps(begin, (float)load_step(begin), 0);
				if (begin + kChunk < end) raw = load_step(begin + kChunk);
			}
			float next_raw = (float)raw;
			if constexpr (!HALF) __syncthreads();
			__syncthreads();
			int turn = 0;
			for (int t0 = begin; t0 < end; t0 += kChunk, turn ^= 1, to += kChunk * y_token)
			{
				if (STEPPER && t0 + kChunk < end)
				{
					if (t0 + 2 * kChunk < end) raw = load_step(t0 + 2 * kChunk);
					make_steps(t0 + kChunk, next_raw, turn ^ 1);
				}
				chunk(which, t0, turn, [&] {
					// (waited for here, ahead of the stores, or the wait at the next chunk's start would be one for them)
					next_raw = (float)raw;
					if constexpr (STEPPER) asm volatile("" : "+v"(next_raw));
				});
				__syncthreads();
				if constexpr (!DOUBLE)
					if (t0 + kChunk < end) __syncthreads();
			}
		};
		switch (tt)
		{
		case 0: walk(std::integral_constant<int, 0>{}); break;
		case 1: walk(std::integral_constant<int, 1>{}); break;
		case 2: walk(std::integral_constant<int, 2>{}); break;
		default: walk(std::integral_constant<int, 3>{}); break;
		}
		// tokens behind the row's end
		for (int t = (end > begin ? end : begin) + wave; t < limit; t += 4)
			if (lane < rows) y[t * y_token + lane] = (T)0.0f;
	}
}

}  // namespace scan

}  // namespace anygpu
