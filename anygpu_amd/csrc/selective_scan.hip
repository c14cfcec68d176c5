// Selective scan (Mamba2) for gfx950: prompts and chunks of prompts.  y and the final state of
//     H_t = exp(delta_t A) H_{t-1} + delta_t x_t B_t^T,   y_t = H_t C_t + D x_t
// In chunks of 64 tokens on the matrix cores (selective_scan_chunk.hpp); here are the plan of such a launch, and the scan token by token for what the chunks' kernel
// does not take, rows of x, B or C that lie gigabytes apart: a wave has a row of H (one of head_dim), four elements of the state a lane, in registers for the whole
// sequence, and every token waits for its operands (2 x 2048 tokens, 32 heads, state 256, float32: 13.8 ms, in chunks 140 us).
#include "selective_scan.hpp"
#include "selective_scan_chunk.hpp"
#include "launch.hpp"

#include <algorithm>

namespace anygpu {

namespace {

constexpr int kScanThreads = 256;
constexpr int kFloatStates = 128;       // elements of the state whose float32 operands the LDS holds, as two halves each

template <typename T>
__global__ __launch_bounds__(kScanThreads) void selective_scan_token_kernel(const ScanArgs a)
{
	constexpr int ROWS = kScanThreads / 64;
	const int row_blocks = (a.head_dim + ROWS - 1) / ROWS;
	const int bh = blockIdx.x / row_blocks;
	const int p = (blockIdx.x - bh * row_blocks) * ROWS + threadIdx.x / 64;
	const int batch = bh / a.heads, head = bh - batch * a.heads, group = head / (a.heads / a.groups);
	const int n0 = (threadIdx.x % 64) * 4;
	const bool live = p < a.head_dim;
	const int pc = live ? p : 0;
	const T* x = static_cast<const T*>(a.x) + batch * a.x_batch + ((int64_t)head * a.head_dim + pc) * a.x_row;
	const T* dt = static_cast<const T*>(a.dt) + batch * a.dt_batch + head * a.dt_head;
	const T* b = static_cast<const T*>(a.b) + batch * a.b_batch + (int64_t)group * a.state_dim * a.b_row;
	const T* c = static_cast<const T*>(a.c) + batch * a.c_batch + (int64_t)group * a.state_dim * a.c_row;
	T* y = static_cast<T*>(a.y) + ((int64_t)batch * a.seqlen * a.heads + head) * a.head_dim + pc;
	float* state = a.state ? a.state + ((int64_t)bh * a.head_dim + pc) * a.state_dim : nullptr;
	const float rate = a.a[head], bias = a.bias ? a.bias[head] : 0.0f, skip = a.skip ? a.skip[head] : 0.0f;
	const int length = scan_length(a.lengths, batch, a.seqlen);

	float h[4];
#pragma unroll
	for (int i = 0; i < 4; ++i) h[i] = state && n0 + i < a.state_dim ? state[n0 + i] : 0.0f;
	for (int t = 0; t < length; ++t)
	{
		const float delta = scan_delta((float)dt[t * a.dt_seq], bias, a.dt_min, a.dt_max);
		const float keep = expf(delta * rate), xv = (float)x[t], dx = delta * xv;
		float sum = 0.0f;
#pragma unroll
		for (int i = 0; i < 4; ++i)
		{
			if (n0 + i >= a.state_dim) continue;
			h[i] = fmaf(h[i], keep, dx * (float)b[(n0 + i) * a.b_row + t]);
			sum = fmaf(h[i], (float)c[(n0 + i) * a.c_row + t], sum);
		}
		sum = wave_allreduce(sum, SumOp());
		if (live && n0 == 0) y[(int64_t)t * a.heads * a.head_dim] = (T)(a.skip ? fmaf(skip, xv, sum) : sum);
	}
	if (live && n0 == 0)
		for (int t = length; t < a.seqlen; ++t) y[(int64_t)t * a.heads * a.head_dim] = (T)0.0f;
	if (live && state)
	{
#pragma unroll
		for (int i = 0; i < 4; ++i)
			if (n0 + i < a.state_dim) state[n0 + i] = h[i];
	}
}

template <typename T>
hipError_t launch_token(const ScanArgs& a, hipStream_t stream)
{
	constexpr int ROWS = kScanThreads / 64;
	const int64_t blocks = (int64_t)a.batch * a.heads * ((a.head_dim + ROWS - 1) / ROWS);
	if (blocks > 0x7FFFFFFFLL) return hipErrorInvalidConfiguration;
	discard_stale_error();
	selective_scan_token_kernel<T><<<dim3((unsigned)blocks), dim3(kScanThreads), 0, stream>>>(a);
	return hipGetLastError();
}

// Rows of a block: heads of 32 rows take blocks of 32 (4 x 4096 tokens, 64 heads, f16 78 us, in half empty blocks of 64 88; heads of 64 in two blocks of
// 32: 157 against 90, twice the weights and twice the fetching of B and C).
// Segments: sequences whose blocks leave compute units without work are cut, in pieces of four chunks at least.  The pass that finds the segments'
// states costs about half of the other one, so that two blocks on a compute unit (the half precision form up to a state of 64) pay from three segments on, one
// from two on (16384 tokens, 128 heads, f16: uncut 328 us, 4 segments 253, 8 285; 3 x 4096 tokens, 64 heads, f16: uncut 84, 2 segments 97; 2 x 2048 tokens, 64 heads,
// f32: 82, 2 segments 69; one such sequence 81, 4 segments 47, 8 57), and that short sequences stay whole (500 tokens, 64 heads, f16: 15.0 us, cut 15.9; f32 27.6, 26.1).  The first pass takes half a segment per block where all its blocks are then
// still resident at once (16000 tokens, 128 heads, f16: 245 us whole, 231 in halves; 3 x 1001 tokens, 32 heads, state 128, f32: 72, 64; where they
// are not, 8192 tokens, 2 x 32 heads, f16: 67, 68).
scan::Plan make_plan(bool half, int64_t batch, int64_t heads, int64_t head_dim, int64_t state_dim, int64_t seqlen)
{
	scan::Plan plan{};
	plan.rows = head_dim <= 32 && state_dim <= 64 ? 32 : 64;
	plan.row_tiles = (int)((head_dim + plan.rows - 1) / plan.rows);
	const int64_t blocks = batch * heads * plan.row_tiles, chunks = (seqlen + scan::kChunk - 1) / scan::kChunk, cus = device_cu_count();
	plan.blocks = (int)std::min<int64_t>(blocks, 0x7FFFFFFFLL);
	int64_t segments = 1;
	if (chunks > 8 && blocks < cus)
	{
		const bool two = half && state_dim <= 64;
		segments = std::min<int64_t>((two ? 2 : 1) * cus / blocks, chunks / 4);
		if (segments < (two ? 3 : 2)) segments = 1;
	}
	int64_t per = (chunks + segments - 1) / segments;
	plan.segments = (int)((chunks + per - 1) / per);
	const int64_t resident = half ? (state_dim <= 64 ? 3 : state_dim <= 128 ? 2 : 1) : 1;       // blocks of the first pass on a compute unit
	plan.parts = plan.segments > 1 && per >= 4 && 2 * (plan.segments - 1) * blocks <= resident * cus ? 2 : 1;
	if (plan.parts == 2 && per % 2 != 0)
	{
		per += 1;
		plan.segments = (int)((chunks + per - 1) / per);
	}
	plan.segment_tokens = (int)std::min<int64_t>(per * scan::kChunk, 0x7FFFFFFFLL);
	return plan;
}

// the state's size in the kernels' tiles
int padded_state(int64_t size) { return size <= 32 ? 32 : size <= 64 ? 64 : size <= 128 ? 128 : 256; }

int64_t state_bytes(const scan::Plan& plan, int64_t size) { return (int64_t)plan.segments * plan.parts * plan.blocks * padded_state(size) * plan.rows * 4; }

template <typename T, int NT, int R, bool STATES>
hipError_t launch_chunks(const ScanArgs& a, const scan::Plan& plan, int64_t blocks, hipStream_t stream)
{
	static std::atomic<uint64_t> granted{0};
	const auto kernel = scan::selective_scan_chunk_kernel<T, NT, R, STATES>;
	using L = scan::Lds<T, NT, R, STATES>;
	static_assert(L::kBytes <= 160 * 1024, "LDS of a CU");
	const hipError_t e = grant_lds(kernel, L::kBytes, granted);
	if (e != hipSuccess) return e;
	discard_stale_error();
	kernel<<<dim3((unsigned)blocks), dim3(L::kThreads), L::kBytes, stream>>>(a, plan);
	return hipGetLastError();
}

template <typename T, int NT, int R>
hipError_t launch_rows(const ScanArgs& a, scan::Plan plan, void* workspace, hipStream_t stream)
{
	if ((int64_t)plan.blocks * plan.segments * plan.parts > 0x7FFFFFFFLL) return hipErrorInvalidConfiguration;
	if (plan.segments > 1)
	{
		plan.states = static_cast<float*>(workspace);
		plan.decays = plan.states + state_bytes(plan, a.state_dim) / 4;
		scan::Plan first = plan;
		first.segments *= plan.parts;
		first.segment_tokens /= plan.parts;
		first.parts = 1;
		const hipError_t e = launch_chunks<T, NT, R, true>(a, first, (int64_t)plan.blocks * (plan.segments - 1) * plan.parts, stream);
		if (e != hipSuccess) return e;
	}
	return launch_chunks<T, NT, R, false>(a, plan, (int64_t)plan.blocks * plan.segments, stream);
}

template <typename T, int NT>
hipError_t launch_size(const ScanArgs& a, void* workspace, hipStream_t stream)
{
	const scan::Plan plan = make_plan(sizeof(T) == 2, a.batch, a.heads, a.head_dim, a.state_dim, a.seqlen);
	if constexpr (NT <= 64)
		if (plan.rows == 32) return launch_rows<T, NT, 32>(a, plan, workspace, stream);
	return launch_rows<T, NT, 64>(a, plan, workspace, stream);
}

}  // namespace

int64_t selective_scan_workspace_bytes(int64_t batch, int64_t heads, int64_t head_dim, int64_t state_dim, int64_t seqlen)
{
	int64_t most = 0;
	for (bool half : {false, true})
	{
		const int64_t size = half ? state_dim : std::min<int64_t>(state_dim, kFloatStates);
		const scan::Plan plan = make_plan(half, batch, heads, head_dim, size, seqlen);
		if (plan.segments > 1) most = std::max(most, state_bytes(plan, size) + (int64_t)plan.segments * plan.parts * plan.blocks * 4);
	}
	return most;
}

template <typename T>
hipError_t launch_selective_scan(const ScanArgs& given, void* workspace, hipStream_t stream)
{
	// the chunks' kernel counts bytes inside of a head's tile of x and of a group's B and C in 32 bits
	const int64_t widest = std::max(64 * given.x_row, padded_state(given.state_dim) * std::max(given.b_row, given.c_row));
	if (widest > (0xFFFFFFFFLL - 1024) / (int64_t)sizeof(T)) return launch_token<T>(given, stream);
	ScanArgs a = given;
	a.state_row = a.state_dim;
	if (sizeof(T) == 4 && a.state_dim > kFloatStates)
	{
		// y is a sum over the state, whose elements know nothing of each other: the first ones with x's own term, then the others
		a.state_dim = kFloatStates;
		const hipError_t e = launch_size<T, kFloatStates>(a, workspace, stream);
		if (e != hipSuccess) return e;
		a.state_dim = given.state_dim - kFloatStates;
		a.b = static_cast<const T*>(a.b) + kFloatStates * a.b_row;
		a.c = static_cast<const T*>(a.c) + kFloatStates * a.c_row;
		if (a.state != nullptr) a.state += kFloatStates;
		a.skip = nullptr;
		a.add = true;
	}
	switch (padded_state(a.state_dim))
	{
	case 32: return launch_size<T, 32>(a, workspace, stream);
	case 64: return launch_size<T, 64>(a, workspace, stream);
	case 128: return launch_size<T, 128>(a, workspace, stream);
	default: break;
	}
	if constexpr (sizeof(T) == 2) return launch_size<T, 256>(a, workspace, stream);
	return hipErrorInvalidValue;
}

template hipError_t launch_selective_scan<half_t>(const ScanArgs&, void*, hipStream_t);
template hipError_t launch_selective_scan<float>(const ScanArgs&, void*, hipStream_t);

}  // namespace anygpu
