// The cross entropy over a vocabulary for up to eight rows of fp32 (its loss for up to 32): a token or a few of each text that is scored or
// decoded.
//
// The weights are then read for less arithmetic than reading them takes; what counts is that they come once, as they lie, without the
// planes that the tensor core wants of fp32 (vocabulary_loss.cu), and that nothing but fp32 multiply-adds stands between.  A block has
// a stretch of the vocabulary:
//   logits     tiles of 64 entries x 64 elements go through shared memory; four neighbouring threads share an entry, each taking
//              every fourth element for all the rows, two rows per instruction
//   forward    every thread keeps a running maximum and sum for its entries and a quarter of the rows; a block's join in the end
//   backward   dz of the stretch stays in shared memory; then a thread takes columns of the weights down the stretch, reading them once
//              more (out of L2 while they fit), and gives weights_diff as it goes and its part of hidden_diff at the end
// 4 x 203 rows over 106779 entries: loss 38 us, gradients 75 us; by planes 118 and 316.  Eight rows of 1031 over 30011: 70 + 183 us against 128
// + 315; sixteen 190 + 347 against 127 + 322.  16-bit rows are faster on the tensor core from the first on (one row of 1024 over
// 32000 bf16: 20 us there, 57 by this kernel).
#include "vocabulary_few.cuh"

namespace nb200 {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int TILE = FEW_TILE;       // vocabulary entries
constexpr int CHUNK = 64;            // elements of them at a time
constexpr int PITCH = CHUNK + 4;     // 8 entries x 4 elements of a warp's read lie in 32 different banks

// What a warp has in hand of a chunk: its eight entries' elements lane and lane + 32.
struct Staged {
	static constexpr int ROWS = TILE / WARPS;
	float v[ROWS][2];
	__device__ __forceinline__ void load(const FewParams& p, int entry0, int k0)
	{
		const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
		for(int i = 0; i < ROWS; ++i) {
			const int entry = entry0 + warp + i * WARPS;
			const float* const row = p.weights + static_cast<long long>(entry) * p.weightsRow;
#pragma unroll
			for(int j = 0; j < 2; ++j) {
				const int k = k0 + lane + 32 * j;
				v[i][j] = entry < p.vocabulary && k < p.width ? row[k] : 0.f;
			}
		}
	}
	__device__ __forceinline__ void store(float* tile) const
	{
		const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
		for(int i = 0; i < ROWS; ++i) {
			float* const to = tile + (warp + i * WARPS) * PITCH;
			to[lane] = v[i][0];
			to[lane + 32] = v[i][1];
		}
	}
};

// The rows' elements k0 .. k0 + 63, rows without data as zeros; stored as [element][row].
template<int NT>
struct StagedHidden {
	static constexpr int N = CHUNK * NT / THREADS;
	float v[N];
	__device__ __forceinline__ void load(const FewParams& p, int k0)
	{
#pragma unroll
		for(int i = 0; i < N; ++i) {
			const int at = threadIdx.x + i * THREADS, t = at / CHUNK, k = at % CHUNK;
			v[i] = t < p.rows && k0 + k < p.width ? p.hidden[t * p.hiddenRow + k0 + k] : 0.f;
		}
	}
	__device__ __forceinline__ void store(float* to) const
	{
#pragma unroll
		for(int i = 0; i < N; ++i) {
			const int at = threadIdx.x + i * THREADS;
			to[at % CHUNK * NT + at / CHUNK] = v[i];
		}
	}
};

template<int NT>
struct Tiles {
	float weights[2][TILE * PITCH];
	float hidden[2][CHUNK * NT];
};

// The logits of the entries entry0 .. entry0 + 63: this thread's entry is threadIdx.x / 4, and all four threads of an entry get them.
template<int NT>
__device__ __forceinline__ void tile_logits(const FewParams& p, Tiles<NT>& s, Staged& staged, StagedHidden<NT>& hidden, int entry0, int next0, float2 (&z)[NT / 2], int& phase)
{
	const int entry = threadIdx.x >> 2, part = threadIdx.x & 3;
#pragma unroll
	for(int t = 0; t < NT / 2; ++t) z[t] = both(0.f);
	for(int k0 = 0; k0 < p.width; k0 += CHUNK, phase ^= 1) {
		staged.store(s.weights[phase]);
		hidden.store(s.hidden[phase]);
		__syncthreads(); // one a chunk: the buffers alternate
		if(k0 + CHUNK < p.width || next0 >= 0) { // under way while this chunk is worked on
			const int k1 = k0 + CHUNK < p.width ? k0 + CHUNK : 0;
			staged.load(p, k1 > 0 ? entry0 : next0, k1);
			hidden.load(p, k1);
		}
		const float* const w = s.weights[phase] + entry * PITCH + part;
		const float* const h = s.hidden[phase] + part * NT;
#pragma unroll
		for(int k = 0; k < CHUNK / 4; ++k) {
			const float2 x = both(w[4 * k]);
#pragma unroll
			for(int t = 0; t < NT / 4; ++t) {
				const float4 y = *reinterpret_cast<const float4*>(h + 4 * k * NT + 4 * t);
				z[2 * t] = fma2(x, make_float2(y.x, y.y), z[2 * t]);
				z[2 * t + 1] = fma2(x, make_float2(y.z, y.w), z[2 * t + 1]);
			}
		}
	}
#pragma unroll
	for(int o = 1; o < 4; o <<= 1) {
#pragma unroll
		for(int t = 0; t < NT / 2; ++t) {
			z[t] = add2(z[t], make_float2(__shfl_xor_sync(0xffffffffu, z[t].x, o), __shfl_xor_sync(0xffffffffu, z[t].y, o)));
		}
	}
}

__device__ __forceinline__ bool has_target(const FewParams& p, int row, int* label)
{
	*label = row < p.rows ? __ldg(p.labels + row) : -1;
	return *label >= 0 && *label < p.vocabulary;
}

__device__ __forceinline__ float2 join(float2 a, float2 b)
{
	const float t = fmaxf(a.x, b.x), at = t == -INFINITY ? 0.f : t;
	return make_float2(t, a.y * exp2_fast(a.x - at) + b.y * exp2_fast(b.x - at));
}

template<int NT>
__global__ void __launch_bounds__(THREADS) few_forward_kernel(const FewParams p)
{
	extern __shared__ __align__(16) uint8_t room[];
	Tiles<NT>& s = *reinterpret_cast<Tiles<NT>*>(room);
	__shared__ float2 joined[WARPS][NT];
	const int begin = blockIdx.x * p.perBlock, end = min(p.vocabulary, begin + p.perBlock);
	const int part = threadIdx.x & 3;
	float2 running[NT / 4]; // of rows 4 i + part
	int label[NT / 4];
#pragma unroll
	for(int i = 0; i < NT / 4; ++i) {
		running[i] = make_float2(-INFINITY, 0.f);
		if(!has_target(p, 4 * i + part, &label[i])) label[i] = -1;
	}
	Staged staged;
	StagedHidden<NT> hidden;
	staged.load(p, begin, 0);
	hidden.load(p, 0);
	int phase = 0;
	for(int entry0 = begin; entry0 < end; entry0 += TILE) {
		float2 z[NT / 2];
		tile_logits<NT>(p, s, staged, hidden, entry0, entry0 + TILE < end ? entry0 + TILE : -1, z, phase);
		const int entry = entry0 + (threadIdx.x >> 2);
		if(entry < end) {
#pragma unroll
			for(int i = 0; i < NT / 4; ++i) {
				const float own = part == 0 ? z[2 * i].x : part == 1 ? z[2 * i].y : part == 2 ? z[2 * i + 1].x : z[2 * i + 1].y;
				if(entry == label[i]) p.labelled[4 * i + part] = own;
				running[i] = join(running[i], make_float2(own * LOG2E, 1.f));
			}
		}
	}
#pragma unroll
	for(int i = 0; i < NT / 4; ++i) {
#pragma unroll
		for(int o = 4; o < 32; o <<= 1) {
			running[i] = join(running[i], make_float2(__shfl_xor_sync(0xffffffffu, running[i].x, o), __shfl_xor_sync(0xffffffffu, running[i].y, o)));
		}
		if((threadIdx.x & 31) < 4) joined[threadIdx.x >> 5][4 * i + part] = running[i];
	}
	__syncthreads();
	const int row = threadIdx.x;
	if(row < p.rows) {
		float2 all = joined[0][row];
		for(int w = 1; w < WARPS; ++w) all = join(all, joined[w][row]);
		p.partial[static_cast<long long>(blockIdx.x) * p.rows + row] = all;
	}
}

template<int NT>
__global__ void __launch_bounds__(THREADS) few_backward_kernel(const FewParams p)
{
	extern __shared__ __align__(16) uint8_t room[];
	Tiles<NT>& s = *reinterpret_cast<Tiles<NT>*>(room);
	float* const dz = reinterpret_cast<float*>(room + sizeof(Tiles<NT>)); // [perBlock][NT]
	const int begin = blockIdx.x * p.perBlock, end = min(p.vocabulary, begin + p.perBlock);
	const int part = threadIdx.x & 3;
	float logSum2[NT / 4], by[NT / 4];
	int label[NT / 4];
#pragma unroll
	for(int i = 0; i < NT / 4; ++i) {
		const bool used = has_target(p, 4 * i + part, &label[i]);
		by[i] = used ? __ldg(p.lossDiff + 4 * i + part) : 0.f;
		logSum2[i] = used ? __ldg(p.logSum + 4 * i + part) * LOG2E : 0.f;
	}
	Staged staged;
	StagedHidden<NT> hidden;
	staged.load(p, begin, 0);
	hidden.load(p, 0);
	int phase = 0;
	for(int entry0 = begin; entry0 < end; entry0 += TILE) {
		float2 z[NT / 2];
		tile_logits<NT>(p, s, staged, hidden, entry0, entry0 + TILE < end ? entry0 + TILE : -1, z, phase);
		const int entry = entry0 + (threadIdx.x >> 2);
#pragma unroll
		for(int i = 0; i < NT / 4; ++i) {
			const float own = part == 0 ? z[2 * i].x : part == 1 ? z[2 * i].y : part == 2 ? z[2 * i + 1].x : z[2 * i + 1].y;
			// a row without a target has no gradient, whatever its logits
			const float q = exp2_fast(fmaf(own, LOG2E, -logSum2[i])) - (entry == label[i] ? 1.f : 0.f);
			if(entry < end) dz[(entry - begin) * NT + 4 * i + part] = by[i] == 0.f ? 0.f : by[i] * q;
		}
	}
	__syncthreads();
	const float* const weights = p.weights + static_cast<long long>(begin) * p.weightsRow;
	float* const out = p.weightsDiff == nullptr ? nullptr : p.weightsDiff + static_cast<long long>(begin) * p.weightsDiffRow;
	const int count = end - begin;
	for(int c = threadIdx.x; c < p.width; c += THREADS) {
		float2 h[NT / 2], dx[NT / 2]; // pairs of rows
#pragma unroll
		for(int t = 0; t < NT; ++t) {
			int unused;
			const float v = has_target(p, t, &unused) && !(__ldg(p.lossDiff + t) == 0.f) ? p.hidden[t * p.hiddenRow + c] : 0.f;
			(t % 2 == 0 ? h[t / 2].x : h[t / 2].y) = v;
			dx[t / 2] = both(0.f);
		}
		constexpr int AHEAD = 8;
		for(int e0 = 0; e0 < count; e0 += AHEAD) {
			float w[AHEAD];
#pragma unroll
			for(int k = 0; k < AHEAD; ++k) w[k] = p.hiddenPart != nullptr && e0 + k < count ? weights[static_cast<long long>(e0 + k) * p.weightsRow + c] : 0.f;
#pragma unroll
			for(int k = 0; k < AHEAD; ++k) {
				if(e0 + k >= count) break;
				float2 sums = both(0.f);
				const float2 x = both(w[k]);
#pragma unroll
				for(int t = 0; t < NT / 4; ++t) {
					const float4 d = *reinterpret_cast<const float4*>(dz + (e0 + k) * NT + 4 * t);
					const float2 d0 = make_float2(d.x, d.y), d1 = make_float2(d.z, d.w);
					sums = fma2(d1, h[2 * t + 1], fma2(d0, h[2 * t], sums));
					dx[2 * t] = fma2(d0, x, dx[2 * t]);
					dx[2 * t + 1] = fma2(d1, x, dx[2 * t + 1]);
				}
				if(out != nullptr) out[static_cast<long long>(e0 + k) * p.weightsDiffRow + c] = sums.x + sums.y;
			}
		}
		if(p.hiddenPart != nullptr) {
			float* const mine = p.hiddenPart + static_cast<long long>(blockIdx.x) * p.rows * p.width + c;
#pragma unroll
			for(int t = 0; t < NT; ++t) {
				if(t < p.rows) mine[static_cast<long long>(t) * p.width] = t % 2 == 0 ? dx[t / 2].x : dx[t / 2].y;
			}
		}
	}
}

// hidden_diff from the blocks' parts, added in order: 32 columns of a row per block, eight threads a column take every eighth part.
__global__ void __launch_bounds__(256) few_hidden_kernel(const FewParams p, int parts, float* __restrict__ out, long long outRow)
{
	__shared__ float sums[8][32];
	dependent_wait();
	const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
	const int c = blockIdx.x * 32 + lane, t = blockIdx.y;
	float s = 0.f;
	if(c < p.width) {
		const float* const at = p.hiddenPart + static_cast<long long>(t) * p.width + c;
		constexpr int AHEAD = 8;
		for(int i = group; i < parts; i += 8 * AHEAD) {
			float v[AHEAD];
#pragma unroll
			for(int k = 0; k < AHEAD; ++k) v[k] = i + 8 * k < parts ? at[static_cast<long long>(i + 8 * k) * p.rows * p.width] : 0.f;
#pragma unroll
			for(int k = 0; k < AHEAD; ++k) s += v[k];
		}
	}
	sums[group][lane] = s;
	__syncthreads();
	if(group != 0 || c >= p.width) return;
	s = 0.f;
#pragma unroll
	for(int g = 0; g < 8; ++g) s += sums[g][lane];
	out[t * outRow + c] = s;
}

// ---- nine to 32 rows, forward --------------------------------------------------------------------------------------------
// A tile is 128 entries and all the rows.  A warp has eight rows and every KS-th stretch of the elements, a lane four entries 32 apart:
// 32 sums, each of an even and an odd half that one paired multiply-add serves.  Four elements take four 16-byte loads of weights, eight of
// rows (which all lanes share) and 64 paired multiply-adds.  Chunks of 32 elements come by asynchronous copies, two ahead, V elements
// each; 36 words from row to row keep 16-byte loads free of conflicts.  The KS warps' sums meet in shared memory, each warp ends some of the rows.
//   One block per SM: 16 x 4096 rows over 50257 entries 306 us (2.7 TB/s; by planes 667), 16 x 1024 over 32000 58 us (110), 32 x 1024 84 (111);
// with two blocks per SM 407, 61 and 87.  Widths that are odd come by 4-byte copies: 16 x 1861 over 66524 307 us, 1862 222 (419 by planes).
constexpr int GROUP_ROWS = 8, GROUP_TILE = 128, GROUP_CHUNK = 32, GROUP_PITCH = GROUP_CHUNK + 4, GROUP_STAGES = 3;

template<int G, int KS>
struct GroupRoom {
	struct {
		float weights[GROUP_TILE * GROUP_PITCH];
		float hidden[GROUP_ROWS * G * GROUP_PITCH];
	} stages[GROUP_STAGES];
	float logits[KS][GROUP_ROWS * G][GROUP_TILE];
};

template<int V>
__device__ __forceinline__ void copy_words(float* to, const float* from, bool there) // zeros where it is not
{
	if constexpr(V < 4) asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(there ? 4 * V : 0), "n"(4 * V) : "memory");
	else asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}

template<int G, int KS, int V>
__global__ void __launch_bounds__(G * KS * 32) group_forward_kernel(const FewParams p)
{
	extern __shared__ __align__(16) uint8_t room[];
	GroupRoom<G, KS>& s = *reinterpret_cast<GroupRoom<G, KS>*>(room);
	constexpr int WARPS_ALL = G * KS, OWN = GROUP_ROWS / KS; // rows that a warp ends
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	const int group = warp % G, part = warp / G;
	const int own0 = group * GROUP_ROWS + part * OWN;
	const int begin = blockIdx.x * p.perBlock, end = min(p.vocabulary, begin + p.perBlock);
	int label[OWN]; // -1: not in these rows
#pragma unroll
	for(int r = 0; r < OWN; ++r) {
		if(!has_target(p, own0 + r, &label[r])) label[r] = -1;
	}
	// the chunk that is asked for next, and its stage
	int nextEntry = begin, nextK = 0, nextStage = 0;
	auto load = [&] {
		if(nextEntry < end) {
			constexpr int PER_ROW = GROUP_CHUNK / V, AT_ONCE = 32 / PER_ROW; // lanes of an entry, entries of a warp's copy
			const int k = nextK + lane % PER_ROW * V;
			const bool in = k < p.width; // the width is a multiple of V
			float* const weights = s.stages[nextStage].weights + lane % PER_ROW * V;
#pragma unroll 4
			for(int e = warp * AT_ONCE + lane / PER_ROW; e < GROUP_TILE; e += WARPS_ALL * AT_ONCE) {
				const bool there = in && nextEntry + e < p.vocabulary;
				copy_words<V>(weights + e * GROUP_PITCH, there ? p.weights + static_cast<long long>(nextEntry + e) * p.weightsRow + k : p.weights, there);
			}
			float* const hidden = s.stages[nextStage].hidden + lane;
#pragma unroll
			for(int i = 0; i < OWN; ++i) {
				const bool there = nextK + lane < p.width && own0 + i < p.rows;
				copy_words<1>(hidden + (own0 + i) * GROUP_PITCH, there ? p.hidden + (own0 + i) * p.hiddenRow + nextK + lane : p.hidden, there);
			}
			nextK += GROUP_CHUNK;
			if(nextK >= p.width) {
				nextK = 0;
				nextEntry += GROUP_TILE;
			}
			nextStage = nextStage + 1 == GROUP_STAGES ? 0 : nextStage + 1;
		}
		asm volatile("cp.async.commit_group;" ::: "memory"); // an empty one counts too
	};
	float2 running[OWN];
#pragma unroll
	for(int r = 0; r < OWN; ++r) running[r] = make_float2(-INFINITY, 0.f);
	for(int i = 0; i < GROUP_STAGES - 1; ++i) load();
	int stage = 0;
	for(int entry0 = begin; entry0 < end; entry0 += GROUP_TILE) {
		float2 z[4][GROUP_ROWS];
#pragma unroll
		for(int j = 0; j < 4; ++j) {
#pragma unroll
			for(int r = 0; r < GROUP_ROWS; ++r) z[j][r] = both(0.f);
		}
		for(int k0 = 0; k0 < p.width; k0 += GROUP_CHUNK) {
			asm volatile("cp.async.wait_group %0;" ::"n"(GROUP_STAGES - 2) : "memory");
			__syncthreads(); // this chunk is there, and everyone is done with the one before, whose stage is asked for again
			load();
			const float* const w = s.stages[stage].weights + lane * GROUP_PITCH + part * (GROUP_CHUNK / KS);
			const float* const h = s.stages[stage].hidden + group * GROUP_ROWS * GROUP_PITCH + part * (GROUP_CHUNK / KS);
			stage = stage + 1 == GROUP_STAGES ? 0 : stage + 1;
#pragma unroll 2
			for(int k = 0; k < GROUP_CHUNK / KS; k += 4) {
				float4 x[4];
#pragma unroll
				for(int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const float4*>(w + 32 * j * GROUP_PITCH + k);
#pragma unroll
				for(int r = 0; r < GROUP_ROWS; ++r) {
					const float4 y = *reinterpret_cast<const float4*>(h + r * GROUP_PITCH + k);
#pragma unroll
					for(int j = 0; j < 4; ++j) {
						z[j][r] = fma2(make_float2(x[j].x, x[j].y), make_float2(y.x, y.y), z[j][r]);
						z[j][r] = fma2(make_float2(x[j].z, x[j].w), make_float2(y.z, y.w), z[j][r]);
					}
				}
			}
		}
		// (the logits of the tile before were read in front of the chunks' barriers)
#pragma unroll
		for(int j = 0; j < 4; ++j) {
#pragma unroll
			for(int r = 0; r < GROUP_ROWS; ++r) s.logits[part][group * GROUP_ROWS + r][lane + 32 * j] = z[j][r].x + z[j][r].y;
		}
		__syncthreads();
#pragma unroll
		for(int r = 0; r < OWN; ++r) {
			float v[4], top = running[r].x;
#pragma unroll
			for(int j = 0; j < 4; ++j) {
				const int entry = entry0 + lane + 32 * j;
				float value = s.logits[0][own0 + r][lane + 32 * j];
#pragma unroll
				for(int k = 1; k < KS; ++k) value += s.logits[k][own0 + r][lane + 32 * j];
				if(entry == label[r]) p.labelled[own0 + r] = value;
				v[j] = entry < end ? value * LOG2E : -INFINITY;
				top = fmaxf(top, v[j]);
			}
			const float at = top == -INFINITY ? 0.f : top;
			running[r].y *= exp2_fast(running[r].x - at);
#pragma unroll
			for(int j = 0; j < 4; ++j) running[r].y += exp2_fast(v[j] - at);
			running[r].x = top;
		}
	}
#pragma unroll
	for(int r = 0; r < OWN; ++r) {
#pragma unroll
		for(int o = 16; o > 0; o >>= 1) {
			running[r] = join(running[r], make_float2(__shfl_xor_sync(0xffffffffu, running[r].x, o), __shfl_xor_sync(0xffffffffu, running[r].y, o)));
		}
		if(lane == 0 && own0 + r < p.rows) p.partial[static_cast<long long>(blockIdx.x) * p.rows + own0 + r] = running[r];
	}
}

template<int G, int KS>
void launch_group(const FewParams& p, cudaStream_t stream)
{
	constexpr int BYTES = static_cast<int>(sizeof(GroupRoom<G, KS>));
	const bool quads = p.width % 4 == 0 && p.weightsRow % 4 == 0 && aligned16(p.weights);
	const bool pairs = p.width % 2 == 0 && p.weightsRow % 2 == 0 && (reinterpret_cast<uintptr_t>(p.weights) & 7u) == 0;
	const auto kernel = quads ? group_forward_kernel<G, KS, 4> : pairs ? group_forward_kernel<G, KS, 2> : group_forward_kernel<G, KS, 1>;
	cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
	kernel<<<few_blocks(p.rows, p.vocabulary), G * KS * 32, BYTES, stream>>>(p);
	count_launch();
}

template<int NT>
void launch_forward(const FewParams& p, cudaStream_t stream)
{
	few_forward_kernel<NT><<<few_blocks(p.rows, p.vocabulary), THREADS, sizeof(Tiles<NT>), stream>>>(p);
	count_launch();
}

template<int NT>
void launch_backward(const FewParams& p, cudaStream_t stream)
{
	constexpr size_t each = NT * sizeof(float), most = sizeof(Tiles<NT>) + FEW_MOST_ENTRIES * each;
	cudaFuncSetAttribute(few_backward_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
	few_backward_kernel<NT><<<few_blocks(p.rows, p.vocabulary), THREADS, sizeof(Tiles<NT>) + p.perBlock * each, stream>>>(p);
	count_launch();
}

static_assert(sizeof(Tiles<8>) <= 48 * 1024, "more shared memory than a kernel may have without asking");

} // namespace

int few_forward(const FewParams& p, cudaStream_t stream)
{
	if(p.rows <= 4) launch_forward<4>(p, stream);
	else if(p.rows <= 8) launch_forward<8>(p, stream);
	else if(p.rows <= 16) launch_group<2, 4>(p, stream);
	else if(p.rows <= 24) launch_group<3, 4>(p, stream);
	else launch_group<4, 2>(p, stream);
	return check_launch();
}

int few_backward(const FewParams& p, float* hiddenDiff, long long hiddenDiffRow, cudaStream_t stream)
{
	if(p.rows <= 4) launch_backward<4>(p, stream);
	else launch_backward<8>(p, stream);
	if(hiddenDiff != nullptr) {
		launch_dependent(true, few_hidden_kernel, dim3((p.width + 31) / 32, p.rows), dim3(256), 0, stream, p, few_blocks(p.rows, p.vocabulary), hiddenDiff,
			hiddenDiffRow);
		count_launch();
	}
	return check_launch();
}

// Blocks of a stretch each: four on an SM (one of more than eight rows), or as many more as keep a stretch's dz within a
// block's shared memory; whole tiles.
int few_entries(int rows, int vocabulary)
{
	const int tile = rows > FEW_ROWS ? GROUP_TILE : TILE, tiles = (vocabulary + tile - 1) / tile, wanted = sm_count() * (rows > FEW_ROWS ? 1 : 4);
	const int perBlock = (tiles + wanted - 1) / wanted * tile;
	return rows <= FEW_ROWS && perBlock > FEW_MOST_ENTRIES ? FEW_MOST_ENTRIES : perBlock;
}
int few_blocks(int rows, int vocabulary)
{
	const int perBlock = few_entries(rows, vocabulary);
	return (vocabulary + perBlock - 1) / perBlock;
}

} // namespace nb200
