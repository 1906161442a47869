// Softmax cross entropy of hidden rows against a vocabulary's weights, forward and backward, without keeping the logits.
//
//   z = hidden weights^T,  log_sum = log sum_j exp z_j,  loss = log_sum - z_label
//   dz = loss_diff (softmax(z) - [j = label]),  hidden_diff = dz weights,  weights_diff = dz^T hidden
//
// 16-bit types: the forward pass is one product whose epilogue reduces each row's 128 columns to a maximum and a sum, so that
// 8 bytes per row leave the SM for 128 logits (product16.cu).  The backward pass forms the logits anew, piece by piece of the vocabulary: a product
// whose epilogue turns them into dz, and the two products that consume it.  Bound by the tensor core: 8 rows vocabulary
// width multiply-adds in all for forward and backward, where keeping the logits would take 6 and rows x vocabulary memory.
//   dz is kept in the operands' type for those products: the tensor core multiplies like types, and two planes of dz would make six
//   products of four.  It is rounded over the largest |loss_diff|, so that one loss_diff for all rows (a mean's 1 / rows) costs nothing: rounded
//   with it, the labels' elements, which are almost -loss_diff, would all be off alike (1 / 921 in bf16: both gradients 2.2e-3 too small).
//   What is left is half a step per element of the softmax, in no common direction, and a label's p where p - 1 rounds to -1; rows whose
//   loss_diff is another are off by up to half a step each.  Gradients of 4096 x 1024 rows over 50257 entries differ in 5e-4 from those of
//   fp32 dz rounded the same way, 1.66e-3 being that rounding.  In fp16 dz is times 2^14, because softmax values of 1e-7 are below what a
//   half holds; dz between 1 and 2^-38 of the largest then keeps some or all of its bits.  hidden_diff is summed in fp32 over the pieces.
// fp32: the same with three bf16 planes of each operand (product16.cuh), a piece of the weights split at a time: six times the
// multiply-adds, and results as exact as fp32 sums in order give them.  Few rows of fp32: vocabulary_few.cu.
#include "product16.cuh"
#include "vocabulary_few.cuh"

#include <cuda.h>

namespace nb200 {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr long long DIFF_BYTES = 256ll << 20, PIECE_BYTES = 1ll << 30;

__device__ __forceinline__ bool has_target(const int* labels, int row, int vocabulary)
{
	const int label = __ldg(labels + row);
	return label >= 0 && label < vocabulary;
}

// ---- 16-bit types ---------------------------------------------------------------------------------------------------

// Eight 16-bit elements from any address: 32-bit words around them, shifted by half a word where they begin inside one.
__device__ __forceinline__ uint4 gather8(const uint16_t* p)
{
	const uintptr_t a = reinterpret_cast<uintptr_t>(p);
	if((a & 15u) == 0) return *reinterpret_cast<const uint4*>(p);
	const uint32_t* const w = reinterpret_cast<const uint32_t*>(a & ~static_cast<uintptr_t>(3));
	if((a & 3u) == 0) return make_uint4(w[0], w[1], w[2], w[3]);
	const uint32_t v[5] = { w[0], w[1], w[2], w[3], w[4] };
	return make_uint4(__funnelshift_r(v[0], v[1], 16), __funnelshift_r(v[1], v[2], 16), __funnelshift_r(v[2], v[3], 16), __funnelshift_r(v[3], v[4], 16));
}

// Row and unit of a flat index.
__device__ __forceinline__ void row_unit(long long i, int perRow, int* row, int* unit)
{
	const int r = i <= 0xffffffffll ? static_cast<int>(static_cast<uint32_t>(i) / static_cast<uint32_t>(perRow)) : static_cast<int>(i / perRow);
	*row = r;
	*unit = static_cast<int>(i - static_cast<long long>(r) * perRow);
}

// What dz is over and times (the head of this file), and what undoes both: one block.
constexpr int SCALE_THREADS = 1024;
__global__ void __launch_bounds__(SCALE_THREADS) diff_scale_kernel(int rows, const int* __restrict__ labels, const float* __restrict__ lossDiff,
	int vocabulary, float* scale, int type)
{
	__shared__ float slots[SCALE_THREADS / 32];
	dependent_wait();
	float most = 0.f;
	if(type != NB200_TYPE_FP32) {
#pragma unroll 8
		for(int r = threadIdx.x; r < rows; r += SCALE_THREADS) {
			const float diff = fabsf(__ldg(lossDiff + r));
			most = fmaxf(most, has_target(labels, r, vocabulary) ? diff : 0.f);
		}
	}
	most = warp_max_all(most);
	if((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = most;
	__syncthreads();
	if(threadIdx.x == 0) {
		for(int i = 1; i < SCALE_THREADS / 32; ++i) most = fmaxf(most, slots[i]);
		if(!(most > 0.f && most < INFINITY)) most = 1.f;
		const float by = type == NB200_TYPE_FP16 ? 16384.f : 1.f;
		scale[0] = most;
		scale[1] = by;
		scale[2] = most / by;
	}
}

// Rows of 16-bit elements copied to aligned rows of dstRow (a multiple of 8) elements, zeros behind the width.  With labels: a row without a
// target or with a loss_diff of zero becomes zeros -- it has no gradient, whatever it holds.
__global__ void __launch_bounds__(256) copy_rows16_kernel(const uint16_t* __restrict__ src, long long srcRow, int rows, int width,
	uint16_t* __restrict__ dst, int dstRow, const int* __restrict__ labels, const float* __restrict__ lossDiff, int vocabulary)
{
	dependent_wait();
	const int perRow = dstRow / 8;
	const long long total = static_cast<long long>(rows) * perRow;
	for(long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * blockDim.x) {
		int r, u;
		row_unit(i, perRow, &r, &u);
		const uint16_t* const from = src + r * srcRow + u * 8;
		uint4 v = make_uint4(0u, 0u, 0u, 0u);
		if(labels == nullptr || (has_target(labels, r, vocabulary) && !(lossDiff[r] == 0.f))) {
			// a word around the first or the last element of all may reach outside
			const bool inside = u * 8 + 8 <= width && (i != 0 || (reinterpret_cast<uintptr_t>(from) & 3u) == 0) && (r != rows - 1 || u * 8 + 8 < width);
			if(inside || (u * 8 + 8 <= width && (reinterpret_cast<uintptr_t>(from) & 3u) == 0)) {
				v = gather8(from);
			} else {
				uint32_t e[8];
#pragma unroll
				for(int j = 0; j < 8; ++j) e[j] = u * 8 + j < width ? from[j] : 0u;
				v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
			}
		}
		*reinterpret_cast<uint4*>(dst + static_cast<long long>(r) * dstRow + u * 8) = v;
	}
}

// The way back: aligned rows of srcRow > width elements to rows that begin anywhere.
__global__ void __launch_bounds__(256) spread_rows16_kernel(const uint16_t* __restrict__ src, int srcRow, int rows, int width, uint16_t* __restrict__ dst,
	long long dstRow)
{
	dependent_wait();
	const int perRow = (width + 14) / 8;
	const long long total = static_cast<long long>(rows) * perRow;
	for(long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * blockDim.x) {
		int r, u;
		row_unit(i, perRow, &r, &u);
		uint16_t* const to = dst + r * dstRow;
		const int first = u * 8 - static_cast<int>((reinterpret_cast<uintptr_t>(to) & 15u) / 2);
		const uint16_t* const from = src + static_cast<long long>(r) * srcRow;
		if(first >= 0 && first + 8 <= width) {
			*reinterpret_cast<uint4*>(to + first) = gather8(from + first);
		} else {
			for(int j = first < 0 ? 0 : first; j < first + 8 && j < width; ++j) to[j] = from[j];
		}
	}
}

// Joins the partial sums of a row.  32 rows per block, 32 threads a row: 250 parts of 48 rows took 13 us with eight.
//   The loss is formed of the labelled logit's distance from the maximum rather than as log_sum less the logit, whose common size would
// leave its rounding (8e-6 at 100) in a loss of any size.  The distance is in units of log 2, as the exponents were: `products` rounded
// (vocabulary_few.cu), or with the multiply-add that the exponents came from.
constexpr int JOIN_WARPS = 32;
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_partials_kernel(const float2* __restrict__ partial, int parts, int rows,
	const float* __restrict__ labelled, const int* __restrict__ labels, int vocabulary, int products, float* __restrict__ loss,
	float* __restrict__ logSum)
{
	__shared__ float2 slots[JOIN_WARPS][33];
	dependent_wait();
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	const int row = blockIdx.x * 32 + lane;
	auto join = [](float2 a, float2 b) {
		const float t = fmaxf(a.x, b.x), at = t == -INFINITY ? 0.f : t;
		return make_float2(t, a.y * exp2f(a.x - at) + b.y * exp2f(b.x - at));
	};
	float2 mine = make_float2(-INFINITY, 0.f);
	constexpr int AHEAD = 4;
	for(int i = warp; i < parts; i += JOIN_WARPS * AHEAD) {
		float2 next[AHEAD];
#pragma unroll
		for(int k = 0; k < AHEAD; ++k) {
			next[k] = make_float2(-INFINITY, 0.f);
			if(row < rows && i + k * JOIN_WARPS < parts) next[k] = partial[static_cast<long long>(i + k * JOIN_WARPS) * rows + row];
		}
		mine = join(mine, join(join(next[0], next[1]), join(next[2], next[3])));
	}
	slots[warp][lane] = mine;
	__syncthreads();
	// a warp per row now
	mine = slots[lane][warp];
#pragma unroll
	for(int o = 16; o > 0; o >>= 1) {
		mine = join(mine, make_float2(__shfl_xor_sync(0xffffffffu, mine.x, o), __shfl_xor_sync(0xffffffffu, mine.y, o)));
	}
	const int own = blockIdx.x * 32 + warp;
	if(lane == 0 && own < rows) {
		const float rest = logf(mine.y);
		logSum[own] = mine.x / LOG2E + rest;
		float value = 0.f;
		if(has_target(labels, own, vocabulary)) {
			const float z = labelled[own];
			value = rest - (products ? __fadd_rn(__fmul_rn(z, LOG2E), -mine.x) : fmaf(z, LOG2E, -mine.x)) / LOG2E;
		}
		loss[own] = value;
	}
}

// out[row][col] = sum of the planes times *by: `group` neighbouring threads (1 or 8) share four columns, each adds every group-th plane in
// order, and their sums meet in a tree.
template<typename T>
__global__ void __launch_bounds__(256) sum_planes_kernel(const float* __restrict__ planes, int count, long long planeSize, long long ldPlane,
	int rows, int width, int group, const float* __restrict__ by, T* __restrict__ out, long long outRow)
{
	dependent_wait();
	const float scale = __ldg(by);
	const int member = threadIdx.x & (group - 1);
	const int quads = (width + 3) / 4;
	const bool vector = (outRow & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7u) == 0;
	const long long total = static_cast<long long>(rows) * quads;
	const long long step = static_cast<long long>(gridDim.x) * blockDim.x / group;
	for(long long i = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / group; i < total; i += step) {
		const long long row = i / quads;
		const int col = static_cast<int>(i - row * quads) * 4;
		float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
		constexpr int AHEAD = 8;
		for(int k = member; k < count; k += AHEAD * group) {
			float4 w[AHEAD];
#pragma unroll
			for(int j = 0; j < AHEAD; ++j) {
				w[j] = make_float4(0.f, 0.f, 0.f, 0.f);
				if(k + j * group < count) w[j] = *reinterpret_cast<const float4*>(planes + (k + j * group) * planeSize + row * ldPlane + col);
			}
#pragma unroll
			for(int j = 0; j < AHEAD; ++j) {
				v.x += w[j].x; v.y += w[j].y; v.z += w[j].z; v.w += w[j].w;
			}
		}
		if(group > 1) {
			const unsigned mask = 0xffu << (threadIdx.x & 24u); // the eight of them
#pragma unroll
			for(int o = 4; o > 0; o >>= 1) {
				v.x += __shfl_xor_sync(mask, v.x, o);
				v.y += __shfl_xor_sync(mask, v.y, o);
				v.z += __shfl_xor_sync(mask, v.z, o);
				v.w += __shfl_xor_sync(mask, v.w, o);
			}
			if(member != 0) continue;
		}
		T* const to = out + row * outRow + col;
		if constexpr(sizeof(T) == 4) {
			const float f[4] = { v.x * scale, v.y * scale, v.z * scale, v.w * scale };
			if((outRow & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0 && col + 4 <= width) {
				*reinterpret_cast<float4*>(to) = make_float4(f[0], f[1], f[2], f[3]);
			} else {
				for(int j = 0; j < 4 && col + j < width; ++j) to[j] = f[j];
			}
		} else if(vector && col + 4 <= width) {
			*reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(v.x * scale, v.y * scale), pack2<T>(v.z * scale, v.w * scale));
		} else {
			const float f[4] = { v.x, v.y, v.z, v.w };
			for(int j = 0; j < 4 && col + j < width; ++j) to[j] = from_float<T>(f[j] * scale);
		}
	}
}

// Rows of fp32 elements as three bf16 planes that add up to them.  Labels and lossDiff as above.
__global__ void __launch_bounds__(256) split_rows_kernel(const float* __restrict__ src, long long srcRow, int rows, int width,
	__nv_bfloat16* __restrict__ dst, int dstRow, long long plane, const int* __restrict__ labels, const float* __restrict__ lossDiff, int vocabulary)
{
	dependent_wait();
	const int perRow = dstRow / 8;
	const long long total = static_cast<long long>(rows) * perRow;
	const bool vector = (srcRow & 3) == 0 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
	for(long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * blockDim.x) {
		int r, u;
		row_unit(i, perRow, &r, &u);
		const float* const from = src + r * srcRow + u * 8;
		float v[8];
#pragma unroll
		for(int j = 0; j < 8; ++j) v[j] = 0.f;
		if(labels == nullptr || (has_target(labels, r, vocabulary) && !(lossDiff[r] == 0.f))) {
			if(vector && u * 8 + 8 <= width) {
				Unit16<float>::unpack(reinterpret_cast<const uint4*>(from)[0], v);
				Unit16<float>::unpack(reinterpret_cast<const uint4*>(from)[1], v + 4);
			} else {
#pragma unroll
				for(int j = 0; j < 8; ++j) v[j] = u * 8 + j < width ? from[j] : 0.f;
			}
		}
		__nv_bfloat16* const to = dst + static_cast<long long>(r) * dstRow + u * 8;
#pragma unroll
		for(int k = 0; k < 3; ++k) {
			uint32_t w[4];
#pragma unroll
			for(int j = 0; j < 4; ++j) {
				w[j] = pack2<__nv_bfloat16>(v[2 * j], v[2 * j + 1]);
				const float2 taken = unpack2<__nv_bfloat16>(w[j]); // (an infinite or undefined element stays one in every plane)
				v[2 * j] -= taken.x;
				v[2 * j + 1] -= taken.y;
			}
			*reinterpret_cast<uint4*>(to + k * plane) = make_uint4(w[0], w[1], w[2], w[3]);
		}
	}
}

__global__ void __launch_bounds__(256) zero_rows_kernel(uint8_t* p, long long rowBytes, long long widthBytes, int rows)
{
	for(long long r = blockIdx.x; r < rows; r += gridDim.x) {
		for(long long i = threadIdx.x; i < widthBytes; i += blockDim.x) p[r * rowBytes + i] = 0;
	}
}

// ---- scratch memory ---------------------------------------------------------------------------------------------------

struct Problem {
	int type, rows, width, vocabulary;
	const void *hidden, *weights;
	long long hiddenRow, weightsRow;
};

// Hands out pieces of the scratch memory, or only counts them.
struct Room {
	uint8_t* base;
	size_t used = 0;
	template<typename T>
	T* take(size_t count)
	{
		T* const p = reinterpret_cast<T*>(base + used);
		used += (count * sizeof(T) + 255) / 256 * 256;
		return p;
	}
};

int round_up(long long v, int to) { return static_cast<int>((v + to - 1) / to * to); }

bool rows_for_tma(const void* p, long long row) { return aligned16(p) && row % 8 == 0; }

// Rows of weights_diff that do not begin on 16-byte boundaries: a tile's threads, which have a row each, would store element by element
// (gradient of 5000 x 1030 fp16 weights by 1000 rows: 177 us).  16-bit ones go to aligned rows first, fp32 ones to the planes that
// parts of K are added up from.
bool odd_rows(const Problem& q) { return q.width % (q.type == NB200_TYPE_FP32 ? 4 : 8) != 0; }

// Columns of the vocabulary that are handled at a time: dz of a piece takes at most DIFF_BYTES; the planes of its weights (fp32) and the
// aligned rows of odd_rows() take at most PIECE_BYTES each, which leaves a tile per SM for 128 rows of 4096 elements (with a
// quarter of it, 75 x 4043 rows over 35434 entries ran on 35 of 148 SMs).  The 16-bit forward pass needs none of them.
int piece_of(const Problem& q, bool backward)
{
	const bool fp32 = q.type == NB200_TYPE_FP32;
	const long long whole = round_up(q.vocabulary, PRODUCT16_N), ld = round_up(q.width, 8);
	long long piece = whole;
	auto limit = [&](long long bytes, long long perColumn) {
		if(perColumn > 0 && bytes / perColumn < piece) piece = bytes / perColumn;
	};
	if(fp32) limit(PIECE_BYTES, 6 * ld);
	if(backward) {
		limit(DIFF_BYTES, (fp32 ? 6ll : 2ll) * q.rows);
		if(odd_rows(q)) limit(PIECE_BYTES, type_size(q.type) * ld);
	}
	if(piece >= whole) return static_cast<int>(whole);
	piece = piece / PRODUCT16_N * PRODUCT16_N;
	if(piece < PRODUCT16_N) piece = PRODUCT16_N;
	const long long pieces = (whole + piece - 1) / piece;   // of equal size
	return round_up((whole + pieces - 1) / pieces, PRODUCT16_N);
}

// Parts of K where a product has few tiles: enough for one tile per SM, none shorter than 8 steps of 64.  (26 x 207 fp32 by 78703: 34 us in 148
// parts, 52 in 64.)
int splits_of(long long tiles, int kBlocks)
{
	const int sms = sm_count();
	if(tiles * 2 > sms) return 1;
	long long splits = sms / tiles;
	if(splits > kBlocks / 8) splits = kBlocks / 8;
	return splits < 1 ? 1 : static_cast<int>(splits);
}

// Tiles of 64 columns for the products with the weights' rows where all of them find an SM at once: a step of such a tile takes two thirds
// of one of 256 columns (59 x 3596 fp32 rows over 6319 entries, 99 tiles: 76 us against 137 with 25; 11 x 334 over 16431, 257 tiles in two
// rounds: 36 us against 23 with 65).
bool narrow(const Problem& q, int piece)
{
	const long long columns = q.vocabulary < piece ? q.vocabulary : piece;
	return static_cast<long long>((q.rows + PRODUCT16_M - 1) / PRODUCT16_M) * ((columns + PRODUCT16_NARROW - 1) / PRODUCT16_NARROW) <= sm_count();
}
int tile_columns(bool narrow) { return narrow ? PRODUCT16_NARROW : PRODUCT16_N; }

// An operand as TMA takes it: where it lies, and how far its rows and planes are apart.
struct Aligned {
	const void* p;
	long long row, plane;
};

// Few rows of fp32 go to kernels of their own, whose blocks have stretches of the vocabulary: up to eight where it is not shorter than the
// rows (6 x 4007 rows over 119 entries, two blocks: 240 us), more, forward only, where half of the SMs have a stretch (16 x 2048 rows over
// 12000 entries 58 us, by planes 116; 24 x 3596 over 6319 118 and 113, 9 x 1031 over 8000 49 and 43).
bool few_rows(const Problem& q, bool backward)
{
	if(q.type != NB200_TYPE_FP32) return false;
	if(q.rows <= FEW_ROWS) return q.vocabulary >= q.width;
	return !backward && q.rows <= FEW_FORWARD_ROWS && q.vocabulary >= 64 * sm_count();
}

struct FewRoom {
	float2* partial;
	float *labelled, *hiddenPart;
	FewRoom(const Problem& q, bool backward, Room& room)
	{
		const size_t blocks = few_blocks(q.rows, q.vocabulary);
		partial = backward ? nullptr : room.take<float2>(blocks * q.rows);
		labelled = backward ? nullptr : room.take<float>(q.rows);
		hiddenPart = backward ? room.take<float>(blocks * q.rows * q.width) : nullptr;
	}
};

struct Forward {
	int piece, tileColumns, parts; // parts: of a row's sums
	float2* partial;
	float* labelled;
	uint16_t *hidden, *weights; // copies in aligned rows, or planes; null: as they are
	Forward(const Problem& q, Room& room)
	{
		const bool fp32 = q.type == NB200_TYPE_FP32;
		const size_t ld = round_up(q.width, 8);
		piece = piece_of(q, false);
		tileColumns = tile_columns(narrow(q, piece));
		parts = (q.vocabulary + tileColumns - 1) / tileColumns * 2;
		partial = room.take<float2>(static_cast<size_t>(parts) * q.rows);
		labelled = room.take<float>(q.rows);
		hidden = fp32 ? room.take<uint16_t>(3 * q.rows * ld) : rows_for_tma(q.hidden, q.hiddenRow) ? nullptr : room.take<uint16_t>(q.rows * ld);
		weights = fp32 ? room.take<uint16_t>(3 * piece * ld) : rows_for_tma(q.weights, q.weightsRow) ? nullptr : room.take<uint16_t>(q.vocabulary * ld);
	}
};

struct Backward {
	int piece, tileColumns, hiddenSplits, weightsSplits;
	float* scale;
	uint16_t *hidden, *weights, *diff;
	float *hiddenPlanes, *weightsPlanes;
	uint16_t* weightsRows; // weights_diff in aligned rows; null: straight to the caller
	Backward(const Problem& q, Room& room)
	{
		const bool fp32 = q.type == NB200_TYPE_FP32;
		const size_t ld = round_up(q.width, 8), planes = fp32 ? 3 : 1;
		piece = piece_of(q, true);
		tileColumns = tile_columns(narrow(q, piece));
		const long long mTiles = (q.rows + PRODUCT16_M - 1) / PRODUCT16_M, dTiles = (q.width + PRODUCT16_N - 1) / PRODUCT16_N;
		hiddenSplits = splits_of(mTiles * dTiles, piece / PRODUCT16_K);
		// its result goes straight to the caller where K is not split
		weightsSplits = splits_of(piece / PRODUCT16_M * dTiles, (q.rows + PRODUCT16_K - 1) / PRODUCT16_K);
		scale = room.take<float>(3);
		hidden = room.take<uint16_t>(planes * q.rows * ld);
		weights = fp32 ? room.take<uint16_t>(3 * piece * ld) : rows_for_tma(q.weights, q.weightsRow) ? nullptr : room.take<uint16_t>(q.vocabulary * ld);
		diff = room.take<uint16_t>(planes * q.rows * piece);
		hiddenPlanes = room.take<float>(static_cast<size_t>(hiddenSplits) * q.rows * ld);
		weightsPlanes = weightsSplits > 1 || (fp32 && odd_rows(q)) ? room.take<float>(static_cast<size_t>(weightsSplits) * piece * ld) : nullptr;
		weightsRows = weightsPlanes == nullptr && odd_rows(q) ? room.take<uint16_t>(piece * ld) : nullptr;
	}
};

bool valid(const Problem& q)
{
	if(!type_valid(q.type) || q.rows < 0 || q.width < 1 || q.vocabulary < 1 || q.hiddenRow < q.width || q.weightsRow < q.width) return false;
	return type_aligned(q.hidden, q.type) && type_aligned(q.weights, q.type);
}
bool too_big(const Problem& q)
{
	return q.rows > (1 << 24) || q.vocabulary > (1 << 28) || q.width > (1 << 24);
}

// ---- launches -----------------------------------------------------------------------------------------------------------

dim3 units_grid(int rows, int perRow) { return dim3(grid_for(static_cast<long long>(rows) * perRow, 256, 8)); }

void copy_rows(const void* src, long long srcRow, int rows, int width, uint16_t* dst, const int* labels, const float* lossDiff, int vocabulary,
	cudaStream_t stream)
{
	const int ld = round_up(width, 8);
	launch_dependent(true, copy_rows16_kernel, units_grid(rows, ld / 8), dim3(256), 0, stream, static_cast<const uint16_t*>(src), srcRow, rows, width, dst,
		ld, labels, lossDiff, vocabulary);
	count_launch();
}

void split_rows(const void* src, long long srcRow, int rows, int width, uint16_t* dst, long long plane, const int* labels, const float* lossDiff,
	int vocabulary, cudaStream_t stream)
{
	const int ld = round_up(width, 8);
	launch_dependent(true, split_rows_kernel, units_grid(rows, ld / 8), dim3(256), 0, stream, static_cast<const float*>(src), srcRow, rows, width,
		reinterpret_cast<__nv_bfloat16*>(dst), ld, plane, labels, lossDiff, vocabulary);
	count_launch();
}

// Columns [first, first + columns) of the weights: planes made here (fp32), the copy made before, or as they are.
Aligned weights_piece(const Problem& q, uint16_t* room, int first, int columns, int piece, cudaStream_t stream)
{
	const long long ld = round_up(q.width, 8);
	if(q.type == NB200_TYPE_FP32) {
		split_rows(static_cast<const float*>(q.weights) + first * q.weightsRow, q.weightsRow, columns, q.width, room, piece * ld, nullptr, nullptr, 0, stream);
		return { room, ld, piece * ld };
	}
	const uint16_t* const all = room != nullptr ? room : static_cast<const uint16_t*>(q.weights);
	const long long row = room != nullptr ? ld : q.weightsRow;
	return { all + first * row, row, 0 };
}

Product16Params params_of(const Problem& q, int m, int n, int splits, int k, bool mFast, int tileColumns = PRODUCT16_N)
{
	Product16Params p = {};
	p.m = m; p.n = n;
	p.mTiles = (m + PRODUCT16_M - 1) / PRODUCT16_M;
	p.nTiles = (n + tileColumns - 1) / tileColumns;
	p.narrow = tileColumns == PRODUCT16_N ? 0 : 1;
	p.boxA = product16_box_a(m);
	p.splits = splits;
	p.kBlocks = (k + PRODUCT16_K - 1) / PRODUCT16_K;
	p.kBlocksPerSplit = (p.kBlocks + splits - 1) / splits;
	p.mFast = mFast ? 1 : 0;
	p.fp32 = q.type == NB200_TYPE_FP32 ? 1 : 0;
	p.bf16 = q.type == NB200_TYPE_FP16 ? 0 : 1;
	p.status = device_status_word();
	return p;
}

FewParams few_params(const Problem& q, const int* labels)
{
	FewParams p = {};
	p.hidden = static_cast<const float*>(q.hidden); p.weights = static_cast<const float*>(q.weights); p.hiddenRow = q.hiddenRow; p.weightsRow = q.weightsRow;
	p.rows = q.rows; p.width = q.width; p.vocabulary = q.vocabulary; p.perBlock = few_entries(q.rows, q.vocabulary);
	p.labels = labels;
	return p;
}

void join_partials(const Problem& q, const float2* partial, int parts, const float* labelled, const int* labels, bool products, float* loss,
	float* logSum, cudaStream_t stream)
{
	launch_dependent(true, join_partials_kernel, dim3((q.rows + 31) / 32), dim3(JOIN_WARPS * 32), 0, stream, partial, parts, q.rows, labelled, labels,
		q.vocabulary, products ? 1 : 0, loss, logSum);
	count_launch();
}

int forward(const Problem& q, const int* labels, float* loss, float* logSum, void* scratch, cudaStream_t stream)
{
	Room room = { static_cast<uint8_t*>(scratch) };
	if(few_rows(q, false)) {
		const FewRoom w(q, false, room);
		FewParams p = few_params(q, labels);
		p.partial = w.partial; p.labelled = w.labelled;
		const int rc = few_forward(p, stream);
		if(rc != NB200_OK) return rc;
		join_partials(q, w.partial, few_blocks(q.rows, q.vocabulary), w.labelled, labels, true, loss, logSum, stream);
		return check_launch();
	}
	const Forward f(q, room);
	const bool fp32 = q.type == NB200_TYPE_FP32, bf16 = q.type != NB200_TYPE_FP16;
	const long long ld = round_up(q.width, 8);
	if(fp32) split_rows(q.hidden, q.hiddenRow, q.rows, q.width, f.hidden, q.rows * ld, nullptr, nullptr, 0, stream);
	else if(f.hidden != nullptr) copy_rows(q.hidden, q.hiddenRow, q.rows, q.width, f.hidden, nullptr, nullptr, 0, stream);
	if(!fp32 && f.weights != nullptr) copy_rows(q.weights, q.weightsRow, q.vocabulary, q.width, f.weights, nullptr, nullptr, 0, stream);
	CUtensorMap a, b;
	if(!product16_map(&a, f.hidden ? f.hidden : q.hidden, bf16, q.width, q.rows, f.hidden ? ld : q.hiddenRow, product16_box_a(q.rows), fp32 ? q.rows * ld : 0)) return NB200_EINVAL;
	for(int first = 0; first < q.vocabulary; first += f.piece) {
		const int columns = q.vocabulary - first < f.piece ? q.vocabulary - first : f.piece;
		const Aligned w = weights_piece(q, f.weights, first, columns, f.piece, stream);
		if(!product16_map(&b, w.p, bf16, q.width, columns, w.row, f.tileColumns, w.plane)) return NB200_EINVAL;
		Product16Params p = params_of(q, q.rows, columns, 1, q.width, true, f.tileColumns);
		p.partial = f.partial + static_cast<long long>(first / f.tileColumns) * 2 * q.rows;
		p.labelled = f.labelled; p.labels = labels; p.firstColumn = first; p.columns = q.vocabulary;
		const int rc = product16(PRODUCT16_STATS, false, false, p, &a, &b, stream);
		if(rc != NB200_OK) return rc;
	}
	join_partials(q, f.partial, f.parts, f.labelled, labels, false, loss, logSum, stream);
	return check_launch();
}

template<typename T>
void sum_planes_of(const Problem& q, const float* planes, int count, int rows, const float* by, void* out, long long outRow, cudaStream_t stream)
{
	const long long ld = round_up(q.width, 8);
	const long long quads = static_cast<long long>(rows) * ((q.width + 3) / 4);
	// few results of many planes: 11 x 334 of 64 planes took 11 us with one thread, 4.5 with eight
	const int group = count > 8 && quads * 8 <= sm_count() * 2048ll ? 8 : 1;
	const dim3 grid(grid_for(quads * group, 256, 16));
	launch_dependent(true, sum_planes_kernel<T>, grid, dim3(256), 0, stream, planes, count, rows * ld, ld, rows, q.width, group, by, static_cast<T*>(out), outRow);
	count_launch();
}
void sum_planes(const Problem& q, const float* planes, int count, int rows, const float* by, void* out, long long outRow, cudaStream_t stream)
{
	if(q.type == NB200_TYPE_FP32) sum_planes_of<float>(q, planes, count, rows, by, out, outRow, stream);
	else if(q.type == NB200_TYPE_FP16) sum_planes_of<__half>(q, planes, count, rows, by, out, outRow, stream);
	else sum_planes_of<__nv_bfloat16>(q, planes, count, rows, by, out, outRow, stream);
}

int backward(const Problem& q, const float* lossDiff, const int* labels, const float* logSum, void* hiddenDiff, long long hiddenDiffRow,
	void* weightsDiff, long long weightsDiffRow, void* scratch, cudaStream_t stream)
{
	Room room = { static_cast<uint8_t*>(scratch) };
	if(few_rows(q, true)) {
		const FewRoom few(q, true, room);
		FewParams p = few_params(q, labels);
		p.logSum = logSum; p.lossDiff = lossDiff;
		p.weightsDiff = static_cast<float*>(weightsDiff); p.weightsDiffRow = weightsDiffRow;
		p.hiddenPart = hiddenDiff != nullptr ? few.hiddenPart : nullptr;
		return few_backward(p, static_cast<float*>(hiddenDiff), hiddenDiffRow, stream);
	}
	const Backward w(q, room);
	const bool fp32 = q.type == NB200_TYPE_FP32, bf16 = q.type != NB200_TYPE_FP16;
	const long long ld = round_up(q.width, 8), hiddenPlane = fp32 ? q.rows * ld : 0, diffPlane = fp32 ? static_cast<long long>(q.rows) * w.piece : 0;
	if(fp32) split_rows(q.hidden, q.hiddenRow, q.rows, q.width, w.hidden, hiddenPlane, labels, lossDiff, q.vocabulary, stream);
	else copy_rows(q.hidden, q.hiddenRow, q.rows, q.width, w.hidden, labels, lossDiff, q.vocabulary, stream);
	launch_dependent(true, diff_scale_kernel, dim3(1), dim3(SCALE_THREADS), 0, stream, q.rows, labels, lossDiff, q.vocabulary, w.scale, q.type);
	count_launch();
	if(!fp32 && w.weights != nullptr) copy_rows(q.weights, q.weightsRow, q.vocabulary, q.width, w.weights, nullptr, nullptr, 0, stream);
	CUtensorMap hidden, hiddenAcross, rows, across, diff, diffAcross;
	if(!product16_map(&hidden, w.hidden, bf16, q.width, q.rows, ld, product16_box_a(q.rows), hiddenPlane)
		|| !product16_map(&hiddenAcross, w.hidden, bf16, q.width, q.rows, ld, PRODUCT16_BOX_ACROSS, hiddenPlane)
		|| !product16_map(&diff, w.diff, bf16, w.piece, q.rows, w.piece, product16_box_a(q.rows), diffPlane)
		|| !product16_map(&diffAcross, w.diff, bf16, w.piece, q.rows, w.piece, PRODUCT16_BOX_ACROSS, diffPlane)) return NB200_EINVAL;
	for(int first = 0; first < q.vocabulary; first += w.piece) {
		const int columns = q.vocabulary - first < w.piece ? q.vocabulary - first : w.piece;
		const Aligned piece = weights_piece(q, w.weights, first, columns, w.piece, stream);
		if(!product16_map(&rows, piece.p, bf16, q.width, columns, piece.row, w.tileColumns, piece.plane)
			|| !product16_map(&across, piece.p, bf16, q.width, columns, piece.row, PRODUCT16_BOX_ACROSS, piece.plane)) return NB200_EINVAL;
		Product16Params p = params_of(q, q.rows, columns, 1, q.width, true, w.tileColumns);
		p.labels = labels; p.firstColumn = first; p.columns = q.vocabulary;
		p.logSum = logSum; p.rowScale = lossDiff; p.scale = w.scale;
		p.out = w.diff; p.ldOut = w.piece; p.outPlane = diffPlane;
		int rc = product16(PRODUCT16_DIFF, false, false, p, &hidden, &rows, stream);
		if(rc != NB200_OK) return rc;
		if(hiddenDiff != nullptr) {
			// dz ends in zeros behind the vocabulary, up to whole K blocks
			p = params_of(q, q.rows, q.width, w.hiddenSplits, columns, false);
			p.plane = w.hiddenPlanes; p.ldPlane = ld; p.accumulate = first > 0;
			rc = product16(PRODUCT16_SUM, false, true, p, &diff, &across, stream);
			if(rc != NB200_OK) return rc;
		}
		if(weightsDiff != nullptr) {
			void* const out = static_cast<uint8_t*>(weightsDiff) + first * weightsDiffRow * type_size(q.type);
			p = params_of(q, columns, q.width, w.weightsSplits, q.rows, false);
			if(w.weightsPlanes != nullptr) {
				p.plane = w.weightsPlanes; p.ldPlane = ld;
				rc = product16(PRODUCT16_SUM, true, true, p, &diffAcross, &hiddenAcross, stream);
				if(rc != NB200_OK) return rc;
				sum_planes(q, w.weightsPlanes, p.splits, columns, w.scale + 2, out, weightsDiffRow, stream);
			} else {
				p.out = w.weightsRows != nullptr ? w.weightsRows : out;
				p.ldOut = w.weightsRows != nullptr ? ld : weightsDiffRow;
				p.resultScale = w.scale + 2;
				rc = product16(PRODUCT16_STORE, true, true, p, &diffAcross, &hiddenAcross, stream);
				if(rc != NB200_OK) return rc;
				if(w.weightsRows != nullptr) {
					launch_dependent(true, spread_rows16_kernel, units_grid(columns, (q.width + 14) / 8), dim3(256), 0, stream,
						static_cast<const uint16_t*>(w.weightsRows), static_cast<int>(ld), columns, q.width, static_cast<uint16_t*>(out), weightsDiffRow);
					count_launch();
				}
			}
		}
	}
	if(hiddenDiff != nullptr) sum_planes(q, w.hiddenPlanes, w.hiddenSplits, q.rows, w.scale + 2, hiddenDiff, hiddenDiffRow, stream);
	return check_launch();
}

bool scratch_valid(const void* scratch) { return scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 255u) == 0; }

} // namespace

} // namespace nb200

using namespace nb200;

extern "C" {

size_t nb200_vocabulary_cross_entropy_scratch_bytes(int type, const void* hidden, int rows, int width, long long hidden_row_size,
	const void* weights, int vocabulary, long long weights_row_size, int backward)
{
	const Problem q = { type, rows, width, vocabulary, hidden, weights, hidden_row_size, weights_row_size };
	if(!valid(q) || rows == 0 || too_big(q)) return 0;
	Room room = { nullptr };
	if(few_rows(q, backward != 0)) FewRoom(q, backward != 0, room);
	else if(backward) Backward(q, room);
	else Forward(q, room);
	return room.used;
}

int nb200_vocabulary_cross_entropy(void* stream, int type, const void* hidden, int rows, int width, long long hidden_row_size,
	const void* weights, int vocabulary, long long weights_row_size, const int* labels, float* loss, float* log_sum, void* scratch)
{
	const Problem q = { type, rows, width, vocabulary, hidden, weights, hidden_row_size, weights_row_size };
	if(!valid(q)) return NB200_EINVAL;
	if(rows == 0) return NB200_OK;
	if(too_big(q)) return NB200_ETOOBIG; // before the scratch memory, which has no size then
	if(hidden == nullptr || weights == nullptr || labels == nullptr || loss == nullptr || log_sum == nullptr || !scratch_valid(scratch)
		|| !words_aligned(labels, loss, log_sum)) return NB200_EINVAL;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	return forward(q, labels, loss, log_sum, scratch, as_stream(stream));
}

int nb200_vocabulary_cross_entropy_backward(void* stream, int type, const float* loss_diff, const void* hidden, int rows, int width,
	long long hidden_row_size, const void* weights, int vocabulary, long long weights_row_size, const int* labels, const float* log_sum,
	void* hidden_diff, long long hidden_diff_row_size, void* weights_diff, long long weights_diff_row_size, void* scratch)
{
	const Problem q = { type, rows, width, vocabulary, hidden, weights, hidden_row_size, weights_row_size };
	if(!valid(q)) return NB200_EINVAL;
	if((hidden_diff != nullptr && hidden_diff_row_size < width) || (weights_diff != nullptr && weights_diff_row_size < width)
		|| !type_aligned(hidden_diff, type) || !type_aligned(weights_diff, type)) return NB200_EINVAL;
	if(hidden_diff == nullptr && weights_diff == nullptr) return NB200_OK;
	if(too_big(q)) return NB200_ETOOBIG;
	if(rows > 0 && (hidden == nullptr || weights == nullptr || labels == nullptr || loss_diff == nullptr || log_sum == nullptr
		|| !scratch_valid(scratch) || !words_aligned(loss_diff, labels, log_sum))) return NB200_EINVAL;
	if(rows == 0 && weights_diff == nullptr) return NB200_OK;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	if(rows == 0) { // sums over no rows
		zero_rows_kernel<<<grid_for(vocabulary, 1, 16), 256, 0, as_stream(stream)>>>(static_cast<uint8_t*>(weights_diff),
			weights_diff_row_size * type_size(type), static_cast<long long>(width) * type_size(type), vocabulary);
		count_launch();
		return check_launch();
	}
	return backward(q, loss_diff, labels, log_sum, hidden_diff, hidden_diff_row_size, weights_diff, weights_diff_row_size, scratch,
		as_stream(stream));
}

} // extern "C"
