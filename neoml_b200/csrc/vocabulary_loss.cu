// Softmax cross entropy of hidden rows against a vocabulary's weights, forward and backward, without keeping the logits.
//
//   z = hidden weights^T,  log_sum = log sum_j exp z_j,  loss = log_sum - z_label
//   dz = loss_diff (softmax(z) - [j = label]),  hidden_diff = dz weights,  weights_diff = dz^T hidden
//
// 16-bit types: the forward pass is one product whose epilogue reduces each row's 128 columns to a maximum and a sum, so that
// 8 bytes per row leave the SM for 128 logits (product16.cu).  The backward pass forms the logits anew, piece by piece of the vocabulary: a product
// whose epilogue turns them into dz, and the two products that consume it.  Bound by the tensor core: 8 rows vocabulary
// width multiply-adds in all for forward and backward, where keeping the logits would take 6 and rows x vocabulary memory.
//   dz is kept in the operands' type for those products: the tensor core multiplies like types, and its rounding, half a
//   step per element with no common direction, is of the size of the results' own.  In fp16 it is scaled by a power
//   of two that puts the largest loss_diff at 2^14, because softmax values of 1e-7 are below what a half holds; dz between 1
//   and 2^-38 of the largest then keeps some or all of its bits.  hidden_diff is summed in fp32 over the pieces.
// fp32: the library's own products of fp32 matrices (three tensor-core products of split operands) over pieces of logits in scratch
// memory, with a pass over them for the sums or for dz and its transposed copy.  The tensor core's own additions cut off rather than
// round: a sum's error grows by about 1.1e-9 of its value per element (measured: 1.3e-6 of the result's norm at a depth of 1023,
// 3.5e-5 at 30011), so that no product here is deeper than 1024; what is deeper is summed from such parts, in fp32 and in order.
#include "product16.cuh"

#include <cuda.h>

namespace nb200 {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int DEPTH = 1024;                    // of one fp32 product
constexpr long long PIECE_BYTES = 256ll << 20; // of dz (16-bit), of logits and their transposed copy (fp32)

__device__ __forceinline__ bool has_target(const int* labels, int row, int vocabulary)
{
	const int label = __ldg(labels + row);
	return label >= 0 && label < vocabulary;
}

// ---- 16-bit types ---------------------------------------------------------------------------------------------------

// Rows of 16-bit elements copied to aligned rows.  With labels: a row without a target or with a loss_diff of zero becomes
// zeros -- it has no gradient, whatever it holds -- and the first block finds the scale of dz.
__global__ void __launch_bounds__(256) copy_rows16_kernel(const uint16_t* __restrict__ src, long long srcRow, int rows, int width,
	uint16_t* __restrict__ dst, int dstRow, const int* __restrict__ labels, const float* __restrict__ lossDiff, int vocabulary,
	float* scale, int fp16)
{
	int block = blockIdx.x, blocks = gridDim.x;
	if(scale != nullptr) {
		if(block == 0) {
			__shared__ float slots[8];
			float most = 0.f;
			for(int r = threadIdx.x; r < rows; r += blockDim.x) {
				if(has_target(labels, r, vocabulary)) most = fmaxf(most, fabsf(lossDiff[r]));
			}
			most = warp_max_all(most);
			if((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = most;
			__syncthreads();
			if(threadIdx.x == 0) {
				for(int i = 1; i < 8; ++i) most = fmaxf(most, slots[i]);
				int e = 0;
				if(fp16 && most > 0.f && most < INFINITY) {
					e = 14 - ilogbf(most);
					e = e > 100 ? 100 : e < -100 ? -100 : e;
				}
				scale[0] = ldexpf(1.f, e);
				scale[1] = ldexpf(1.f, -e);
			}
			return;
		}
		--block;
		--blocks;
	}
	const bool vector = (srcRow & 7) == 0 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
	for(long long r = block; r < rows; r += blocks) {
		const bool keep = labels == nullptr || (has_target(labels, static_cast<int>(r), vocabulary) && !(lossDiff[r] == 0.f));
		const uint16_t* const from = src + r * srcRow;
		uint16_t* const to = dst + r * dstRow;
		if(vector) {
			for(int i = threadIdx.x * 8; i < width; i += blockDim.x * 8) {
				if(i + 8 <= width) {
					*reinterpret_cast<uint4*>(to + i) = keep ? *reinterpret_cast<const uint4*>(from + i) : make_uint4(0u, 0u, 0u, 0u);
				} else {
					for(int j = i; j < dstRow; ++j) to[j] = keep && j < width ? from[j] : 0;
				}
			}
		} else {
			for(int i = threadIdx.x; i < dstRow; i += blockDim.x) to[i] = keep && i < width ? from[i] : 0;
		}
	}
}

// Joins the partial sums of a row.  32 rows per block, eight threads a row.
__global__ void __launch_bounds__(256) join_partials_kernel(const float2* __restrict__ partial, int parts, int rows,
	const float* __restrict__ labelled, const int* __restrict__ labels, int vocabulary, float* __restrict__ loss, float* __restrict__ logSum)
{
	__shared__ float2 slots[8][32];
	dependent_wait();
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	const int row = blockIdx.x * 32 + lane;
	float top = -INFINITY, sum = 0.f;
	auto join = [&](float2 o) {
		const float t = fmaxf(top, o.x), at = t == -INFINITY ? 0.f : t;
		sum = sum * exp2f(top - at) + o.y * exp2f(o.x - at);
		top = t;
	};
	if(row < rows) {
		for(int i = warp; i < parts; i += 8) join(partial[static_cast<long long>(i) * rows + row]);
	}
	slots[warp][lane] = make_float2(top, sum);
	__syncthreads();
	if(warp != 0 || row >= rows) return;
	for(int i = 1; i < 8; ++i) join(slots[i][lane]);
	const float value = top / LOG2E + logf(sum);
	logSum[row] = value;
	loss[row] = has_target(labels, row, vocabulary) ? value - labelled[row] : 0.f;
}

// out[row][col] = sum of the planes, in order, times *by
template<typename T>
__global__ void __launch_bounds__(256) sum_planes_kernel(const float* __restrict__ planes, int count, long long planeSize, long long ldPlane,
	int rows, int width, const float* __restrict__ by, T* __restrict__ out, long long outRow)
{
	dependent_wait();
	const float scale = __ldg(by);
	const int quads = (width + 3) / 4;
	const bool vector = (outRow & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7u) == 0;
	const long long total = static_cast<long long>(rows) * quads;
	const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
	for(long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
		const long long row = i / quads;
		const int col = static_cast<int>(i - row * quads) * 4;
		float4 v = *reinterpret_cast<const float4*>(planes + row * ldPlane + col);
		for(int k = 1; k < count; ++k) {
			const float4 w = *reinterpret_cast<const float4*>(planes + k * planeSize + row * ldPlane + col);
			v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
		}
		T* const to = out + row * outRow + col;
		if(vector && col + 4 <= width) {
			*reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(v.x * scale, v.y * scale), pack2<T>(v.z * scale, v.w * scale));
		} else {
			const float f[4] = { v.x, v.y, v.z, v.w };
			for(int j = 0; j < 4 && col + j < width; ++j) to[j] = from_float<T>(f[j] * scale);
		}
	}
}

// ---- fp32 -----------------------------------------------------------------------------------------------------------

// A row's running maximum, sum and labelled logit over one more piece; the last piece gives the results.
__global__ void __launch_bounds__(256) fp32_stats_kernel(const float* __restrict__ z, int ld, int columns, int firstColumn, int first,
	int last, int vocabulary, const int* __restrict__ labels, float2* __restrict__ running, float* __restrict__ labelled,
	float* __restrict__ loss, float* __restrict__ logSum)
{
	__shared__ float2 slots[8];
	const long long row = blockIdx.x;
	const float* const x = z + row * ld;
	float top = -INFINITY, sum = 0.f;
	auto join = [&](float t2, float s2) {
		const float t = fmaxf(top, t2), at = t == -INFINITY ? 0.f : t;
		sum = sum * exp2f(top - at) + s2 * exp2f(t2 - at);
		top = t;
	};
	for(int c = threadIdx.x; c < columns; c += blockDim.x) join(x[c] * LOG2E, 1.f);
#pragma unroll
	for(int o = 16; o > 0; o >>= 1) {
		const float t2 = __shfl_xor_sync(0xffffffffu, top, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
		join(t2, s2);
	}
	if((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = make_float2(top, sum);
	__syncthreads();
	if(threadIdx.x != 0) return;
	for(int w = 1; w < 8; ++w) join(slots[w].x, slots[w].y);
	if(!first) join(running[row].x, running[row].y);
	running[row] = make_float2(top, sum);
	const int label = labels[row];
	const bool used = label >= 0 && label < vocabulary;
	if(used && label >= firstColumn && label - firstColumn < columns) labelled[row] = x[label - firstColumn];
	if(last) {
		const float value = top / LOG2E + logf(sum);
		logSum[row] = value;
		loss[row] = used ? value - labelled[row] : 0.f;
	}
}

// dz of a piece of logits in the two forms that the products take: `along`, [parts of DEPTH columns][rows][DEPTH], the last part
// filled up with zeros, and `across`, [columns][ldAcross]; each null where it is not wanted.  32 x 32 squares.
__global__ void __launch_bounds__(256) fp32_diff_kernel(const float* __restrict__ z, int ld, int rows, int columns, int firstColumn,
	int vocabulary, const int* __restrict__ labels, const float* __restrict__ logSum, const float* __restrict__ lossDiff,
	float* __restrict__ along, float* __restrict__ across, int ldAcross)
{
	__shared__ float square[32][33];
	const int c0 = blockIdx.x * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
	const int part = c0 / DEPTH, inPart = c0 - part * DEPTH;
	for(int r0 = blockIdx.y * 32; r0 < rows; r0 += gridDim.y * 32) {
		for(int k = ty; k < 32; k += 8) {
			const int row = r0 + k, c = c0 + tx;
			float v = 0.f;
			if(row < rows) {
				if(c < columns) {
					const int label = labels[row];
					const float by = label >= 0 && label < vocabulary ? lossDiff[row] : 0.f;
					if(!(by == 0.f)) {
						v = expf(z[static_cast<long long>(row) * ld + c] - logSum[row]) - (label == firstColumn + c ? 1.f : 0.f);
						v *= by;
					}
				}
				if(along != nullptr) along[(static_cast<long long>(part) * rows + row) * DEPTH + inPart + tx] = v;
			}
			square[k][tx] = v;
		}
		__syncthreads();
		if(across != nullptr) {
			for(int k = ty; k < 32; k += 8) {
				const int c = c0 + k, row = r0 + tx;
				if(c < columns && row < rows) across[static_cast<long long>(c) * ldAcross + row] = square[tx][k];
			}
		}
		__syncthreads();
	}
}

// dst[c][r] = src[r][c].  With labels, rows without a gradient become zeros.  partRows > 0: the rows in parts of as many,
// [part][columns][partRows], the last one filled up with zeros (partRows is a multiple of 32).
__global__ void __launch_bounds__(256) fp32_across_kernel(const float* __restrict__ src, long long srcRow, int rows, int columns,
	float* __restrict__ dst, int dstRow, int partRows, const int* __restrict__ labels, const float* __restrict__ lossDiff, int vocabulary)
{
	__shared__ float square[32][33];
	const int c0 = blockIdx.x * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
	const int end = partRows > 0 ? (rows + partRows - 1) / partRows * partRows : rows;
	for(int r0 = blockIdx.y * 32; r0 < end; r0 += gridDim.y * 32) {
		for(int k = ty; k < 32; k += 8) {
			const int row = r0 + k, c = c0 + tx;
			float v = 0.f;
			if(row < rows && c < columns && (labels == nullptr || (has_target(labels, row, vocabulary) && !(lossDiff[row] == 0.f)))) {
				v = src[row * srcRow + c];
			}
			square[k][tx] = v;
		}
		__syncthreads();
		const int part = partRows > 0 ? r0 / partRows : 0;
		float* const to = partRows > 0 ? dst + static_cast<long long>(part) * columns * partRows + (r0 - part * partRows) : dst + r0;
		for(int k = ty; k < 32; k += 8) {
			const int c = c0 + k;
			if(c < columns && r0 + tx < end) to[static_cast<long long>(c) * dstRow + tx] = square[tx][k];
		}
		__syncthreads();
	}
}

// out (+)= the planes, one after another
__global__ void __launch_bounds__(256) fp32_sum_kernel(const float* __restrict__ planes, int count, long long planeSize, int ldPlane, int rows,
	int width, float* __restrict__ out, long long outRow, int accumulate)
{
	const long long total = static_cast<long long>(rows) * width;
	const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
	for(long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
		const long long row = i / width, col = i - row * width;
		float v = accumulate ? out[row * outRow + col] : 0.f;
		for(int k = 0; k < count; ++k) v += planes[k * planeSize + row * ldPlane + col];
		out[row * outRow + col] = v;
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

// Columns of the vocabulary that are handled at a time.
int piece_of(const Problem& q)
{
	const long long perColumn = q.type == NB200_TYPE_FP32 ? 12ll * round_up(q.rows, 4) : 2ll * q.rows;
	const long long whole = round_up(q.vocabulary, PRODUCT16_N);
	long long piece = PIECE_BYTES / perColumn / PRODUCT16_N * PRODUCT16_N;
	if(q.type == NB200_TYPE_FP32) { // the fp32 products count the elements of an operand in 31 bits
		const long long row = q.weightsRow > q.width ? q.weightsRow : q.width;
		const long long most = (1ll << 30) / row / PRODUCT16_N * PRODUCT16_N;
		if(piece > most) piece = most;
	}
	if(piece < PRODUCT16_N) piece = PRODUCT16_N;
	if(piece >= whole) return static_cast<int>(whole);
	const long long pieces = (whole + piece - 1) / piece;   // of equal size
	return round_up((whole + pieces - 1) / pieces, PRODUCT16_N);
}

// Parts of K where a product has few tiles: enough for one tile per SM, none shorter than 8 steps of 64.
int splits_of(long long tiles, int kBlocks)
{
	const int sms = sm_count();
	if(tiles * 2 > sms) return 1;
	long long splits = sms / tiles;
	if(splits > kBlocks / 8) splits = kBlocks / 8;
	if(splits > 64) splits = 64;
	return splits < 1 ? 1 : static_cast<int>(splits);
}

struct Forward16 {
	float2* partial;
	float* labelled;
	uint16_t *hidden, *weights; // copies in aligned rows; null: as they are
	Forward16(const Problem& q, Room& room)
	{
		const int nTiles = (q.vocabulary + PRODUCT16_N - 1) / PRODUCT16_N;
		partial = room.take<float2>(static_cast<size_t>(nTiles) * 2 * q.rows);
		labelled = room.take<float>(q.rows);
		hidden = rows_for_tma(q.hidden, q.hiddenRow) ? nullptr : room.take<uint16_t>(static_cast<size_t>(q.rows) * round_up(q.width, 8));
		weights = rows_for_tma(q.weights, q.weightsRow) ? nullptr : room.take<uint16_t>(static_cast<size_t>(q.vocabulary) * round_up(q.width, 8));
	}
};

struct Backward16 {
	int piece, hiddenSplits, weightsSplits;
	float* scale;
	uint16_t *hidden, *weights, *diff;
	float *hiddenPlanes, *weightsPlanes;
	Backward16(const Problem& q, Room& room)
	{
		piece = piece_of(q);
		const long long mTiles = (q.rows + PRODUCT16_M - 1) / PRODUCT16_M, dTiles = (q.width + PRODUCT16_N - 1) / PRODUCT16_N;
		hiddenSplits = splits_of(mTiles * dTiles, piece / PRODUCT16_K);
		// its result goes straight to the caller where K is not split
		weightsSplits = splits_of(piece / PRODUCT16_M * dTiles, (q.rows + PRODUCT16_K - 1) / PRODUCT16_K);
		const size_t ld = round_up(q.width, 8);
		scale = room.take<float>(2);
		hidden = room.take<uint16_t>(q.rows * ld);
		weights = rows_for_tma(q.weights, q.weightsRow) ? nullptr : room.take<uint16_t>(q.vocabulary * ld);
		diff = room.take<uint16_t>(static_cast<size_t>(q.rows) * piece);
		hiddenPlanes = room.take<float>(static_cast<size_t>(hiddenSplits) * q.rows * ld);
		weightsPlanes = weightsSplits > 1 ? room.take<float>(static_cast<size_t>(weightsSplits) * piece * ld) : nullptr;
	}
};

// Floats of work space for any of the fp32 products that a pass makes.
size_t product_room(const Problem& q, int piece, int parts, bool backward)
{
	size_t most = 0;
	auto need = [&](int batch, int m, int n, int k, long long ldb) {
		const size_t s = nb200_matrix_product_scratch_floats(batch, m, n, k, static_cast<int>(ldb));
		if(s > most) most = s;
	};
	const int lastColumns = q.vocabulary - (q.vocabulary - 1) / piece * piece;
	const int lastWidth = q.width - (q.width - 1) / DEPTH * DEPTH, lastRows = q.rows - (q.rows - 1) / DEPTH * DEPTH;
	for(int columns : { q.vocabulary < piece ? q.vocabulary : piece, lastColumns }) {
		for(int depth : { q.width < DEPTH ? q.width : DEPTH, lastWidth }) need(1, q.rows, columns, depth, q.weightsRow);
		if(backward) {
			for(int depth : { q.rows < DEPTH ? q.rows : DEPTH, lastRows }) need(1, columns, q.width, depth, round_up(q.rows, 4));
		}
	}
	if(backward) {
		for(int batch = 1; batch <= parts; ++batch) need(batch, q.rows, q.width, DEPTH, DEPTH);
	}
	return most;
}

struct Forward32 {
	int piece;
	float *z, *labelled, *product;
	float2* running;
	Forward32(const Problem& q, Room& room)
	{
		piece = piece_of(q);
		z = room.take<float>(static_cast<size_t>(q.rows) * piece);
		running = room.take<float2>(q.rows);
		labelled = room.take<float>(q.rows);
		product = room.take<float>(product_room(q, piece, 0, false));
	}
};

struct Backward32 {
	int piece, parts; // parts of DEPTH columns that are multiplied at a time: enough for two tiles per SM
	float *z, *diffAlong, *diffAcross, *hiddenAcross, *weightsAcross, *planes, *product;
	Backward32(const Problem& q, Room& room)
	{
		piece = piece_of(q);
		const int whole = (piece + DEPTH - 1) / DEPTH;
		const long long tiles = static_cast<long long>((q.rows + 127) / 128) * ((q.width + 127) / 128);
		parts = static_cast<int>((2ll * sm_count() + tiles - 1) / tiles);
		if(parts > whole) parts = whole;
		z = room.take<float>(static_cast<size_t>(q.rows) * piece);
		diffAlong = room.take<float>(static_cast<size_t>(q.rows) * whole * DEPTH);
		diffAcross = room.take<float>(static_cast<size_t>(piece) * round_up(q.rows, 4));
		hiddenAcross = room.take<float>(static_cast<size_t>(q.width) * round_up(q.rows, 4));
		weightsAcross = room.take<float>(static_cast<size_t>(q.width) * whole * DEPTH);
		planes = room.take<float>(static_cast<size_t>(parts) * q.rows * round_up(q.width, 4));
		product = room.take<float>(product_room(q, piece, parts, true));
	}
};

bool valid(const Problem& q)
{
	if(!type_valid(q.type) || q.rows < 0 || q.width < 1 || q.vocabulary < 1 || q.hiddenRow < q.width || q.weightsRow < q.width) return false;
	return type_aligned(q.hidden, q.type) && type_aligned(q.weights, q.type);
}
bool too_big(const Problem& q)
{
	if(q.rows > (1 << 22) || q.vocabulary > (1 << 28) || q.width > (1 << 22) || q.hiddenRow > 0x7fffffff || q.weightsRow > 0x7fffffff) return true;
	// the fp32 products count the elements of an operand in 31 bits
	const long long most = 0x7fffffff;
	return q.type == NB200_TYPE_FP32 && (q.rows * q.hiddenRow > most || static_cast<long long>(round_up(q.rows, 4)) * q.width > most
		|| PRODUCT16_N * (q.weightsRow > q.width ? q.weightsRow : q.width) > most);
}

// ---- launches -----------------------------------------------------------------------------------------------------------

void copy_rows(const void* src, long long srcRow, int rows, int width, uint16_t* dst, const int* labels, const float* lossDiff,
	int vocabulary, float* scale, int fp16, cudaStream_t stream)
{
	copy_rows16_kernel<<<grid_for(rows, 1, 16) + (scale != nullptr ? 1 : 0), 256, 0, stream>>>(static_cast<const uint16_t*>(src), srcRow, rows, width, dst,
		round_up(width, 8), labels, lossDiff, vocabulary, scale, fp16);
	count_launch();
}

int forward16(const Problem& q, const int* labels, float* loss, float* logSum, void* scratch, cudaStream_t stream)
{
	Room room = { static_cast<uint8_t*>(scratch) };
	const Forward16 f(q, room);
	const bool bf16 = q.type == NB200_TYPE_BF16;
	const int ld = round_up(q.width, 8);
	if(f.hidden != nullptr) copy_rows(q.hidden, q.hiddenRow, q.rows, q.width, f.hidden, nullptr, nullptr, 0, nullptr, 0, stream);
	if(f.weights != nullptr) copy_rows(q.weights, q.weightsRow, q.vocabulary, q.width, f.weights, nullptr, nullptr, 0, nullptr, 0, stream);
	CUtensorMap a, b;
	if(!product16_map(&a, f.hidden ? f.hidden : q.hidden, bf16, q.width, q.rows, f.hidden ? ld : q.hiddenRow, PRODUCT16_BOX_A)
		|| !product16_map(&b, f.weights ? f.weights : q.weights, bf16, q.width, q.vocabulary, f.weights ? ld : q.weightsRow, PRODUCT16_BOX_B)) {
		return NB200_EINVAL;
	}
	Product16Params p = {};
	p.m = q.rows; p.n = q.vocabulary;
	p.mTiles = (q.rows + PRODUCT16_M - 1) / PRODUCT16_M;
	p.nTiles = (q.vocabulary + PRODUCT16_N - 1) / PRODUCT16_N;
	p.splits = 1;
	p.kBlocks = p.kBlocksPerSplit = (q.width + PRODUCT16_K - 1) / PRODUCT16_K;
	p.mFast = 1; p.bf16 = bf16; p.status = device_status_word();
	p.partial = f.partial; p.labelled = f.labelled; p.labels = labels; p.columns = q.vocabulary;
	const int rc = product16(PRODUCT16_STATS, false, false, p, &a, &b, stream);
	if(rc != NB200_OK) return rc;
	launch_dependent(true, join_partials_kernel, dim3((q.rows + 31) / 32), dim3(256), 0, stream, static_cast<const float2*>(f.partial),
		p.nTiles * 2, q.rows, static_cast<const float*>(f.labelled), labels, q.vocabulary, loss, logSum);
	count_launch();
	return check_launch();
}

void sum_planes(const Problem& q, const float* planes, int count, int rows, const float* by, void* out, long long outRow, cudaStream_t stream)
{
	const long long ld = round_up(q.width, 8);
	const dim3 grid(grid_for(static_cast<long long>(rows) * ((q.width + 3) / 4), 256, 16));
	if(q.type == NB200_TYPE_BF16) {
		launch_dependent(true, sum_planes_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, planes, count, rows * ld, ld, rows, q.width, by,
			static_cast<__nv_bfloat16*>(out), outRow);
	} else {
		launch_dependent(true, sum_planes_kernel<__half>, grid, dim3(256), 0, stream, planes, count, rows * ld, ld, rows, q.width, by,
			static_cast<__half*>(out), outRow);
	}
	count_launch();
}

int backward16(const Problem& q, const float* lossDiff, const int* labels, const float* logSum, void* hiddenDiff, long long hiddenDiffRow,
	void* weightsDiff, long long weightsDiffRow, void* scratch, cudaStream_t stream)
{
	Room room = { static_cast<uint8_t*>(scratch) };
	const Backward16 w(q, room);
	const bool bf16 = q.type == NB200_TYPE_BF16;
	const int ld = round_up(q.width, 8);
	copy_rows(q.hidden, q.hiddenRow, q.rows, q.width, w.hidden, labels, lossDiff, q.vocabulary, w.scale, bf16 ? 0 : 1, stream);
	if(w.weights != nullptr) copy_rows(q.weights, q.weightsRow, q.vocabulary, q.width, w.weights, nullptr, nullptr, 0, nullptr, 0, stream);
	const void* const weights = w.weights ? w.weights : q.weights;
	const long long weightsRow = w.weights ? ld : q.weightsRow;
	CUtensorMap hidden, hiddenAcross, rows, across, diff, diffAcross;
	if(!product16_map(&hidden, w.hidden, bf16, q.width, q.rows, ld, PRODUCT16_BOX_A)
		|| !product16_map(&hiddenAcross, w.hidden, bf16, q.width, q.rows, ld, PRODUCT16_BOX_ACROSS)
		|| !product16_map(&rows, weights, bf16, q.width, q.vocabulary, weightsRow, PRODUCT16_BOX_B)
		|| !product16_map(&across, weights, bf16, q.width, q.vocabulary, weightsRow, PRODUCT16_BOX_ACROSS)
		|| !product16_map(&diff, w.diff, bf16, w.piece, q.rows, w.piece, PRODUCT16_BOX_A)
		|| !product16_map(&diffAcross, w.diff, bf16, w.piece, q.rows, w.piece, PRODUCT16_BOX_ACROSS)) return NB200_EINVAL;
	const int dTiles = (q.width + PRODUCT16_N - 1) / PRODUCT16_N, mTiles = (q.rows + PRODUCT16_M - 1) / PRODUCT16_M;
	for(int first = 0; first < q.vocabulary; first += w.piece) {
		const int columns = q.vocabulary - first < w.piece ? q.vocabulary - first : w.piece;
		Product16Params p = {};
		p.m = q.rows; p.n = columns;
		p.mTiles = mTiles;
		p.nTiles = (columns + PRODUCT16_N - 1) / PRODUCT16_N;
		p.splits = 1;
		p.kBlocks = p.kBlocksPerSplit = (q.width + PRODUCT16_K - 1) / PRODUCT16_K;
		p.mFast = 1; p.bf16 = bf16; p.status = device_status_word();
		p.bOffset = first;
		p.labels = labels; p.firstColumn = first; p.columns = q.vocabulary;
		p.logSum = logSum; p.rowScale = lossDiff; p.scale = w.scale;
		p.out16 = w.diff; p.ldOut = w.piece;
		int rc = product16(PRODUCT16_DIFF, false, false, p, &hidden, &rows, stream);
		if(rc != NB200_OK) return rc;
		if(hiddenDiff != nullptr) {
			p = {};
			p.m = q.rows; p.n = q.width;
			p.mTiles = mTiles; p.nTiles = dTiles; p.splits = w.hiddenSplits;
			// dz ends in zeros behind the vocabulary, up to a whole tile's columns
			p.kBlocks = (columns + PRODUCT16_K - 1) / PRODUCT16_K;
			p.kBlocksPerSplit = (p.kBlocks + p.splits - 1) / p.splits;
			p.bkOffset = first;
			p.mFast = 0; p.bf16 = bf16; p.status = device_status_word();
			p.plane = w.hiddenPlanes; p.ldPlane = ld; p.accumulate = first > 0;
			rc = product16(PRODUCT16_SUM, false, true, p, &diff, &across, stream);
			if(rc != NB200_OK) return rc;
		}
		if(weightsDiff != nullptr) {
			void* const out = static_cast<uint16_t*>(weightsDiff) + first * weightsDiffRow;
			p = {};
			p.m = columns; p.n = q.width;
			p.mTiles = (columns + PRODUCT16_M - 1) / PRODUCT16_M; p.nTiles = dTiles; p.splits = w.weightsSplits;
			p.kBlocks = (q.rows + PRODUCT16_K - 1) / PRODUCT16_K;
			p.kBlocksPerSplit = (p.kBlocks + p.splits - 1) / p.splits;
			p.mFast = 0; p.bf16 = bf16; p.status = device_status_word();
			if(p.splits > 1) {
				p.plane = w.weightsPlanes; p.ldPlane = ld;
				rc = product16(PRODUCT16_SUM, true, true, p, &diffAcross, &hiddenAcross, stream);
				if(rc != NB200_OK) return rc;
				sum_planes(q, w.weightsPlanes, p.splits, columns, w.scale + 1, out, weightsDiffRow, stream);
			} else {
				p.out16 = out; p.ldOut = weightsDiffRow; p.resultScale = w.scale + 1;
				rc = product16(PRODUCT16_STORE, true, true, p, &diffAcross, &hiddenAcross, stream);
				if(rc != NB200_OK) return rc;
			}
		}
	}
	if(hiddenDiff != nullptr) sum_planes(q, w.hiddenPlanes, w.hiddenSplits, q.rows, w.scale + 1, hiddenDiff, hiddenDiffRow, stream);
	return check_launch();
}

// A product of fp32 matrices of any depth, in parts of DEPTH that are added up in c.
int product32(const float* a, int m, int k, long long lda, const float* b, int n, long long ldb, float* c, long long ldc, float* product,
	int precision, cudaStream_t stream)
{
	for(int at = 0; at < k; at += DEPTH) {
		nb200_epilogue epilogue = {};
		epilogue.accumulate = at > 0;
		const int rc = nb200_multiply_matrix_by_transposed_matrix_with_scratch(stream, 1, a + at, m, k - at < DEPTH ? k - at : DEPTH,
			static_cast<int>(lda), b + at, n, static_cast<int>(ldb), c, static_cast<int>(ldc), product, &epilogue, precision);
		if(rc != NB200_OK) return rc;
	}
	return NB200_OK;
}

int logits32(const Problem& q, int first, int columns, float* z, float* product, int precision, cudaStream_t stream)
{
	return product32(static_cast<const float*>(q.hidden), q.rows, q.width, q.hiddenRow, static_cast<const float*>(q.weights) + first * q.weightsRow,
		columns, q.weightsRow, z, round_up(columns, 4), product, precision, stream);
}

int forward32(const Problem& q, const int* labels, float* loss, float* logSum, void* scratch, int precision, cudaStream_t stream)
{
	Room room = { static_cast<uint8_t*>(scratch) };
	const Forward32 f(q, room);
	for(int first = 0; first < q.vocabulary; first += f.piece) {
		const int columns = q.vocabulary - first < f.piece ? q.vocabulary - first : f.piece;
		const int rc = logits32(q, first, columns, f.z, f.product, precision, stream);
		if(rc != NB200_OK) return rc;
		fp32_stats_kernel<<<q.rows, 256, 0, stream>>>(f.z, round_up(columns, 4), columns, first, first == 0, first + columns == q.vocabulary, q.vocabulary,
			labels, f.running, f.labelled, loss, logSum);
		count_launch();
	}
	return check_launch();
}

dim3 squares(int rows, int columns)
{
	const int y = (rows + 31) / 32;
	return dim3((columns + 31) / 32, y < 65535 ? y : 65535);
}

int backward32(const Problem& q, const float* lossDiff, const int* labels, const float* logSum, float* hiddenDiff, long long hiddenDiffRow,
	float* weightsDiff, long long weightsDiffRow, void* scratch, int precision, cudaStream_t stream)
{
	Room room = { static_cast<uint8_t*>(scratch) };
	const Backward32 w(q, room);
	const int ldRows = round_up(q.rows, 4);
	if(weightsDiff != nullptr) {
		fp32_across_kernel<<<squares(q.rows, q.width), 256, 0, stream>>>(static_cast<const float*>(q.hidden), q.hiddenRow, q.rows, q.width, w.hiddenAcross,
			ldRows, 0, labels, lossDiff, q.vocabulary);
		count_launch();
	}
	for(int first = 0; first < q.vocabulary; first += w.piece) {
		const int columns = q.vocabulary - first < w.piece ? q.vocabulary - first : w.piece;
		const int parts = (columns + DEPTH - 1) / DEPTH;
		int rc = logits32(q, first, columns, w.z, w.product, precision, stream);
		if(rc != NB200_OK) return rc;
		fp32_diff_kernel<<<squares(q.rows, parts * DEPTH), 256, 0, stream>>>(w.z, round_up(columns, 4), q.rows, columns, first, q.vocabulary, labels,
			logSum, lossDiff, hiddenDiff != nullptr ? w.diffAlong : nullptr, weightsDiff != nullptr ? w.diffAcross : nullptr, ldRows);
		count_launch();
		if(hiddenDiff != nullptr) {
			fp32_across_kernel<<<squares(parts * DEPTH, q.width), 256, 0, stream>>>(static_cast<const float*>(q.weights) + first * q.weightsRow,
				q.weightsRow, columns, q.width, w.weightsAcross, DEPTH, DEPTH, nullptr, nullptr, 0);
			count_launch();
			const int ldPlane = round_up(q.width, 4);
			for(int part = 0; part < parts; part += w.parts) {
				const int batch = parts - part < w.parts ? parts - part : w.parts;
				rc = nb200_multiply_matrix_by_transposed_matrix_with_scratch(stream, batch, w.diffAlong + static_cast<long long>(part) * q.rows * DEPTH,
					q.rows, DEPTH, DEPTH, w.weightsAcross + static_cast<long long>(part) * q.width * DEPTH, q.width, DEPTH, w.planes, ldPlane, w.product,
					nullptr, precision);
				if(rc != NB200_OK) return rc;
				fp32_sum_kernel<<<grid_for(static_cast<long long>(q.rows) * q.width, 256, 16), 256, 0, stream>>>(w.planes, batch,
					static_cast<long long>(q.rows) * ldPlane, ldPlane, q.rows, q.width, hiddenDiff, hiddenDiffRow, first > 0 || part > 0);
				count_launch();
			}
		}
		if(weightsDiff != nullptr) {
			rc = product32(w.diffAcross, columns, q.rows, ldRows, w.hiddenAcross, q.width, ldRows, weightsDiff + first * weightsDiffRow, weightsDiffRow,
				w.product, precision, stream);
			if(rc != NB200_OK) return rc;
		}
	}
	return check_launch();
}

bool precision_valid(int precision)
{
	return precision == NB200_PREC_3XTF32 || precision == NB200_PREC_TF32 || precision == NB200_PREC_FP32_SIMT;
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
	if(type == NB200_TYPE_FP32) {
		if(backward) Backward32(q, room);
		else Forward32(q, room);
	} else {
		if(backward) Backward16(q, room);
		else Forward16(q, room);
	}
	return room.used;
}

int nb200_vocabulary_cross_entropy(void* stream, int type, const void* hidden, int rows, int width, long long hidden_row_size,
	const void* weights, int vocabulary, long long weights_row_size, const int* labels, float* loss, float* log_sum, void* scratch,
	int precision)
{
	const Problem q = { type, rows, width, vocabulary, hidden, weights, hidden_row_size, weights_row_size };
	if(!valid(q) || !precision_valid(precision)) return NB200_EINVAL;
	if(rows == 0) return NB200_OK;
	if(hidden == nullptr || weights == nullptr || labels == nullptr || loss == nullptr || log_sum == nullptr || !scratch_valid(scratch)) return NB200_EINVAL;
	if(too_big(q)) return NB200_ETOOBIG;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	return type == NB200_TYPE_FP32 ? forward32(q, labels, loss, log_sum, scratch, precision, as_stream(stream))
		: forward16(q, labels, loss, log_sum, scratch, as_stream(stream));
}

int nb200_vocabulary_cross_entropy_backward(void* stream, int type, const float* loss_diff, const void* hidden, int rows, int width,
	long long hidden_row_size, const void* weights, int vocabulary, long long weights_row_size, const int* labels, const float* log_sum,
	void* hidden_diff, long long hidden_diff_row_size, void* weights_diff, long long weights_diff_row_size, void* scratch, int precision)
{
	const Problem q = { type, rows, width, vocabulary, hidden, weights, hidden_row_size, weights_row_size };
	if(!valid(q) || !precision_valid(precision)) return NB200_EINVAL;
	if((hidden_diff != nullptr && hidden_diff_row_size < width) || (weights_diff != nullptr && weights_diff_row_size < width)
		|| !type_aligned(hidden_diff, type) || !type_aligned(weights_diff, type)) return NB200_EINVAL;
	if(hidden_diff == nullptr && weights_diff == nullptr) return NB200_OK;
	if(rows > 0 && (hidden == nullptr || weights == nullptr || labels == nullptr || loss_diff == nullptr || log_sum == nullptr
		|| !scratch_valid(scratch))) return NB200_EINVAL;
	if(too_big(q) || hidden_diff_row_size > 0x7fffffff || weights_diff_row_size > 0x7fffffff) return NB200_ETOOBIG;
	if(rows == 0 && weights_diff == nullptr) return NB200_OK;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	if(rows == 0) { // sums over no rows
		zero_rows_kernel<<<grid_for(vocabulary, 1, 16), 256, 0, as_stream(stream)>>>(static_cast<uint8_t*>(weights_diff),
			weights_diff_row_size * type_size(type), static_cast<long long>(width) * type_size(type), vocabulary);
		count_launch();
		return check_launch();
	}
	return type == NB200_TYPE_FP32
		? backward32(q, loss_diff, labels, log_sum, static_cast<float*>(hidden_diff), hidden_diff_row_size, static_cast<float*>(weights_diff),
			weights_diff_row_size, scratch, precision, as_stream(stream))
		: backward16(q, loss_diff, labels, log_sum, hidden_diff, hidden_diff_row_size, weights_diff, weights_diff_row_size, scratch,
			as_stream(stream));
}

} // extern "C"
