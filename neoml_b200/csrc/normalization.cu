// Layer normalisation of matrix rows, forward and backward.
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + epsilon), u = (x - m) r, y = u scale + free
//   g = dy scale:  dx = r (g - mean(g) - u mean(g u)),  dscale = sum over rows of dy u,  dfree = sum over rows of dy
//
// Both passes are bound by memory (forward: x in, y out; backward: x and dy in, dx out) as long as a row is read once, so
// a row lives in registers between its statistics and its result, the variance is taken of centred values (no
// cancellation), and the parameters of a thread's columns stay in registers for all the rows that it meets.
//
// A row is cut into 16-byte units of memory, whatever its first address: the units at both ends hold elements of the
// neighbouring rows too, which are left out of sums and stores (and a unit that would reach outside the matrix is read by
// elements).  A block's rows are a multiple of a whole unit's elements apart, so that all of them have the same
// alignment and a thread's columns never change.  Loads and stores of rows of odd width are whole units too then; what bounds
// those is the tests of every unit against the row's ends (16384 x 4096 bf16: 49 us forward, 5.5 TB/s; 40000 x 1031: 86 us, 1.9 TB/s).
// Operands whose rows are aligned differently from one another (a view of some columns) take the form with units of one element.
#include "types16.cuh"
#include <atomic>

namespace nb200 {

namespace {

constexpr int MAX_ROW_WARPS = 16; // of a block
constexpr int WIDE_THREADS = MAX_ROW_WARPS * 32; // of the blocks that loop over a row
constexpr int WIDE_BYTES = 200 * 1024; // and the shared memory that they stage a row in, at most
constexpr int SMALL_BLOCK = 128;  // threads of a block whose rows are a warp's or less: several rows at a time
constexpr int SMALL_WIDTH = 1024; // and what such a row holds at most

struct NormParams {
	const void* x;
	const void* dy;        // backward
	const void* scale;     // null: ones
	const void* free_term; // null: zeros
	void* out;             // y, dx
	float* mean;
	float* inv;
	float* partial;        // backward: [blocks][2][width]
	long long xRow, dyRow, outRow; // elements between rows
	int height, width;
	int lanes;             // threads that share a row: 4 to 32, or whole warps
	int rowStep;           // rows between two that a thread takes
	float epsilon;
};

// Sums over groups of `lanes` threads of a warp (32 and more: over the warp), several side by side.
template<int N>
__device__ __forceinline__ void lane_sums(float (&v)[N], int lanes)
{
	if(lanes >= 32) {
#pragma unroll
		for(int o = 16; o > 0; o >>= 1) {
#pragma unroll
			for(int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
		}
	} else {
		for(int o = lanes >> 1; o > 0; o >>= 1) {
#pragma unroll
			for(int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
		}
	}
}
__device__ __forceinline__ float lane_sum(float v, int lanes)
{
	float one[1] = { v };
	lane_sums<1>(one, lanes);
	return one[0];
}

// A unit's floats in pairs; the second of a unit of one element stays zero.
template<int V>
struct Pairs {
	static constexpr int N = V > 1 ? V / 2 : 1;
	float2 v[N];
};

template<typename T, int V, bool EDGES>
__device__ __forceinline__ void unit_pairs(const uint4& raw, int first, int width, Pairs<V>& out)
{
	float v[V > 1 ? V : 2];
	v[1] = 0.f;
	whole_floats<T, V, EDGES>(raw, first, width, v);
#pragma unroll
	for(int j = 0; j < Pairs<V>::N; ++j) out.v[j] = make_float2(v[2 * j], v[2 * j + 1]);
}

// Zeros where the unit is not the row's (units of one element: where the row has ended, and beside the element).
template<int V, bool EDGES>
__device__ __forceinline__ void clear_outside(int first, int width, Pairs<V>& p)
{
	if(V > 1 && whole<V, EDGES>(first, width)) return;
#pragma unroll
	for(int j = 0; j < Pairs<V>::N; ++j) {
		if(!inside<V, EDGES>(first, 2 * j, width)) p.v[j].x = 0.f;
		if(V == 1 || !inside<V, EDGES>(first, 2 * j + 1, width)) p.v[j].y = 0.f;
	}
}

// The parameters of a thread's columns.
template<typename P, int V, int C, bool EDGES>
__device__ __forceinline__ void load_parameters(const void* from, float missing, int t, int lanes, int offset, int width, Pairs<V> (&v)[C])
{
#pragma unroll
	for(int c = 0; c < C; ++c) {
		const int first = (c * lanes + t) * V - offset;
		auto one = [&](int j) {
			return from != nullptr && j < V && inside<V, EDGES>(first, j, width) ? to_float(static_cast<const P*>(from)[first + j]) : missing;
		};
#pragma unroll
		for(int j = 0; j < Pairs<V>::N; ++j) v[c].v[j] = make_float2(one(2 * j), one(2 * j + 1));
	}
}

// C units per thread, ROWS rows at a time (a row's sums are a chain of shuffles that leaves the SM idle: a second row fills it);
// the rows that follow are under way while these are worked on.
template<typename T, typename P, int V, int C, bool EDGES, int ROWS>
__global__ void __launch_bounds__(MAX_ROW_WARPS * 32) norm_forward_kernel(const NormParams p)
{
	__shared__ float4 joined[2][ROWS][MAX_ROW_WARPS];
	const int lanes = p.lanes;
	const int t = threadIdx.x & (lanes <= 32 ? lanes - 1 : 1023);
	const int rowsAtOnce = lanes <= 32 ? blockDim.x / lanes : 1;
	int r = blockIdx.x * rowsAtOnce + (lanes <= 32 ? threadIdx.x / lanes : 0);
	const T* const x = static_cast<const T*>(p.x);
	Row<T, V> row;
	row.begin = x;
	row.end = x + (p.height - 1) * p.xRow + p.width;
	const int offset = EDGES ? row_offset<T, V>(x + r * p.xRow) : 0;
	Pairs<V> scale[C], free[C];
	load_parameters<P, V, C, EDGES>(p.scale, 1.f, t, lanes, offset, p.width, scale);
	load_parameters<P, V, C, EDGES>(p.free_term, 0.f, t, lanes, offset, p.width, free);
	const float overWidth = 1.f / static_cast<float>(p.width);
	// the elements that this group of lanes holds of a row
	float count = 0.f;
#pragma unroll
	for(int c = 0; c < C; ++c) {
		const int first = (c * lanes + t) * V - offset;
#pragma unroll
		for(int j = 0; j < V; ++j) count += inside<V, EDGES>(first, j, p.width) ? 1.f : 0.f;
	}
	count = lane_sum(count, lanes);
	const float overCount = count > 0.f ? 1.f / count : 0.f;
	int phase = 0;
	uint4 next[ROWS][C];
	auto load = [&](int at) {
#pragma unroll
		for(int k = 0; k < ROWS; ++k) {
			// aligned rows: one behind the last is the last once more, and not stored
			const int at_k = at + k * p.rowStep;
			row.p = x + (EDGES ? at_k : min(at_k, p.height - 1)) * p.xRow;
#pragma unroll
			for(int c = 0; c < C; ++c) {
				next[k][c] = make_uint4(0u, 0u, 0u, 0u);
				if(!EDGES || at_k < p.height) load_unit<T, V, EDGES>(row, (c * lanes + t) * V - offset, p.width, next[k][c]);
			}
		}
	};
	load(r);
	// all threads of a warp stay to the end of its last row
	for(int left = r - (lanes <= 32 ? (threadIdx.x & 31) / lanes : 0); left < p.height; left += ROWS * p.rowStep, r += ROWS * p.rowStep) {
		Pairs<V> v[ROWS][C];
		float mean[ROWS], square[ROWS], groupMean[ROWS];
#pragma unroll
		for(int k = 0; k < ROWS; ++k) {
			float2 sums = both(0.f);
#pragma unroll
			for(int c = 0; c < C; ++c) {
				unit_pairs<T, V, EDGES>(next[k][c], (c * lanes + t) * V - offset, p.width, v[k][c]);
#pragma unroll
				for(int j = 0; j < Pairs<V>::N; ++j) sums = add2(sums, v[k][c].v[j]);
			}
			mean[k] = sums.x + sums.y;
		}
		load(r + ROWS * p.rowStep);
		// the mean of this group of lanes, and the squares around it; a row of several warps joins theirs:
		// squares around the row's mean = sum over the warps of (their squares + count (their mean - the row's)^2)
		lane_sums<ROWS>(mean, lanes);
#pragma unroll
		for(int k = 0; k < ROWS; ++k) {
			groupMean[k] = mean[k] *= overCount;
			float2 squares = both(0.f);
#pragma unroll
			for(int c = 0; c < C; ++c) {
#pragma unroll
				for(int j = 0; j < Pairs<V>::N; ++j) v[k][c].v[j] = add2(v[k][c].v[j], both(-mean[k]));
				clear_outside<V, EDGES>((c * lanes + t) * V - offset, p.width, v[k][c]);
#pragma unroll
				for(int j = 0; j < Pairs<V>::N; ++j) squares = fma2(v[k][c].v[j], v[k][c].v[j], squares);
			}
			square[k] = squares.x + squares.y;
		}
		lane_sums<ROWS>(square, lanes);
		if(lanes > 32) {
			if((threadIdx.x & 31) == 0) {
#pragma unroll
				for(int k = 0; k < ROWS; ++k) joined[phase][k][threadIdx.x >> 5] = make_float4(mean[k], square[k], count, 0.f);
			}
			__syncthreads(); // one for these rows: the slots alternate
			const int w = threadIdx.x & (MAX_ROW_WARPS - 1);
			float4 o[ROWS];
#pragma unroll
			for(int k = 0; k < ROWS; ++k) {
				o[k] = w < (lanes >> 5) ? joined[phase][k][w] : make_float4(0.f, 0.f, 0.f, 0.f);
				mean[k] = o[k].x * o[k].z;
			}
			lane_sums<ROWS>(mean, MAX_ROW_WARPS);
#pragma unroll
			for(int k = 0; k < ROWS; ++k) {
				mean[k] *= overWidth;
				square[k] = fmaf((o[k].x - mean[k]) * (o[k].x - mean[k]), o[k].z, o[k].y);
			}
			lane_sums<ROWS>(square, MAX_ROW_WARPS);
			phase ^= 1;
		}
#pragma unroll
		for(int k = 0; k < ROWS; ++k) {
			const int at = r + k * p.rowStep;
			if(at >= p.height) continue;
			const float inv = rsqrtf(square[k] * overWidth + p.epsilon);
			T* const out = static_cast<T*>(p.out) + at * p.outRow;
			const float2 shift = both(groupMean[k] - mean[k]), by = both(inv);
#pragma unroll
			for(int c = 0; c < C; ++c) {
				float y[V > 1 ? V : 2];
#pragma unroll
				for(int j = 0; j < Pairs<V>::N; ++j) {
					const float2 f = fma2(mul2(add2(v[k][c].v[j], shift), by), scale[c].v[j], free[c].v[j]);
					y[2 * j] = f.x;
					y[2 * j + 1] = f.y;
				}
				store_unit<T, V, EDGES>(out, (c * lanes + t) * V - offset, p.width, y);
			}
			if(t == 0) {
				if(p.mean != nullptr) p.mean[at] = mean[k];
				if(p.inv != nullptr) p.inv[at] = inv;
			}
		}
	}
}

// Sum over a block of WIDE_THREADS threads; every one of them gets it.  Two calls in a row use different slots.
__device__ __forceinline__ float block_sum(float v, float* slots)
{
	v = warp_sum_all(v);
	if((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
	__syncthreads();
	return warp_sum_all((threadIdx.x & 31) < WIDE_THREADS / 32 ? slots[threadIdx.x & 31] : 0.f);
}

// Units of a row in shared memory where it fits (STAGED), or read again out of L2.
template<typename T, int V, bool STAGED>
struct WideRow {
	Row<T, V> row;
	uint4* staged;
	int offset, width, units;
	__device__ __forceinline__ void set(const T* x, long long rowSize, int r, uint4* room, int w)
	{
		row.p = x + r * rowSize;
		staged = room;
		width = w;
		offset = row_offset<T, V>(row.p);
		units = (w + offset + V - 1) / V;
	}
	// f(first column, the unit's pairs), the first time or again
	template<bool AGAIN, typename F>
	__device__ __forceinline__ void each(F&& f) const
	{
		constexpr int AHEAD = 4;
		for(int u0 = threadIdx.x; u0 < units; u0 += WIDE_THREADS * AHEAD) {
			uint4 raw[AHEAD];
#pragma unroll
			for(int k = 0; k < AHEAD; ++k) {
				const int u = u0 + k * WIDE_THREADS;
				if(u >= units) continue;
				if(STAGED && AGAIN) raw[k] = staged[u];
				else load_unit<T, V>(row, u * V - offset, width, raw[k]);
			}
#pragma unroll
			for(int k = 0; k < AHEAD; ++k) {
				const int u = u0 + k * WIDE_THREADS;
				if(u >= units) continue;
				if(STAGED && !AGAIN) staged[u] = raw[k];
				Pairs<V> v;
				unit_pairs<T, V, true>(raw[k], u * V - offset, width, v);
				f(u * V - offset, v);
			}
		}
	}
};

// The parameters of a unit's columns: whole vectors where the columns are aligned for it.
template<typename P, int V>
__device__ __forceinline__ void unit_parameters(const void* from, int first, int width, float missing, float* v)
{
	const P* const at = static_cast<const P*>(from) + first;
	if(V > 1 && from != nullptr && first >= 0 && first + V <= width && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
#pragma unroll
		for(int k = 0; k < V / Unit16<P>::N; ++k) Unit16<P>::unpack(reinterpret_cast<const uint4*>(at)[k], v + k * Unit16<P>::N);
	} else {
#pragma unroll
		for(int j = 0; j < V; ++j) v[j] = from != nullptr && first + j >= 0 && first + j < width ? to_float(at[j]) : missing;
	}
}

// Rows longer than a block's registers hold.
template<typename T, typename P, int V, bool STAGED>
__global__ void __launch_bounds__(WIDE_THREADS) norm_forward_wide_kernel(const NormParams p)
{
	extern __shared__ uint4 wideRoom[];
	__shared__ float slots[2][MAX_ROW_WARPS];
	const T* const x = static_cast<const T*>(p.x);
	WideRow<T, V, STAGED> row;
	row.row.begin = x;
	row.row.end = x + (p.height - 1) * p.xRow + p.width;
	const float overWidth = 1.f / static_cast<float>(p.width);
	for(int r = blockIdx.x; r < p.height; r += gridDim.x) {
		row.set(x, p.xRow, r, wideRoom, p.width);
		float2 sums = both(0.f), squares = both(0.f);
		row.template each<false>([&](int, const Pairs<V>& v) {
#pragma unroll
			for(int j = 0; j < Pairs<V>::N; ++j) sums = add2(sums, v.v[j]);
		});
		const float mean = block_sum(sums.x + sums.y, slots[0]) * overWidth;
		row.template each<true>([&](int first, const Pairs<V>& v) {
			Pairs<V> d;
#pragma unroll
			for(int j = 0; j < Pairs<V>::N; ++j) d.v[j] = add2(v.v[j], both(-mean));
			clear_outside<V, true>(first, p.width, d);
#pragma unroll
			for(int j = 0; j < Pairs<V>::N; ++j) squares = fma2(d.v[j], d.v[j], squares);
		});
		const float inv = rsqrtf(block_sum(squares.x + squares.y, slots[1]) * overWidth + p.epsilon);
		T* const out = static_cast<T*>(p.out) + r * p.outRow;
		row.template each<true>([&](int first, const Pairs<V>& v) {
			float y[V > 1 ? V : 2], scale[V], free[V];
			unit_parameters<P, V>(p.scale, first, p.width, 1.f, scale);
			unit_parameters<P, V>(p.free_term, first, p.width, 0.f, free);
#pragma unroll
			for(int j = 0; j < V; ++j) y[j] = fmaf(((j % 2 == 0 ? v.v[j / 2].x : v.v[j / 2].y) - mean) * inv, scale[j], free[j]);
			store_unit<T, V>(out, first, p.width, y);
		});
		if(threadIdx.x == 0) {
			if(p.mean != nullptr) p.mean[r] = mean;
			if(p.inv != nullptr) p.inv[r] = inv;
		}
		// a unit is staged again, and rewritten in place, by the thread that read it: no barrier
	}
}

// Backward.  A thread's sums of dy u and dy stay in registers over all its rows; a block's go to `partial` once.
template<typename T, typename P, int V, int C, bool EDGES>
__global__ void __launch_bounds__(MAX_ROW_WARPS * 32) norm_backward_kernel(const NormParams p)
{
	__shared__ float2 joined[2][MAX_ROW_WARPS];
	__shared__ float sums[2][SMALL_WIDTH];
	const int lanes = p.lanes;
	const int t = threadIdx.x & (lanes <= 32 ? lanes - 1 : 1023);
	const int rowsAtOnce = lanes <= 32 ? blockDim.x / lanes : 1;
	int r = blockIdx.x * rowsAtOnce + (lanes <= 32 ? threadIdx.x / lanes : 0);
	const T* const x = static_cast<const T*>(p.x);
	const T* const dy = static_cast<const T*>(p.dy);
	Row<T, V> xr, dr;
	xr.begin = x;
	xr.end = x + (p.height - 1) * p.xRow + p.width;
	dr.begin = dy;
	dr.end = dy + (p.height - 1) * p.dyRow + p.width;
	const int offset = EDGES ? row_offset<T, V>(x + r * p.xRow) : 0;
	Pairs<V> scale[C], ds[C], db[C];
	load_parameters<P, V, C, EDGES>(p.scale, 1.f, t, lanes, offset, p.width, scale);
#pragma unroll
	for(int c = 0; c < C; ++c) {
#pragma unroll
		for(int j = 0; j < Pairs<V>::N; ++j) ds[c].v[j] = db[c].v[j] = both(0.f);
	}
	const float overWidth = 1.f / static_cast<float>(p.width);
	int phase = 0;
	uint4 nextX[C], nextD[C];
	float nextMean = 0.f, nextInv = 0.f;
	auto load = [&](int at) {
		xr.p = x + at * p.xRow;
		dr.p = dy + at * p.dyRow;
#pragma unroll
		for(int c = 0; c < C; ++c) {
			nextX[c] = nextD[c] = make_uint4(0u, 0u, 0u, 0u);
			if(at < p.height) {
				load_unit<T, V, EDGES>(xr, (c * lanes + t) * V - offset, p.width, nextX[c]);
				load_unit<T, V, EDGES>(dr, (c * lanes + t) * V - offset, p.width, nextD[c]);
			}
		}
		if(at < p.height) {
			nextMean = __ldg(p.mean + at);
			nextInv = __ldg(p.inv + at);
		}
	};
	load(r);
	for(int left = r - (lanes <= 32 ? (threadIdx.x & 31) / lanes : 0); left < p.height; left += p.rowStep, r += p.rowStep, phase ^= 1) {
		const float mean = nextMean, inv = nextInv;
		Pairs<V> u[C], g[C]; // unit rows; gradients times scale
		float2 sumsG = both(0.f), sumsGu = both(0.f);
#pragma unroll
		for(int c = 0; c < C; ++c) {
			const int first = (c * lanes + t) * V - offset;
			unit_pairs<T, V, EDGES>(nextX[c], first, p.width, u[c]); // the neighbours' may be infinite
			unit_pairs<T, V, EDGES>(nextD[c], first, p.width, g[c]); // zeros outside, and so is what they are multiplied by
#pragma unroll
			for(int j = 0; j < Pairs<V>::N; ++j) {
				u[c].v[j] = mul2(add2(u[c].v[j], both(-mean)), both(inv));
				ds[c].v[j] = fma2(g[c].v[j], u[c].v[j], ds[c].v[j]);
				db[c].v[j] = add2(db[c].v[j], g[c].v[j]);
				g[c].v[j] = mul2(g[c].v[j], scale[c].v[j]);
				sumsG = add2(sumsG, g[c].v[j]);
				sumsGu = fma2(g[c].v[j], u[c].v[j], sumsGu);
			}
		}
		load(r + p.rowStep);
		float sumG = sumsG.x + sumsG.y, sumGu = sumsGu.x + sumsGu.y;
		float two[2] = { sumG, sumGu };
		lane_sums<2>(two, lanes);
		sumG = two[0];
		sumGu = two[1];
		if(lanes > 32) {
			if((threadIdx.x & 31) == 0) joined[phase][threadIdx.x >> 5] = make_float2(sumG, sumGu);
			__syncthreads(); // one a row: the slots alternate
			const int w = threadIdx.x & (MAX_ROW_WARPS - 1);
			const float2 o = w < (lanes >> 5) ? joined[phase][w] : make_float2(0.f, 0.f);
			two[0] = o.x;
			two[1] = o.y;
			lane_sums<2>(two, MAX_ROW_WARPS);
			sumG = two[0];
			sumGu = two[1];
		}
		if(r < p.height) {
			const float meanG = sumG * overWidth, meanGu = sumGu * overWidth;
			T* const out = static_cast<T*>(p.out) + r * p.outRow;
#pragma unroll
			for(int c = 0; c < C; ++c) {
				float y[V > 1 ? V : 2];
#pragma unroll
				for(int j = 0; j < Pairs<V>::N; ++j) {
					const float2 f = mul2(fma2(u[c].v[j], both(-meanGu), add2(g[c].v[j], both(-meanG))), both(inv));
					y[2 * j] = f.x;
					y[2 * j + 1] = f.y;
				}
				store_unit<T, V, EDGES>(out, (c * lanes + t) * V - offset, p.width, y);
			}
		}
	}
	if(p.partial == nullptr) return;
	float* const mine = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.width;
	// rows that are worked on at the same time add up in turn
	for(int g = 0; g < rowsAtOnce; ++g) {
		if(rowsAtOnce == 1 || threadIdx.x / lanes == g) {
#pragma unroll
			for(int c = 0; c < C; ++c) {
				const int first = (c * lanes + t) * V - offset;
#pragma unroll
				for(int j = 0; j < V; ++j) {
					if(!inside<V, EDGES>(first, j, p.width)) continue;
					const int column = first + j;
					if(rowsAtOnce == 1) {
						mine[column] = j % 2 == 0 ? ds[c].v[j / 2].x : ds[c].v[j / 2].y;
						mine[p.width + column] = j % 2 == 0 ? db[c].v[j / 2].x : db[c].v[j / 2].y;
					} else {
						sums[0][column] = (g > 0 ? sums[0][column] : 0.f) + (j % 2 == 0 ? ds[c].v[j / 2].x : ds[c].v[j / 2].y);
						sums[1][column] = (g > 0 ? sums[1][column] : 0.f) + (j % 2 == 0 ? db[c].v[j / 2].x : db[c].v[j / 2].y);
					}
				}
			}
		}
		if(rowsAtOnce > 1) __syncthreads();
	}
	if(rowsAtOnce > 1) {
		for(int i = threadIdx.x; i < 2 * p.width; i += blockDim.x) mine[i] = i < p.width ? sums[0][i] : sums[1][i - p.width];
	}
}

// Rows longer than a block's registers hold: dx here, the parameters' sums in a kernel of their own (which reads both again).
template<typename T, typename P, int V, bool STAGED>
__global__ void __launch_bounds__(WIDE_THREADS) norm_backward_wide_kernel(const NormParams p)
{
	extern __shared__ uint4 wideRoom[];
	__shared__ float slots[2][2][MAX_ROW_WARPS];
	const T* const x = static_cast<const T*>(p.x);
	const T* const dy = static_cast<const T*>(p.dy);
	WideRow<T, V, STAGED> row, diff;
	row.row.begin = x;
	row.row.end = x + (p.height - 1) * p.xRow + p.width;
	diff.row.begin = dy;
	diff.row.end = dy + (p.height - 1) * p.dyRow + p.width;
	const float overWidth = 1.f / static_cast<float>(p.width);
	const int room = (p.width + 2 * V - 1) / V + 1;
	int phase = 0;
	for(int r = blockIdx.x; r < p.height; r += gridDim.x, phase ^= 1) {
		row.set(x, p.xRow, r, wideRoom, p.width);
		diff.set(dy, p.dyRow, r, wideRoom + room, p.width);
		const float mean = __ldg(p.mean + r), inv = __ldg(p.inv + r);
		// both rows are cut alike; f(first column, gradients times scale, unit rows)
		auto each = [&](bool again, auto f) {
			constexpr int AHEAD = 2;
			for(int u0 = threadIdx.x; u0 < row.units; u0 += WIDE_THREADS * AHEAD) {
				uint4 rx[AHEAD], rd[AHEAD];
#pragma unroll
				for(int k = 0; k < AHEAD; ++k) {
					const int u = u0 + k * WIDE_THREADS;
					if(u >= row.units) continue;
					if(STAGED && again) {
						rx[k] = row.staged[u];
						rd[k] = diff.staged[u];
					} else {
						load_unit<T, V>(row.row, u * V - row.offset, p.width, rx[k]);
						load_unit<T, V>(diff.row, u * V - row.offset, p.width, rd[k]);
					}
				}
#pragma unroll
				for(int k = 0; k < AHEAD; ++k) {
					const int u = u0 + k * WIDE_THREADS, first = u * V - row.offset;
					if(u >= row.units) continue;
					if(STAGED && !again) {
						row.staged[u] = rx[k];
						diff.staged[u] = rd[k];
					}
					Pairs<V> vx, vd;
					unit_pairs<T, V, true>(rx[k], first, p.width, vx);
					unit_pairs<T, V, true>(rd[k], first, p.width, vd);
					float g[V > 1 ? V : 2], unit[V > 1 ? V : 2], scale[V];
					unit_parameters<P, V>(p.scale, first, p.width, 1.f, scale);
#pragma unroll
					for(int j = 0; j < V; ++j) {
						g[j] = (j % 2 == 0 ? vd.v[j / 2].x : vd.v[j / 2].y) * scale[j];
						unit[j] = ((j % 2 == 0 ? vx.v[j / 2].x : vx.v[j / 2].y) - mean) * inv;
					}
					f(first, g, unit);
				}
			}
		};
		float sumG = 0.f, sumGu = 0.f;
		each(false, [&](int, const float* g, const float* unit) {
#pragma unroll
			for(int j = 0; j < V; ++j) {
				sumG += g[j];
				sumGu = fmaf(g[j], unit[j], sumGu);
			}
		});
		const float meanG = block_sum(sumG, slots[phase][0]) * overWidth;
		const float meanGu = block_sum(sumGu, slots[phase][1]) * overWidth;
		T* const out = static_cast<T*>(p.out) + r * p.outRow;
		each(true, [&](int first, float* g, const float* unit) {
#pragma unroll
			for(int j = 0; j < V; ++j) g[j] = ((g[j] - meanG) - unit[j] * meanGu) * inv;
			store_unit<T, V>(out, first, p.width, g);
		});
	}
}

// The sums of dy u and dy over a slice of the rows, a thread per column (two of 16 bits where rows are aligned for it).
template<typename T, int W>
__global__ void __launch_bounds__(256) norm_sums_kernel(const NormParams p)
{
	const int column = (blockIdx.x * 256 + threadIdx.x) * W;
	if(column >= p.width) return;
	const T* const x = static_cast<const T*>(p.x) + column;
	const T* const dy = static_cast<const T*>(p.dy) + column;
	float ds[W], db[W];
#pragma unroll
	for(int w = 0; w < W; ++w) ds[w] = db[w] = 0.f;
#pragma unroll 8
	for(int r = blockIdx.y; r < p.height; r += gridDim.y) {
		const float mean = __ldg(p.mean + r), inv = __ldg(p.inv + r);
		float vx[W], vd[W];
		if constexpr(W == 2) {
			const float2 a = unpack2<T>(*reinterpret_cast<const uint32_t*>(x + r * p.xRow)), b = unpack2<T>(*reinterpret_cast<const uint32_t*>(dy + r * p.dyRow));
			vx[0] = a.x; vx[1] = a.y; vd[0] = b.x; vd[1] = b.y;
		} else {
			vx[0] = to_float(x[r * p.xRow]);
			vd[0] = to_float(dy[r * p.dyRow]);
		}
#pragma unroll
		for(int w = 0; w < W; ++w) {
			ds[w] = fmaf(vd[w], (vx[w] - mean) * inv, ds[w]);
			db[w] += vd[w];
		}
	}
	float* const mine = p.partial + static_cast<long long>(blockIdx.y) * 2 * p.width;
#pragma unroll
	for(int w = 0; w < W; ++w) {
		mine[column + w] = ds[w];
		mine[p.width + column + w] = db[w];
	}
}

// dscale and dfree from the blocks' sums, added in block order.  A block has 32 columns; its 16 warps take every 16th
// partial row each.
template<typename P>
__global__ void __launch_bounds__(512) norm_parameters_kernel(const float* __restrict__ partial, int parts, int width,
	P* __restrict__ scaleDiff, P* __restrict__ freeDiff)
{
	__shared__ float sums[16][33];
	dependent_wait();
	const int which = blockIdx.y;
	const int column = blockIdx.x * 32 + (threadIdx.x & 31);
	const int lane = threadIdx.x >> 5;
	float s = 0.f;
	if(column < width) {
		const float* const at = partial + static_cast<long long>(which) * width + column;
#pragma unroll 8
		for(int i = lane; i < parts; i += 16) s += at[static_cast<long long>(i) * 2 * width];
	}
	sums[lane][threadIdx.x & 31] = s;
	__syncthreads();
	if(lane == 0 && column < width) {
		s = 0.f;
#pragma unroll
		for(int i = 0; i < 16; ++i) s += sums[i][threadIdx.x];
		P* const out = which == 0 ? scaleDiff : freeDiff;
		if(out != nullptr) out[column] = from_float<P>(s);
	}
}

template<typename P>
__global__ void __launch_bounds__(256) zero_parameters_kernel(P* a, P* b, int width)
{
	for(int i = blockIdx.x * blockDim.x + threadIdx.x; i < width; i += gridDim.x * blockDim.x) {
		if(a != nullptr) a[i] = from_float<P>(0.f);
		if(b != nullptr) b[i] = from_float<P>(0.f);
	}
}

// How a call is cut up; the same for the scratch size and the launch.
struct Shape {
	bool wide;      // rows longer than registers hold
	int unit;       // elements of a unit
	bool edges;     // rows may begin or end inside a unit
	int units;      // per thread: 1 to 4, 6 or 8, or 8 units of one element
	int lanes;      // threads of a row
	int threads;    // per block
	int rowsAtOnce; // of a block
	int blocks;
};

// A thread holds 16 elements (forward: 24 of 16 bits in a row that is one warp's, 32 in rows that are too long for MAX_ROW_WARPS
// warps otherwise): more of them, with the parameters or sums beside them, would not stay in registers.
// Rows of at most 32 lanes need no barrier.  Longer ones take the fewest threads, then the fewest warps, that hold them.
Shape shape_of(int type, int height, int width, bool alike, bool aligned, bool forward)
{
	Shape s = {};
	const int size = type_size(type);
	s.unit = alike ? 16 / size : 1;
	s.edges = !aligned || width % s.unit != 0;
	// a row that begins inside a unit touches one more
	const int units = alike && !aligned ? (width + 2 * (s.unit - 1)) / s.unit : (width + s.unit - 1) / s.unit;
	const int most = alike ? 16 / s.unit : 8;
	if(units <= 32 * (forward && alike && size == 2 ? 3 : most) && width <= SMALL_WIDTH) {
		s.lanes = 32;
		while(s.lanes > 4 && units <= s.lanes / 2) s.lanes /= 2;
		s.threads = SMALL_BLOCK;
		s.rowsAtOnce = SMALL_BLOCK / s.lanes;
		s.units = alike ? (units + s.lanes - 1) / s.lanes : 8;
	} else {
		int hold = units > MAX_ROW_WARPS * 32 * most && forward && alike ? 2 * most : most;
		auto warps_for = [&](int h) { return (units + 32 * h - 1) / (32 * h); };
		s.wide = warps_for(hold) > MAX_ROW_WARPS;
		if(alike && !s.wide) { // a thread's share of a row's sums costs about as much as 1.7 units; more than 24 elements do not stay in registers
			auto cost = [&](int h) { return warps_for(h) * (17 + 10 * h) * (h * s.unit > 24 ? 3 : 2); };
			for(int h = hold - 1; h >= 1 && warps_for(h) <= MAX_ROW_WARPS; --h) {
				if(cost(h) < cost(hold)) hold = h;
			}
		}
		s.threads = s.lanes = (s.wide ? MAX_ROW_WARPS : warps_for(hold)) * 32;
		s.rowsAtOnce = 1;
		s.units = alike ? (units + s.lanes - 1) / s.lanes : 8;
	}
	// at most: the launch goes by what fits (launch_rows)
	if(s.wide) { // of the parameters' sums: slices of the rows, eight blocks per SM with those side by side
		const int across = (width + 511) / 512, slices = (sm_count() * 8 + across - 1) / across;
		s.blocks = height < slices ? height : slices;
		return s;
	}
	const int most_blocks = sm_count() * (1024 / s.threads > 1 ? 1024 / s.threads : 1) + s.unit;
	const int wanted = (height + s.rowsAtOnce - 1) / s.rowsAtOnce;
	s.blocks = wanted < most_blocks ? wanted : most_blocks / s.unit * s.unit;
	return s;
}

struct Operand {
	const void* p;
	long long row;
};

// all operands' rows begin at the same offset from a 16-byte boundary, row by row
bool aligned_alike(int type, int height, const Operand* o, int n)
{
	const int size = type_size(type);
	for(int i = 1; i < n; ++i) {
		if(((reinterpret_cast<uintptr_t>(o[i].p) ^ reinterpret_cast<uintptr_t>(o[0].p)) & 15u) != 0) return false;
		if(height > 1 && ((o[i].row - o[0].row) * size & 15) != 0) return false;
	}
	return true;
}

// Every operand's rows all begin on a 16-byte boundary.
bool all_aligned(int type, int height, const Operand* o, int n)
{
	for(int i = 0; i < n; ++i) {
		if(!aligned16(o[i].p) || (height > 1 && (o[i].row * type_size(type) & 15) != 0)) return false;
	}
	return true;
}

using Kernel = void (*)(const NormParams);

// Blocks of a kernel that the device holds at a time; asked once per kernel and block size.
template<Kernel KERNEL>
int resident_blocks(int threads)
{
	static std::atomic<int> known[MAX_ROW_WARPS + 1];
	std::atomic<int>& slot = known[threads / 32];
	int perSm = slot.load(std::memory_order_relaxed);
	if(perSm == 0) {
		if(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&perSm, KERNEL, threads, 0) != cudaSuccess || perSm < 1) perSm = 1;
		slot.store(perSm, std::memory_order_relaxed);
	}
	return perSm * sm_count();
}

// Launches as many blocks of the shape as are resident; returns their number.
template<Kernel KERNEL>
int launch_rows(NormParams p, const Shape& s, cudaStream_t stream)
{
	int blocks = s.blocks;
	const int resident = resident_blocks<KERNEL>(s.threads);
	if(blocks > resident) {
		// a block's rows are a multiple of a unit's elements apart: all of them begin at the same offset in a unit
		blocks = resident;
		while(blocks * s.rowsAtOnce % s.unit != 0) --blocks;
	}
	p.rowStep = blocks * s.rowsAtOnce;
	KERNEL<<<blocks, s.threads, 0, stream>>>(p);
	return blocks;
}

// Two rows at a time where a thread has as many; `units` above 16 elements leave no registers for it.
template<typename T, typename P, int V, int C, bool EDGES>
void launch_forward_rows(const NormParams& p, const Shape& s, cudaStream_t stream)
{
	if(V * C <= 16 && p.height > s.blocks * s.rowsAtOnce) launch_rows<norm_forward_kernel<T, P, V, C, EDGES, V * C <= 16 ? 2 : 1>>(p, s, stream);
	else launch_rows<norm_forward_kernel<T, P, V, C, EDGES, 1>>(p, s, stream);
}

template<typename T, typename P, bool EDGES>
void launch_forward_units(const NormParams& p, const Shape& s, cudaStream_t stream)
{
	constexpr int V = Unit16<T>::N;
	if(s.units <= 1) launch_forward_rows<T, P, V, 1, EDGES>(p, s, stream);
	else if(s.units == 2) launch_forward_rows<T, P, V, 2, EDGES>(p, s, stream);
	else if(s.units == 3) launch_forward_rows<T, P, V, 3, EDGES>(p, s, stream);
	else if(s.units == 4) launch_forward_rows<T, P, V, 4, EDGES>(p, s, stream);
	else if constexpr(V == 4) {
		if(s.units <= 6) launch_forward_rows<T, P, V, 6, EDGES>(p, s, stream);
		else launch_forward_rows<T, P, V, 8, EDGES>(p, s, stream);
	}
}

// Blocks of a kernel for long rows: two on an SM where their shared memory allows it.
template<Kernel STAGED, Kernel AGAIN>
void launch_wide(const NormParams& p, long long bytes, cudaStream_t stream)
{
	const int most = sm_count() * (bytes > 100 * 1024 && bytes <= WIDE_BYTES ? 1 : 2);
	const int blocks = p.height < most ? p.height : most;
	if(bytes <= WIDE_BYTES) {
		cudaFuncSetAttribute(STAGED, cudaFuncAttributeMaxDynamicSharedMemorySize, WIDE_BYTES);
		STAGED<<<blocks, WIDE_THREADS, static_cast<size_t>(bytes), stream>>>(p);
	} else {
		AGAIN<<<blocks, WIDE_THREADS, 0, stream>>>(p);
	}
}

template<typename T, typename P, int V>
void launch_forward_wide(const NormParams& p, cudaStream_t stream)
{
	const long long bytes = ((p.width + 2ll * V - 1) / V + 1) * 16;
	launch_wide<norm_forward_wide_kernel<T, P, V, true>, norm_forward_wide_kernel<T, P, V, false>>(p, bytes, stream);
}

template<typename T, typename P, int V>
void launch_backward_wide(const NormParams& p, int slices, cudaStream_t stream)
{
	if(p.partial != nullptr) { // first: dx may take the place of dy or x
		const bool pairs = sizeof(T) == 2 && p.width % 2 == 0 && p.xRow % 2 == 0 && p.dyRow % 2 == 0
			&& ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.dy)) & 3u) == 0;
		constexpr int W = sizeof(T) == 2 ? 2 : 1;
		const int perBlock = pairs ? 256 * W : 256;
		const dim3 grid((p.width + perBlock - 1) / perBlock, slices);
		if(pairs) norm_sums_kernel<T, W><<<grid, 256, 0, stream>>>(p);
		else norm_sums_kernel<T, 1><<<grid, 256, 0, stream>>>(p);
		count_launch();
	}
	const long long bytes = 2 * ((p.width + 2ll * V - 1) / V + 1) * 16;
	launch_wide<norm_backward_wide_kernel<T, P, V, true>, norm_backward_wide_kernel<T, P, V, false>>(p, bytes, stream);
}

template<typename T, typename P>
void launch_forward(const NormParams& p, const Shape& s, cudaStream_t stream)
{
	if(s.wide) s.unit == 1 ? launch_forward_wide<T, P, 1>(p, stream) : launch_forward_wide<T, P, Unit16<T>::N>(p, stream);
	else if(s.unit == 1) launch_forward_rows<T, P, 1, 8, true>(p, s, stream);
	else if(s.edges) launch_forward_units<T, P, true>(p, s, stream);
	else launch_forward_units<T, P, false>(p, s, stream);
}

template<typename T, typename P, bool EDGES>
int launch_backward_units(const NormParams& p, const Shape& s, cudaStream_t stream)
{
	constexpr int V = Unit16<T>::N;
	if(s.units <= 1) return launch_rows<norm_backward_kernel<T, P, V, 1, EDGES>>(p, s, stream);
	if constexpr(V == 4) {
		if(s.units == 3) return launch_rows<norm_backward_kernel<T, P, V, 3, EDGES>>(p, s, stream);
		if(s.units == 4) return launch_rows<norm_backward_kernel<T, P, V, 4, EDGES>>(p, s, stream);
	}
	return launch_rows<norm_backward_kernel<T, P, V, 2, EDGES>>(p, s, stream);
}

template<typename T, typename P>
void launch_backward(const NormParams& p, const Shape& s, void* scaleDiff, void* freeDiff, cudaStream_t stream)
{
	int blocks = s.blocks;
	if(s.wide) s.unit == 1 ? launch_backward_wide<T, P, 1>(p, blocks, stream) : launch_backward_wide<T, P, Unit16<T>::N>(p, blocks, stream);
	else if(s.unit == 1) blocks = launch_rows<norm_backward_kernel<T, P, 1, 8, true>>(p, s, stream);
	else if(s.edges) blocks = launch_backward_units<T, P, true>(p, s, stream);
	else blocks = launch_backward_units<T, P, false>(p, s, stream);
	count_launch();
	if(p.partial != nullptr) {
		const dim3 grid((p.width + 31) / 32, 2);
		launch_dependent(true, norm_parameters_kernel<P>, grid, dim3(512), 0, stream, static_cast<const float*>(p.partial),
			blocks, p.width, static_cast<P*>(scaleDiff), static_cast<P*>(freeDiff));
		count_launch();
	}
}

// Calls f with values of the element and the parameter type; parameters are of the rows' type or fp32.
template<typename F>
void with_types(int type, int parameterType, F&& f)
{
	if(type == NB200_TYPE_FP32) f(float(), float());
	else if(type == NB200_TYPE_FP16) parameterType == NB200_TYPE_FP32 ? f(__half(), float()) : f(__half(), __half());
	else parameterType == NB200_TYPE_FP32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
}

bool sizes_valid(int type, int parameterType, int height, int width)
{
	return type_valid(type) && (parameterType == type || parameterType == NB200_TYPE_FP32) && height >= 0 && width >= 1;
}

} // namespace

} // namespace nb200

using namespace nb200;

extern "C" {

int nb200_layer_normalization(void* stream, int type, int parameter_type, const void* x, int height, int width,
	long long x_row_size, const void* scale, const void* free_term, float epsilon, void* y, long long y_row_size, float* mean,
	float* inverse_deviation)
{
	if(!sizes_valid(type, parameter_type, height, width) || x_row_size < width || y_row_size < width) return NB200_EINVAL;
	if(height == 0) return NB200_OK;
	if(height > (1 << 30) || width > (1 << 30)) return NB200_ETOOBIG;
	if(x == nullptr || y == nullptr || !type_aligned(x, type) || !type_aligned(y, type)
		|| !type_aligned(scale, parameter_type) || !type_aligned(free_term, parameter_type)
		|| !words_aligned(mean, inverse_deviation)) return NB200_EINVAL;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	const Operand operands[] = { { x, x_row_size }, { y, y_row_size } };
	const Shape s = shape_of(type, height, width, aligned_alike(type, height, operands, 2), all_aligned(type, height, operands, 2), true);
	NormParams p = {};
	p.x = x; p.scale = scale; p.free_term = free_term; p.out = y; p.mean = mean; p.inv = inverse_deviation;
	p.xRow = x_row_size; p.outRow = y_row_size;
	p.height = height; p.width = width; p.lanes = s.lanes; p.epsilon = epsilon;
	with_types(type, parameter_type, [&](auto t, auto q) { launch_forward<decltype(t), decltype(q)>(p, s, as_stream(stream)); });
	count_launch();
	return check_launch();
}

size_t nb200_layer_normalization_backward_scratch_floats(int type, int height, int width)
{
	if(!type_valid(type) || height <= 0 || width <= 0 || height > (1 << 30) || width > (1 << 30)) return 0;
	// whichever form the operands' alignment selects
	int blocks = 0;
	for(int form = 0; form < 3; ++form) {
		const int n = shape_of(type, height, width, form > 0, form > 1, false).blocks;
		if(n > blocks) blocks = n;
	}
	return static_cast<size_t>(blocks) * 2 * width;
}

int nb200_layer_normalization_backward(void* stream, int type, int parameter_type, const void* dy, long long dy_row_size,
	const void* x, int height, int width, long long x_row_size, const void* scale, const float* mean,
	const float* inverse_deviation, void* dx, long long dx_row_size, void* scale_diff, void* free_term_diff, float* scratch)
{
	if(!sizes_valid(type, parameter_type, height, width) || x_row_size < width || dy_row_size < width || dx_row_size < width) {
		return NB200_EINVAL;
	}
	const bool parameters = scale_diff != nullptr || free_term_diff != nullptr;
	if(!type_aligned(scale, parameter_type) || !type_aligned(scale_diff, parameter_type)
		|| !type_aligned(free_term_diff, parameter_type) || !words_aligned(mean, inverse_deviation, scratch)) return NB200_EINVAL;
	if(height > 0 && (x == nullptr || dy == nullptr || dx == nullptr || mean == nullptr || inverse_deviation == nullptr
		|| !type_aligned(x, type) || !type_aligned(dy, type) || !type_aligned(dx, type)
		|| (parameters && scratch == nullptr))) return NB200_EINVAL;
	if(height == 0 && !parameters) return NB200_OK;
	if(height > (1 << 30) || width > (1 << 30)) return NB200_ETOOBIG;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	if(height == 0) { // sums over no rows
		const int grid = grid_for(width, 256);
		with_types(type, parameter_type, [&](auto, auto q) {
			using P = decltype(q);
			zero_parameters_kernel<P><<<grid, 256, 0, as_stream(stream)>>>(static_cast<P*>(scale_diff), static_cast<P*>(free_term_diff), width);
		});
		count_launch();
		return check_launch();
	}
	const Operand operands[] = { { x, x_row_size }, { dy, dy_row_size }, { dx, dx_row_size } };
	const Shape s = shape_of(type, height, width, aligned_alike(type, height, operands, 3), all_aligned(type, height, operands, 3), false);
	NormParams p = {};
	p.x = x; p.dy = dy; p.scale = scale; p.out = dx;
	p.mean = const_cast<float*>(mean); p.inv = const_cast<float*>(inverse_deviation);
	p.partial = parameters ? scratch : nullptr;
	p.xRow = x_row_size; p.dyRow = dy_row_size; p.outRow = dx_row_size;
	p.height = height; p.width = width; p.lanes = s.lanes;
	with_types(type, parameter_type, [&](auto t, auto q) {
		launch_backward<decltype(t), decltype(q)>(p, s, scale_diff, free_term_diff, as_stream(stream));
	});
	return check_launch();
}

} // extern "C"
