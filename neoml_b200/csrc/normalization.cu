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
// alignment and a thread's columns never change.  This is why rows of odd width run at the same rate as even ones.
// Operands whose rows are aligned differently from one another (a view of some columns) take the form with units of one element.
#include "types16.cuh"

namespace nb200 {

namespace {

constexpr int MAX_WARPS = 32;     // of the kernels that loop over a row
constexpr int MAX_ROW_WARPS = 16; // of those that hold it: 128 registers a thread
constexpr int ROWS_PER_WARP_BLOCK = 4; // rows at a time of a block whose warps have a row each

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
	int height, width, warpsPerRow;
	int rowStep;           // rows between two that a warp (or a block) takes
	float epsilon;
};

// Sum over the threads that share a row; every one of them gets it.  `slots` holds a float per warp; the two calls of a
// row use different ones, so that one barrier each is enough.
__device__ __forceinline__ float row_sum(float v, int warps, float* slots)
{
	v = warp_sum_all(v);
	if(warps == 1) return v;
	if((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
	__syncthreads();
	float s = (threadIdx.x & 31) < warps ? slots[threadIdx.x & 31] : 0.f;
	return warp_sum_all(s);
}

// C units per thread.  A row per block of warpsPerRow warps, or (warpsPerRow == 1) a row per warp.
template<typename T, typename P, int V, int C>
__global__ void __launch_bounds__(MAX_ROW_WARPS * 32) norm_forward_kernel(const NormParams p)
{
	__shared__ float slots[2][MAX_WARPS];
	const int warps = p.warpsPerRow;
	const int lanes = warps * 32;
	const int t = warps == 1 ? threadIdx.x & 31 : threadIdx.x;
	int r = warps == 1 ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
	if(r >= p.height) return; // a whole warp, or a whole block
	const T* const x = static_cast<const T*>(p.x);
	Row<T, V> row;
	row.begin = x;
	row.end = x + (p.height - 1) * p.xRow + p.width;
	const int offset = row_offset<T, V>(x + r * p.xRow);
	float scale[C][V], free[C][V];
#pragma unroll
	for(int c = 0; c < C; ++c) {
		const int first = (c * lanes + t) * V - offset;
#pragma unroll
		for(int j = 0; j < V; ++j) {
			const bool in = inside<V>(first, j, p.width);
			scale[c][j] = in && p.scale != nullptr ? to_float(static_cast<const P*>(p.scale)[first + j]) : 1.f;
			free[c][j] = in && p.free_term != nullptr ? to_float(static_cast<const P*>(p.free_term)[first + j]) : 0.f;
		}
	}
	const float overWidth = 1.f / static_cast<float>(p.width);
	for(; r < p.height; r += p.rowStep) {
		row.p = x + r * p.xRow;
		uint4 raw[C];
#pragma unroll
		for(int c = 0; c < C; ++c) load_unit<T, V>(row, (c * lanes + t) * V - offset, p.width, raw[c]);
		float sum = 0.f;
#pragma unroll
		for(int c = 0; c < C; ++c) {
			const int first = (c * lanes + t) * V - offset;
			float v[V];
			unit_floats<T, V>(raw[c], v);
#pragma unroll
			for(int j = 0; j < V; ++j) sum += inside<V>(first, j, p.width) ? v[j] : 0.f;
		}
		const float mean = row_sum(sum, warps, slots[0]) * overWidth;
		float square = 0.f;
#pragma unroll
		for(int c = 0; c < C; ++c) {
			const int first = (c * lanes + t) * V - offset;
			float v[V];
			unit_floats<T, V>(raw[c], v);
#pragma unroll
			for(int j = 0; j < V; ++j) {
				const float d = inside<V>(first, j, p.width) ? v[j] - mean : 0.f;
				square = fmaf(d, d, square);
			}
		}
		const float inv = rsqrtf(row_sum(square, warps, slots[1]) * overWidth + p.epsilon);
		T* const out = static_cast<T*>(p.out) + r * p.outRow;
#pragma unroll
		for(int c = 0; c < C; ++c) {
			const int first = (c * lanes + t) * V - offset;
			float v[V];
			unit_floats<T, V>(raw[c], v);
#pragma unroll
			for(int j = 0; j < V; ++j) v[j] = fmaf((v[j] - mean) * inv, scale[c][j], free[c][j]);
			store_unit<T, V>(out, first, p.width, v);
		}
		if(t == 0) {
			if(p.mean != nullptr) p.mean[r] = mean;
			if(p.inv != nullptr) p.inv[r] = inv;
		}
	}
}

// Rows longer than a block's registers hold: three passes over the row, the second and third out of L2.
template<typename T, typename P>
__global__ void __launch_bounds__(1024) norm_forward_wide_kernel(const NormParams p)
{
	__shared__ float slots[2][MAX_WARPS];
	const float overWidth = 1.f / static_cast<float>(p.width);
	for(int r = blockIdx.x; r < p.height; r += gridDim.x) {
		const T* const x = static_cast<const T*>(p.x) + r * p.xRow;
		T* const out = static_cast<T*>(p.out) + r * p.outRow;
		float sum = 0.f;
		for(int i = threadIdx.x; i < p.width; i += blockDim.x) sum += to_float(x[i]);
		const float mean = row_sum(sum, MAX_WARPS, slots[0]) * overWidth;
		float square = 0.f;
		for(int i = threadIdx.x; i < p.width; i += blockDim.x) {
			const float d = to_float(x[i]) - mean;
			square = fmaf(d, d, square);
		}
		const float inv = rsqrtf(row_sum(square, MAX_WARPS, slots[1]) * overWidth + p.epsilon);
		for(int i = threadIdx.x; i < p.width; i += blockDim.x) {
			const float s = p.scale != nullptr ? to_float(static_cast<const P*>(p.scale)[i]) : 1.f;
			const float b = p.free_term != nullptr ? to_float(static_cast<const P*>(p.free_term)[i]) : 0.f;
			out[i] = from_float<T>(fmaf((to_float(x[i]) - mean) * inv, s, b));
		}
		if(threadIdx.x == 0) {
			if(p.mean != nullptr) p.mean[r] = mean;
			if(p.inv != nullptr) p.inv[r] = inv;
		}
		// every element of this thread's columns has been read by the thread that rewrites it: in place needs no barrier
	}
}

// Backward.  A block's sums of dy u and dy stay in registers over all its rows and go to `partial` once.
template<typename T, typename P, int V, int C>
__global__ void __launch_bounds__(MAX_ROW_WARPS * 32) norm_backward_kernel(const NormParams p)
{
	__shared__ float slots[2][2][MAX_WARPS];
	const int warps = p.warpsPerRow;
	const int lanes = warps * 32;
	const int t = warps == 1 ? threadIdx.x & 31 : threadIdx.x;
	int r = warps == 1 ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
	const T* const x = static_cast<const T*>(p.x);
	const T* const dy = static_cast<const T*>(p.dy);
	Row<T, V> xr, dr;
	xr.begin = x;
	xr.end = x + (p.height - 1) * p.xRow + p.width;
	dr.begin = dy;
	dr.end = dy + (p.height - 1) * p.dyRow + p.width;
	const int offset = row_offset<T, V>(x + (r < p.height ? r : 0) * p.xRow);
	float scale[C][V], ds[C][V], db[C][V];
#pragma unroll
	for(int c = 0; c < C; ++c) {
		const int first = (c * lanes + t) * V - offset;
#pragma unroll
		for(int j = 0; j < V; ++j) {
			scale[c][j] = inside<V>(first, j, p.width) && p.scale != nullptr ? to_float(static_cast<const P*>(p.scale)[first + j]) : 1.f;
			ds[c][j] = db[c][j] = 0.f;
		}
	}
	const float overWidth = 1.f / static_cast<float>(p.width);
	int phase = 0;
	for(; r < p.height; r += p.rowStep, phase ^= 1) {
		xr.p = x + r * p.xRow;
		dr.p = dy + r * p.dyRow;
		uint4 rx[C], rd[C];
#pragma unroll
		for(int c = 0; c < C; ++c) {
			load_unit<T, V>(xr, (c * lanes + t) * V - offset, p.width, rx[c]);
			load_unit<T, V>(dr, (c * lanes + t) * V - offset, p.width, rd[c]);
		}
		const float mean = __ldg(p.mean + r), inv = __ldg(p.inv + r);
		float sumG = 0.f, sumGu = 0.f;
#pragma unroll
		for(int c = 0; c < C; ++c) {
			const int first = (c * lanes + t) * V - offset;
			float u[V], g[V];
			unit_floats<T, V>(rx[c], u);
			unit_floats<T, V>(rd[c], g);
#pragma unroll
			for(int j = 0; j < V; ++j) {
				const bool in = inside<V>(first, j, p.width);
				const float d = in ? g[j] : 0.f, unit = in ? (u[j] - mean) * inv : 0.f;
				ds[c][j] = fmaf(d, unit, ds[c][j]);
				db[c][j] += d;
				const float by = d * scale[c][j];
				sumG += by;
				sumGu = fmaf(by, unit, sumGu);
			}
		}
		sumG = warp_sum_all(sumG);
		sumGu = warp_sum_all(sumGu);
		if(warps > 1) {
			if((threadIdx.x & 31) == 0) {
				slots[phase][0][threadIdx.x >> 5] = sumG;
				slots[phase][1][threadIdx.x >> 5] = sumGu;
			}
			__syncthreads(); // one a row: the slots alternate
			const int w = threadIdx.x & 31;
			sumG = warp_sum_all(w < warps ? slots[phase][0][w] : 0.f);
			sumGu = warp_sum_all(w < warps ? slots[phase][1][w] : 0.f);
		}
		const float meanG = sumG * overWidth, meanGu = sumGu * overWidth;
		T* const out = static_cast<T*>(p.out) + r * p.outRow;
#pragma unroll
		for(int c = 0; c < C; ++c) {
			const int first = (c * lanes + t) * V - offset;
			float u[V], g[V];
			unit_floats<T, V>(rx[c], u);
			unit_floats<T, V>(rd[c], g);
#pragma unroll
			for(int j = 0; j < V; ++j) {
				const float unit = (u[j] - mean) * inv;
				g[j] = (fmaf(g[j], scale[c][j], -meanG) - unit * meanGu) * inv;
			}
			store_unit<T, V>(out, first, p.width, g);
		}
	}
	if(p.partial == nullptr) return;
	// one row of partial sums per block; the warps that had rows of their own write one each
	float* const mine = p.partial + static_cast<long long>(warps == 1 ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x) * 2 * p.width;
#pragma unroll
	for(int c = 0; c < C; ++c) {
		const int first = (c * lanes + t) * V - offset;
#pragma unroll
		for(int j = 0; j < V; ++j) {
			if(inside<V>(first, j, p.width)) {
				mine[first + j] = ds[c][j];
				mine[p.width + first + j] = db[c][j];
			}
		}
	}
}

// Rows longer than a block's registers hold: sums, then dx, out of L2.
template<typename T, typename P>
__global__ void __launch_bounds__(1024) norm_backward_wide_kernel(const NormParams p)
{
	__shared__ float slots[2][2][MAX_WARPS];
	const float overWidth = 1.f / static_cast<float>(p.width);
	int phase = 0;
	float* const mine = p.partial == nullptr ? nullptr : p.partial + static_cast<long long>(blockIdx.x) * 2 * p.width;
	bool started = false;
	for(int r = blockIdx.x; r < p.height; r += gridDim.x, phase ^= 1) {
		const T* const x = static_cast<const T*>(p.x) + r * p.xRow;
		const T* const dy = static_cast<const T*>(p.dy) + r * p.dyRow;
		T* const out = static_cast<T*>(p.out) + r * p.outRow;
		const float mean = __ldg(p.mean + r), inv = __ldg(p.inv + r);
		float sumG = 0.f, sumGu = 0.f;
		for(int i = threadIdx.x; i < p.width; i += blockDim.x) {
			const float unit = (to_float(x[i]) - mean) * inv, d = to_float(dy[i]);
			const float by = d * (p.scale != nullptr ? to_float(static_cast<const P*>(p.scale)[i]) : 1.f);
			sumG += by;
			sumGu = fmaf(by, unit, sumGu);
			if(mine != nullptr) { // a column belongs to one thread
				mine[i] = started ? fmaf(d, unit, mine[i]) : d * unit;
				mine[p.width + i] = started ? mine[p.width + i] + d : d;
			}
		}
		started = true;
		const float meanG = row_sum(sumG, MAX_WARPS, slots[phase][0]) * overWidth;
		const float meanGu = row_sum(sumGu, MAX_WARPS, slots[phase][1]) * overWidth;
		for(int i = threadIdx.x; i < p.width; i += blockDim.x) {
			const float unit = (to_float(x[i]) - mean) * inv;
			const float s = p.scale != nullptr ? to_float(static_cast<const P*>(p.scale)[i]) : 1.f;
			out[i] = from_float<T>((fmaf(to_float(dy[i]), s, -meanG) - unit * meanGu) * inv);
		}
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
	int units;      // per thread: 1, 2, 4 (or 16 units of one element)
	int warps;      // per row
	int threads;    // per block
	int rowsAtOnce; // of a block
	int blocks;
	int parts() const { return wide || warps > 1 ? blocks : blocks * rowsAtOnce; }
};

// `most`: elements a thread may hold.  Few enough warps that a block's barriers cost little, enough threads that the
// device is filled: the fewest warps per row whose threads hold the row.
Shape shape_of(int type, int height, int width, bool alike, int most)
{
	Shape s = {};
	const int whole = alike ? 16 / type_size(type) : 1;
	s.unit = whole;
	const int units = (width + whole - 1) / whole + (whole > 1 ? 1 : 0); // the row may begin inside a unit
	const int unitsPerThread = alike ? most / whole : 16;
	s.warps = 1;
	while(s.warps < MAX_ROW_WARPS && static_cast<long long>(s.warps) * 32 * unitsPerThread < units) s.warps *= 2;
	const int perThread = (units + s.warps * 32 - 1) / (s.warps * 32);
	s.wide = perThread > unitsPerThread;
	if(s.wide) {
		s.warps = MAX_WARPS;
		s.threads = 1024;
		s.rowsAtOnce = 1;
		s.blocks = height < sm_count() * 2 ? height : sm_count() * 2;
		return s;
	}
	s.units = alike ? (perThread <= 1 ? 1 : perThread <= 2 ? 2 : perThread <= 4 ? 4 : 8) : 16;
	s.rowsAtOnce = s.warps == 1 ? ROWS_PER_WARP_BLOCK : 1;
	s.threads = s.warps * 32 * s.rowsAtOnce;
	// a block's rows are a multiple of a unit's elements apart
	const long long wanted = (static_cast<long long>(height) + s.rowsAtOnce - 1) / s.rowsAtOnce;
	long long resident = static_cast<long long>(sm_count()) * (1024 / s.threads > 0 ? 1024 / s.threads : 1);
	if(wanted > resident) {
		while(resident * s.rowsAtOnce % whole != 0) ++resident;
		s.blocks = static_cast<int>(resident);
	} else {
		s.blocks = static_cast<int>(wanted);
	}
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

template<typename T, typename P>
void launch_forward(const NormParams& p, const Shape& s, cudaStream_t stream)
{
	constexpr int V = Unit16<T>::N;
	if(s.wide) norm_forward_wide_kernel<T, P><<<s.blocks, s.threads, 0, stream>>>(p);
	else if(s.unit == 1) norm_forward_kernel<T, P, 1, 16><<<s.blocks, s.threads, 0, stream>>>(p);
	else if(s.units == 1) norm_forward_kernel<T, P, V, 1><<<s.blocks, s.threads, 0, stream>>>(p);
	else if(s.units == 2) norm_forward_kernel<T, P, V, 2><<<s.blocks, s.threads, 0, stream>>>(p);
	else if(s.units == 4) norm_forward_kernel<T, P, V, 4><<<s.blocks, s.threads, 0, stream>>>(p);
	else if constexpr(V == 4) norm_forward_kernel<T, P, V, 8><<<s.blocks, s.threads, 0, stream>>>(p);
}

template<typename T, typename P>
void launch_backward(const NormParams& p, const Shape& s, void* scaleDiff, void* freeDiff, cudaStream_t stream)
{
	constexpr int V = Unit16<T>::N;
	if(s.wide) norm_backward_wide_kernel<T, P><<<s.blocks, s.threads, 0, stream>>>(p);
	else if(s.unit == 1) norm_backward_kernel<T, P, 1, 16><<<s.blocks, s.threads, 0, stream>>>(p);
	else if(s.units == 1) norm_backward_kernel<T, P, V, 1><<<s.blocks, s.threads, 0, stream>>>(p);
	else if(s.units == 2) norm_backward_kernel<T, P, V, 2><<<s.blocks, s.threads, 0, stream>>>(p);
	else if constexpr(V == 4) norm_backward_kernel<T, P, V, 4><<<s.blocks, s.threads, 0, stream>>>(p);
	count_launch();
	if(p.partial != nullptr) {
		const dim3 grid((p.width + 31) / 32, 2);
		launch_dependent(true, norm_parameters_kernel<P>, grid, dim3(512), 0, stream, static_cast<const float*>(p.partial),
			s.parts(), p.width, static_cast<P*>(scaleDiff), static_cast<P*>(freeDiff));
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

constexpr int FORWARD_ELEMENTS = 32, BACKWARD_ELEMENTS = 16; // registers: three floats an element there, one more sum here

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
	if(x == nullptr || y == nullptr || !type_aligned(x, type) || !type_aligned(y, type)
		|| !type_aligned(scale, parameter_type) || !type_aligned(free_term, parameter_type)) return NB200_EINVAL;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	const Operand operands[] = { { x, x_row_size }, { y, y_row_size } };
	const Shape s = shape_of(type, height, width, aligned_alike(type, height, operands, 2), FORWARD_ELEMENTS);
	NormParams p = {};
	p.x = x; p.scale = scale; p.free_term = free_term; p.out = y; p.mean = mean; p.inv = inverse_deviation;
	p.xRow = x_row_size; p.outRow = y_row_size;
	p.height = height; p.width = width; p.warpsPerRow = s.warps; p.rowStep = s.blocks * s.rowsAtOnce; p.epsilon = epsilon;
	with_types(type, parameter_type, [&](auto t, auto q) { launch_forward<decltype(t), decltype(q)>(p, s, as_stream(stream)); });
	count_launch();
	return check_launch();
}

size_t nb200_layer_normalization_backward_scratch_floats(int type, int height, int width)
{
	if(!type_valid(type) || height <= 0 || width <= 0) return 0;
	// whichever form the operands' alignment selects
	const int a = shape_of(type, height, width, true, BACKWARD_ELEMENTS).parts();
	const int b = shape_of(type, height, width, false, BACKWARD_ELEMENTS).parts();
	return static_cast<size_t>(a > b ? a : b) * 2 * width;
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
		|| !type_aligned(free_term_diff, parameter_type)) return NB200_EINVAL;
	if(height > 0 && (x == nullptr || dy == nullptr || dx == nullptr || mean == nullptr || inverse_deviation == nullptr
		|| !type_aligned(x, type) || !type_aligned(dy, type) || !type_aligned(dx, type)
		|| (parameters && scratch == nullptr))) return NB200_EINVAL;
	if(height == 0 && !parameters) return NB200_OK;
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
	const Shape s = shape_of(type, height, width, aligned_alike(type, height, operands, 3), BACKWARD_ELEMENTS);
	NormParams p = {};
	p.x = x; p.dy = dy; p.scale = scale; p.out = dx;
	p.mean = const_cast<float*>(mean); p.inv = const_cast<float*>(inverse_deviation);
	p.partial = parameters ? scratch : nullptr;
	p.xRow = x_row_size; p.dyRow = dy_row_size; p.outRow = dx_row_size;
	p.height = height; p.width = width; p.warpsPerRow = s.warps; p.rowStep = s.blocks * s.rowsAtOnce;
	with_types(type, parameter_type, [&](auto t, auto q) {
		launch_backward<decltype(t), decltype(q)>(p, s, scale_diff, free_term_diff, as_stream(stream));
	});
	return check_launch();
}

} // extern "C"
