// Distillation from a teacher's top logits: a student's logits [rows][V] against K kept logits of each row's teacher.
//
//   p = softmax(teacher / tau) over the kept entries, q = softmax(logits / tau) over all V
//   loss = tau^2 sum_k p_k (log p_k - log q_k),   d logits = tau dloss (q - p)
//
// Bound by memory: the forward pass reads the logits once (running maximum and sum), the backward pass reads and writes
// them once.  Rows move in aligned 16-byte units whatever their width (types16.cuh).  Few rows are split: into a cluster's blocks that
// join their sums through distributed shared memory, and backward simply into more blocks.
#include "types16.cuh"
#include <cooperative_groups.h>

namespace nb200 {

namespace {

namespace cg = cooperative_groups;

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int KEPT_MAX = NB200_DISTILLATION_KEPT_MAX;
constexpr int MAX_PARTS = 8;
constexpr int UNROLL = 4;      // units in flight per thread
constexpr float LOG2E = 1.4426950408889634f;

struct DistillParams {
	const void* logits;
	const void* teacher;   // [rows][kept]
	const int* indices;    // [rows][kept]
	const float* lossDiff; // backward
	float* logSum;
	float* loss;
	void* out;             // backward: gradient of the logits
	long long row, outRow;
	int vocabulary, kept;
	int parts;             // blocks of a row
	float temperature;
};

// Maximum and the sum of 2^(x - maximum).
struct Running {
	float top, sum;
	__device__ __forceinline__ void join(const Running& o)
	{
		const float t = fmaxf(top, o.top);
		const float at = t == -INFINITY ? 0.f : t;
		sum = sum * exp2f(top - at) + o.sum * exp2f(o.top - at);
		top = t;
	}
};

__device__ __forceinline__ float block_sum(float v, float* slots)
{
	v = warp_sum_all(v);
	__syncthreads(); // slots of the call before
	if((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
	__syncthreads();
	return warp_sum_all((threadIdx.x & 31) < WARPS ? slots[threadIdx.x & 31] : 0.f);
}
__device__ __forceinline__ float block_max(float v, float* slots)
{
	v = warp_max_all(v);
	__syncthreads();
	if((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
	__syncthreads();
	return warp_max_all((threadIdx.x & 31) < WARPS ? slots[threadIdx.x & 31] : -INFINITY);
}

struct Kept {
	float p[KEPT_MAX];  // the teacher's probabilities; zero for entries that are not used
	float z[KEPT_MAX];  // the student's logit
	int at[KEPT_MAX];   // column, -1 for entries that are not used
};

// The teacher's probabilities of a row.  An index outside the vocabulary marks an entry that is not used.  False: no entry is.
template<typename T, typename P>
__device__ __forceinline__ bool teacher_row(const DistillParams& p, int r, const T* logits, Kept& kept, float* slots)
{
	const P* const teacher = static_cast<const P*>(p.teacher) + static_cast<long long>(r) * p.kept;
	const int* const indices = p.indices + static_cast<long long>(r) * p.kept;
	const float c = LOG2E / p.temperature;
	float top = -INFINITY, any = 0.f;
	for(int k = threadIdx.x; k < p.kept; k += THREADS) {
		const int at = __ldg(indices + k);
		const bool used = at >= 0 && at < p.vocabulary;
		const float x = used ? to_float(teacher[k]) * c : -INFINITY;
		kept.at[k] = used ? at : -1;
		kept.z[k] = used ? to_float(logits[at]) : 0.f;
		kept.p[k] = x;
		if(used) any = 1.f;
		top = fmaxf(top, x);
	}
	top = block_max(top, slots);
	any = block_max(any, slots);
	const float reference = top == -INFINITY ? 0.f : top;
	float sum = 0.f;
	for(int k = threadIdx.x; k < p.kept; k += THREADS) {
		const float e = exp2f(kept.p[k] - reference);
		kept.p[k] = e;
		sum += e;
	}
	sum = block_sum(sum, slots);
	if(any == 0.f || sum == 0.f) return false; // a row whose teacher kept nothing, or nothing but minus infinity
	const float over = 1.f / sum;
	for(int k = threadIdx.x; k < p.kept; k += THREADS) kept.p[k] *= over;
	return true;
}

template<typename T, typename P, int V>
__global__ void __launch_bounds__(THREADS) distillation_forward_kernel(const DistillParams p)
{
	__shared__ Kept kept;
	__shared__ float slots[WARPS];
	__shared__ Running parts[MAX_PARTS];
	__shared__ Running warpsOf[WARPS];
	const int blocks = p.parts, r = blockIdx.x / blocks, rank = blockIdx.x - r * blocks;
	if(blocks > 1) cg::this_cluster().sync(); // the others' shared memory exists from here on
	const T* const x = static_cast<const T*>(p.logits) + r * p.row;
	const int offset = row_offset<T, V>(x);
	const int units = (p.vocabulary + offset + V - 1) / V;
	const int perBlock = (units + blocks - 1) / blocks;
	const int end = min(units, (rank + 1) * perBlock);
	const float c = LOG2E / p.temperature;
	Row<T, V> row;
	row.p = x;
	row.begin = x;                     // no element of another row is touched
	row.end = x + p.vocabulary;
	Running mine = { -INFINITY, 0.f };
	for(int u0 = rank * perBlock; u0 < end; u0 += THREADS * UNROLL) {
		uint4 raw[UNROLL];
#pragma unroll
		for(int k = 0; k < UNROLL; ++k) {
			const int u = u0 + k * THREADS + threadIdx.x;
			raw[k] = make_uint4(0u, 0u, 0u, 0u);
			if(u < end) load_unit<T, V>(row, u * V - offset, p.vocabulary, raw[k]);
		}
		float top = mine.top;
		float v[UNROLL][V];
#pragma unroll
		for(int k = 0; k < UNROLL; ++k) {
			const int u = u0 + k * THREADS + threadIdx.x, first = u * V - offset;
			unit_floats<T, V>(raw[k], v[k]);
			const bool whole = u < end && first >= 0 && first + V <= p.vocabulary;
#pragma unroll
			for(int j = 0; j < V; ++j) {
				v[k][j] = whole || (u < end && inside<V>(first, j, p.vocabulary)) ? v[k][j] * c : -INFINITY;
				top = fmaxf(top, v[k][j]);
			}
		}
		const float at = top == -INFINITY ? 0.f : top;
		mine.sum *= exp2f(mine.top - at);
#pragma unroll
		for(int k = 0; k < UNROLL; ++k) {
#pragma unroll
			for(int j = 0; j < V; ++j) mine.sum += exp2f(v[k][j] - at);
		}
		mine.top = top;
	}
#pragma unroll
	for(int o = 16; o > 0; o >>= 1) {
		const Running other = { __shfl_xor_sync(0xffffffffu, mine.top, o), __shfl_xor_sync(0xffffffffu, mine.sum, o) };
		mine.join(other);
	}
	if((threadIdx.x & 31) == 0) warpsOf[threadIdx.x >> 5] = mine;
	__syncthreads();
	mine = warpsOf[0];
#pragma unroll
	for(int w = 1; w < WARPS; ++w) mine.join(warpsOf[w]);
	if(blocks > 1) {
		cg::cluster_group cluster = cg::this_cluster();
		if(threadIdx.x == 0) *cluster.map_shared_rank(&parts[rank], 0) = mine;
		cluster.sync();
		if(rank != 0) return;
		mine = parts[0];
		for(int k = 1; k < blocks; ++k) mine.join(parts[k]);
	}
	// mine.top is in units of log 2
	const float logSum = mine.top / LOG2E + logf(mine.sum);
	const bool used = teacher_row<T, P>(p, r, x, kept, slots);
	float sum = 0.f;
	if(used) {
		for(int k = threadIdx.x; k < p.kept; k += THREADS) {
			const float q = kept.p[k];
			if(kept.at[k] >= 0 && !(q == 0.f)) sum += q * (logf(q) - (kept.z[k] / p.temperature - logSum));
		}
	}
	sum = block_sum(sum, slots);
	if(threadIdx.x == 0) {
		p.logSum[r] = logSum;
		p.loss[r] = used ? p.temperature * p.temperature * sum : 0.f;
	}
}

template<typename T, typename P, int V>
__global__ void __launch_bounds__(THREADS) distillation_backward_kernel(const DistillParams p)
{
	__shared__ Kept kept;
	__shared__ float slots[WARPS];
	const int blocks = p.parts, r = blockIdx.x / blocks, rank = blockIdx.x - r * blocks;
	const T* const x = static_cast<const T*>(p.logits) + r * p.row;
	T* const out = static_cast<T*>(p.out) + r * p.outRow;
	const int offset = row_offset<T, V>(x);
	const int units = (p.vocabulary + offset + V - 1) / V;
	const int perBlock = (units + blocks - 1) / blocks;
	const int begin = rank * perBlock, end = min(units, begin + perBlock);
	const float c = LOG2E / p.temperature;
	// the student's kept logits are read here, before anything is written: the gradient may replace the logits
	const bool used = teacher_row<T, P>(p, r, x, kept, slots);
	const float by = used ? p.temperature * __ldg(p.lossDiff + r) : 0.f;
	const float log2Sum = __ldg(p.logSum + r) * LOG2E;
	__syncthreads();
	Row<T, V> row;
	row.p = x;
	row.begin = x;
	row.end = x + p.vocabulary;
	for(int u0 = begin; u0 < end; u0 += THREADS * UNROLL) {
		uint4 raw[UNROLL];
#pragma unroll
		for(int k = 0; k < UNROLL; ++k) {
			const int u = u0 + k * THREADS + threadIdx.x;
			if(u < end) load_unit<T, V>(row, u * V - offset, p.vocabulary, raw[k]);
		}
#pragma unroll
		for(int k = 0; k < UNROLL; ++k) {
			const int u = u0 + k * THREADS + threadIdx.x;
			if(u >= end) continue;
			float v[V];
			unit_floats<T, V>(raw[k], v);
#pragma unroll
			for(int j = 0; j < V; ++j) v[j] = used ? by * exp2f(fmaf(v[j], c, -log2Sum)) : 0.f;
			store_unit<T, V>(out, u * V - offset, p.vocabulary, v);
		}
	}
	if(!used) return;
	__syncthreads(); // the kept columns of this part have been written, and now get their final value
	for(int k = threadIdx.x; k < p.kept; k += THREADS) {
		const int at = kept.at[k];
		if(at < 0 || (at + offset) / V < begin || (at + offset) / V >= end) continue;
		bool first = true;
		float sum = 0.f;
		for(int o = 0; o < p.kept; ++o) { // a column that was kept twice: its first entry adds them up, in order
			if(kept.at[o] != at) continue;
			if(o < k) first = false;
			sum += kept.p[o];
		}
		if(first) out[at] = from_float<T>(by * (exp2f(fmaf(kept.z[k], c, -log2Sum)) - sum));
	}
}

template<typename F>
void with_types(int type, int teacherType, F&& f)
{
	if(type == NB200_TYPE_FP32) f(float(), float());
	else if(type == NB200_TYPE_FP16) teacherType == NB200_TYPE_FP32 ? f(__half(), float()) : f(__half(), __half());
	else teacherType == NB200_TYPE_FP32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
}

bool arguments_valid(int type, int teacherType, int rows, int vocabulary, long long row, int kept, float temperature)
{
	return type_valid(type) && (teacherType == type || teacherType == NB200_TYPE_FP32) && rows >= 0 && vocabulary >= 1
		&& row >= vocabulary && kept >= 0 && temperature > 0.f && temperature <= 3.4e38f;
}

// Blocks of a row: more than one while the device is not filled and a block still has a few rounds of units.
int parts_of(int type, int rows, int vocabulary)
{
	const int units = (vocabulary + 16 / type_size(type) - 1) / (16 / type_size(type));
	int parts = 1;
	while(parts < MAX_PARTS && static_cast<long long>(rows) * parts < sm_count() * 2 && units > parts * THREADS) parts *= 2;
	return parts;
}

int run(const DistillParams& p, int type, int teacherType, int rows, bool backward, bool alike, cudaStream_t stream)
{
	cudaLaunchConfig_t config = {};
	config.gridDim = dim3(static_cast<unsigned>(rows) * p.parts);
	config.blockDim = dim3(THREADS);
	config.stream = stream;
	cudaLaunchAttribute attribute[1];
	attribute[0].id = cudaLaunchAttributeClusterDimension;
	attribute[0].val.clusterDim.x = p.parts;
	attribute[0].val.clusterDim.y = 1;
	attribute[0].val.clusterDim.z = 1;
	config.attrs = attribute;
	config.numAttrs = p.parts > 1 && !backward ? 1 : 0;
	with_types(type, teacherType, [&](auto t, auto q) {
		using T = decltype(t);
		using P = decltype(q);
		constexpr int V = Unit16<T>::N;
		if(!backward) cudaLaunchKernelEx(&config, distillation_forward_kernel<T, P, V>, p);
		else if(alike) cudaLaunchKernelEx(&config, distillation_backward_kernel<T, P, V>, p);
		else cudaLaunchKernelEx(&config, distillation_backward_kernel<T, P, 1>, p);
	});
	count_launch();
	return check_launch();
}

} // namespace

} // namespace nb200

using namespace nb200;

extern "C" {

int nb200_distillation_loss(void* stream, int type, int teacher_type, const void* logits, int rows, int vocabulary,
	long long row_size, const void* teacher_logits, const int* teacher_indices, int kept, float temperature, float* loss,
	float* log_sum)
{
	if(!arguments_valid(type, teacher_type, rows, vocabulary, row_size, kept, temperature)) return NB200_EINVAL;
	if(rows == 0) return NB200_OK;
	if(logits == nullptr || loss == nullptr || log_sum == nullptr || !type_aligned(logits, type)
		|| !type_aligned(teacher_logits, teacher_type)) return NB200_EINVAL;
	if(kept > 0 && (teacher_logits == nullptr || teacher_indices == nullptr)) return NB200_EINVAL;
	if(kept > KEPT_MAX) return NB200_ETOOBIG;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	DistillParams p = {};
	p.logits = logits; p.teacher = teacher_logits; p.indices = teacher_indices; p.logSum = log_sum; p.loss = loss;
	p.row = row_size; p.vocabulary = vocabulary; p.kept = kept; p.temperature = temperature;
	p.parts = parts_of(type, rows, vocabulary);
	return run(p, type, teacher_type, rows, false, true, as_stream(stream));
}

int nb200_distillation_loss_backward(void* stream, int type, int teacher_type, const float* loss_diff, const void* logits,
	int rows, int vocabulary, long long row_size, const void* teacher_logits, const int* teacher_indices, int kept,
	float temperature, const float* log_sum, void* logits_diff, long long logits_diff_row_size)
{
	if(!arguments_valid(type, teacher_type, rows, vocabulary, row_size, kept, temperature) || logits_diff_row_size < vocabulary) {
		return NB200_EINVAL;
	}
	if(rows == 0) return NB200_OK;
	if(logits == nullptr || loss_diff == nullptr || log_sum == nullptr || logits_diff == nullptr || !type_aligned(logits, type)
		|| !type_aligned(logits_diff, type) || !type_aligned(teacher_logits, teacher_type)) return NB200_EINVAL;
	if(kept > 0 && (teacher_logits == nullptr || teacher_indices == nullptr)) return NB200_EINVAL;
	if(kept > KEPT_MAX) return NB200_ETOOBIG;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	DistillParams p = {};
	p.logits = logits; p.teacher = teacher_logits; p.indices = teacher_indices; p.lossDiff = loss_diff;
	p.logSum = const_cast<float*>(log_sum); p.out = logits_diff;
	p.row = row_size; p.outRow = logits_diff_row_size; p.vocabulary = vocabulary; p.kept = kept; p.temperature = temperature;
	p.parts = parts_of(type, rows, vocabulary);
	// the two rows are cut into the same units where they begin at the same offset from a 16-byte boundary
	const bool alike = ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(logits_diff)) & 15u) == 0
		&& (rows == 1 || ((row_size - logits_diff_row_size) * type_size(type) & 15) == 0);
	return run(p, type, teacher_type, rows, true, alike, as_stream(stream));
}

} // extern "C"
