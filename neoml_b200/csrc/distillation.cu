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

constexpr int BLOCK = 256;     // threads of a row's block; a warp where the row and the teacher's entries are short
constexpr int KEPT_MAX = NB200_DISTILLATION_KEPT_MAX;
constexpr int MAX_PARTS = 8;
constexpr int UNROLL = 4;      // units in flight per thread
constexpr int ENTRIES = KEPT_MAX / BLOCK; // of the teacher, per thread
static_assert(ENTRIES * BLOCK == KEPT_MAX, "every entry has a thread");
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

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

// Maximum of x and the sum of 2^(c (x - maximum)).
struct Running {
	float top, sum;
	__device__ __forceinline__ void join(const Running& o, float c)
	{
		const float t = fmaxf(top, o.top);
		const float at = t == -INFINITY ? 0.f : t;
		sum = sum * exp2_fast((top - at) * c) + o.sum * exp2_fast((o.top - at) * c);
		top = t;
	}
	// log sum exp((x - base) / temperature); the maximum's distance from the base is exact where both are of one size
	__device__ __forceinline__ float log_sum_over(float base, float temperature) const { return (top - base) / temperature + logf(sum); }
};

// The teacher's side of a row, or of some of its entries: maximum of x = log2(e) teacher / tau, sum of 2^(x - maximum), and the sum of
// 2^(x - maximum) (ln 2 (x - maximum) - (z - base) / tau), z being the student's logit and base that of the likeliest entry.  The loss is then
// tau^2 (cross / sum - ln sum + log_sum - base / tau), where the last two are formed as one (log_sum_over): no term is larger than the
// distributions' logarithms, whatever the logits' common offset.
struct Taught {
	float top, sum, cross, base;
	__device__ __forceinline__ void join(const Taught& o, float overTemperature)
	{
		if(sum == 0.f && o.sum == 0.f) return; // neither has an entry (one that is not a number makes the sum none, and leaves no maximum)
		const float t = fmaxf(top, o.top);
		const float d1 = top - t, d2 = o.top - t, f1 = exp2_fast(d1), f2 = exp2_fast(d2);
		// the base is that of the likeliest entry: one that hardly counts may lie at its type's lowest value
		const float from = top >= o.top ? base : o.base;
		const float mine = fmaf((from - base) * overTemperature, sum, cross), its = fmaf((from - o.base) * overTemperature, o.sum, o.cross);
		// what has vanished adds nothing, not even an infinite loss times zero
		cross = (f1 == 0.f ? 0.f : f1 * fmaf(d1 * LN2, sum, mine)) + (f2 == 0.f ? 0.f : f2 * fmaf(d2 * LN2, o.sum, its));
		sum = f1 * sum + f2 * o.sum;
		top = t;
		base = from;
	}
};

// A thread's entries of the teacher.
struct Entry {
	float x, z; // x: minus infinity for one that is not used
	int at;     // column; -1 for one that is not used
};

template<typename T, typename P, int THREADS>
__device__ __forceinline__ void load_entries(const DistillParams& p, int r, const T* logits, Entry (&entries)[ENTRIES])
{
	const P* const teacher = static_cast<const P*>(p.teacher) + static_cast<long long>(r) * p.kept;
	const int* const indices = p.indices + static_cast<long long>(r) * p.kept;
	const float c = LOG2E / p.temperature;
#pragma unroll
	for(int e = 0; e < ENTRIES; ++e) {
		const int k = e * THREADS + threadIdx.x;
		entries[e] = { -INFINITY, 0.f, -1 };
		if(k >= p.kept) continue;
		const int at = __ldg(indices + k);
		if(at < 0 || at >= p.vocabulary) continue;
		entries[e].at = at;
		entries[e].x = to_float(teacher[k]) * c;
		entries[e].z = to_float(logits[at]);
	}
}

// The largest of a unit's elements.
template<typename T>
__device__ __forceinline__ float unit_top(const uint4& raw)
{
	if constexpr(sizeof(T) == 4) {
		return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)), fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
	} else {
		using T2 = typename PairOf<T>::type;
		const uint32_t w[4] = { raw.x, raw.y, raw.z, raw.w };
		const T2 a = __hmax2(__hmax2(*reinterpret_cast<const T2*>(w), *reinterpret_cast<const T2*>(w + 1)),
			__hmax2(*reinterpret_cast<const T2*>(w + 2), *reinterpret_cast<const T2*>(w + 3)));
		const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(&a));
		return fmaxf(f.x, f.y);
	}
}

template<typename T, typename P, int V, int THREADS>
__global__ void __launch_bounds__(THREADS) distillation_forward_kernel(const DistillParams p)
{
	constexpr int WARPS = THREADS / 32;
	__shared__ Running parts[MAX_PARTS];
	__shared__ Running warpsOf[WARPS];
	__shared__ Taught taughtOf[WARPS];
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
	Entry entries[ENTRIES];
	if(rank == 0) load_entries<T, P, THREADS>(p, r, x, entries);
	// exponents are formed of differences: a type's lowest value times c would be infinite
	Running mine = { -INFINITY, 0.f };
	for(int u0 = rank * perBlock; u0 < end; u0 += THREADS * UNROLL) {
		uint4 raw[UNROLL];
		const int mineFirst = u0 + threadIdx.x, mineLast = mineFirst + (UNROLL - 1) * THREADS;
		if(mineLast < end && mineFirst * V - offset >= 0 && mineLast * V - offset + V <= p.vocabulary) { // whole units
#pragma unroll
			for(int k = 0; k < UNROLL; ++k) raw[k] = *reinterpret_cast<const uint4*>(x + ((mineFirst + k * THREADS) * V - offset));
			float top = unit_top<T>(raw[0]);
#pragma unroll
			for(int k = 1; k < UNROLL; ++k) top = fmaxf(top, unit_top<T>(raw[k]));
			top = fmaxf(mine.top, top);
			const float at = top == -INFINITY ? 0.f : top;
			float2 sums = make_float2(mine.sum * exp2_fast((mine.top - at) * c), 0.f);
#pragma unroll
			for(int k = 0; k < UNROLL; ++k) {
				float v[V];
				unit_floats<T, V>(raw[k], v);
#pragma unroll
				for(int j = 0; j < V; j += 2) {
					const float2 e = mul2(add2(make_float2(v[j], v[j + 1]), both(-at)), both(c));
					sums = add2(sums, make_float2(exp2_fast(e.x), exp2_fast(e.y)));
				}
			}
			mine.sum = sums.x + sums.y;
			mine.top = top;
		} else {
			for(int k = 0; k < UNROLL; ++k) {
				const int u = mineFirst + k * THREADS, first = u * V - offset;
				if(u >= end) break;
				uint4 one;
				load_unit<T, V>(row, first, p.vocabulary, one);
				float v[V];
				unit_floats<T, V>(one, v);
				float top = mine.top;
#pragma unroll
				for(int j = 0; j < V; ++j) {
					if(!inside<V>(first, j, p.vocabulary)) v[j] = -INFINITY;
					top = fmaxf(top, v[j]);
				}
				const float at = top == -INFINITY ? 0.f : top;
				mine.sum *= exp2_fast((mine.top - at) * c);
#pragma unroll
				for(int j = 0; j < V; ++j) mine.sum += exp2_fast((v[j] - at) * c);
				mine.top = top;
			}
		}
	}
	Taught taught = { -INFINITY, 0.f, 0.f, 0.f };
	const float overTemperature = 1.f / p.temperature;
	if(rank == 0) {
#pragma unroll
		for(int e = 0; e < ENTRIES; ++e) {
			// (not a number is an entry too)
			if(entries[e].at >= 0 && entries[e].x != -INFINITY) {
				// no base are infinite or undefined logits, and those whose multiples would be
				const bool base = fabsf(entries[e].z) < 1e30f;
				taught.join({ entries[e].x, 1.f, base ? 0.f : -entries[e].z * overTemperature, base ? entries[e].z : 0.f }, overTemperature);
			}
		}
	}
#pragma unroll
	for(int o = 16; o > 0; o >>= 1) {
		mine.join({ __shfl_xor_sync(0xffffffffu, mine.top, o), __shfl_xor_sync(0xffffffffu, mine.sum, o) }, c);
		taught.join({ __shfl_xor_sync(0xffffffffu, taught.top, o), __shfl_xor_sync(0xffffffffu, taught.sum, o),
			__shfl_xor_sync(0xffffffffu, taught.cross, o), __shfl_xor_sync(0xffffffffu, taught.base, o) }, overTemperature);
	}
	if((threadIdx.x & 31) == 0) {
		warpsOf[threadIdx.x >> 5] = mine;
		taughtOf[threadIdx.x >> 5] = taught;
	}
	__syncthreads();
	if(blocks > 1) {
		cg::cluster_group cluster = cg::this_cluster();
		if(threadIdx.x == 0) {
			for(int w = 1; w < WARPS; ++w) mine.join(warpsOf[w], c);
			*cluster.map_shared_rank(&parts[rank], 0) = mine;
		}
		cluster.sync();
	}
	if(rank != 0 || threadIdx.x != 0) return;
	const Running* const all = blocks > 1 ? parts : warpsOf;
	mine = all[0];
	for(int k = 1; k < (blocks > 1 ? blocks : WARPS); ++k) mine.join(all[k], c);
	for(int w = 1; w < WARPS; ++w) taught.join(taughtOf[w], overTemperature);
	p.logSum[r] = mine.log_sum_over(0.f, p.temperature);
	// no entry, or nothing but minus infinity: no loss
	p.loss[r] = taught.top == -INFINITY && taught.sum == 0.f ? 0.f
		: p.temperature * p.temperature * (taught.cross / taught.sum - logf(taught.sum) + mine.log_sum_over(taught.base, p.temperature));
}

template<typename T, typename P, int V, int THREADS>
__global__ void __launch_bounds__(THREADS) distillation_backward_kernel(const DistillParams p)
{
	constexpr int WARPS = THREADS / 32;
	__shared__ int keptAt[ENTRIES * THREADS];
	__shared__ float keptX[ENTRIES * THREADS];
	__shared__ Running warpsOf[WARPS];
	const int blocks = p.parts, r = blockIdx.x / blocks, rank = blockIdx.x - r * blocks;
	const T* const x = static_cast<const T*>(p.logits) + r * p.row;
	T* const out = static_cast<T*>(p.out) + r * p.outRow;
	const int offset = row_offset<T, V>(x);
	const int units = (p.vocabulary + offset + V - 1) / V;
	const int perBlock = (units + blocks - 1) / blocks;
	const int begin = rank * perBlock, end = min(units, begin + perBlock);
	const float c = LOG2E / p.temperature;
	// the student's kept logits are read here, before anything is written: the gradient may replace the logits
	Entry entries[ENTRIES];
	load_entries<T, P, THREADS>(p, r, x, entries);
	Running teacher = { -INFINITY, 0.f };
#pragma unroll
	for(int e = 0; e < ENTRIES; ++e) {
		const int k = e * THREADS + threadIdx.x;
		if(k < p.kept) {
			keptAt[k] = entries[e].at;
			keptX[k] = entries[e].x;
		}
		if(entries[e].at >= 0 && entries[e].x != -INFINITY) teacher.join({ entries[e].x, 1.f }, 1.f);
	}
#pragma unroll
	for(int o = 16; o > 0; o >>= 1) teacher.join({ __shfl_xor_sync(0xffffffffu, teacher.top, o), __shfl_xor_sync(0xffffffffu, teacher.sum, o) }, 1.f);
	if((threadIdx.x & 31) == 0) warpsOf[threadIdx.x >> 5] = teacher;
	const float diff = p.temperature * __ldg(p.lossDiff + r), log2Sum = __ldg(p.logSum + r) * LOG2E;
	__syncthreads();
	teacher = warpsOf[0];
#pragma unroll
	for(int w = 1; w < WARPS; ++w) teacher.join(warpsOf[w], 1.f);
	const bool used = !(teacher.top == -INFINITY && teacher.sum == 0.f);
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
			for(int j = 0; j < V; ++j) v[j] = used ? diff * exp2_fast(fmaf(v[j], c, -log2Sum)) : 0.f;
			store_unit<T, V>(out, u * V - offset, p.vocabulary, v);
		}
	}
	if(!used) return;
	__syncthreads(); // the kept columns of this part have been written, and now get their final value
#pragma unroll
	for(int e = 0; e < ENTRIES; ++e) {
		const int k = e * THREADS + threadIdx.x, at = entries[e].at;
		if(at < 0 || (at + offset) / V < begin || (at + offset) / V >= end) continue;
		bool first = true;
		float sum = 0.f;
		for(int o = 0; o < p.kept; ++o) { // a column that was kept twice: its first entry adds them up, in order
			if(keptAt[o] != at) continue;
			if(o < k) first = false;
			sum += exp2_fast(keptX[o] - teacher.top);
		}
		if(first) out[at] = from_float<T>(diff * (exp2_fast(fmaf(entries[e].z, c, -log2Sum)) - sum / teacher.sum));
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
	while(parts < MAX_PARTS && static_cast<long long>(rows) * parts < sm_count() * 2 && units > parts * BLOCK) parts *= 2;
	return parts;
}

int run(const DistillParams& p, int type, int teacherType, int rows, bool backward, bool alike, cudaStream_t stream)
{
	cudaLaunchConfig_t config = {};
	config.gridDim = dim3(static_cast<unsigned>(rows) * p.parts);
	config.stream = stream;
	cudaLaunchAttribute attribute[1];
	attribute[0].id = cudaLaunchAttributeClusterDimension;
	attribute[0].val.clusterDim.x = p.parts;
	attribute[0].val.clusterDim.y = 1;
	attribute[0].val.clusterDim.z = 1;
	config.attrs = attribute;
	config.numAttrs = p.parts > 1 && !backward ? 1 : 0;
	// a warp per row: the loss of 8000 rows of 1000 bf16 takes 36 us with blocks of 256 and 15 with warps, its gradient 41 and 13
	const bool small = p.parts == 1 && p.kept <= ENTRIES * 32 && p.vocabulary <= 32 * 8 * (16 / type_size(type)) && rows >= sm_count();
	config.blockDim = dim3(small ? 32 : BLOCK);
	with_types(type, teacherType, [&](auto t, auto q) {
		using T = decltype(t);
		using P = decltype(q);
		constexpr int V = Unit16<T>::N;
		if(!backward) cudaLaunchKernelEx(&config, small ? distillation_forward_kernel<T, P, V, 32> : distillation_forward_kernel<T, P, V, BLOCK>, p);
		else if(alike) cudaLaunchKernelEx(&config, small ? distillation_backward_kernel<T, P, V, 32> : distillation_backward_kernel<T, P, V, BLOCK>, p);
		else {
			config.blockDim = dim3(BLOCK);
			cudaLaunchKernelEx(&config, distillation_backward_kernel<T, P, 1, BLOCK>, p);
		}
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
		|| !type_aligned(teacher_logits, teacher_type) || !words_aligned(teacher_indices, loss, log_sum)) return NB200_EINVAL;
	if(kept > 0 && (teacher_logits == nullptr || teacher_indices == nullptr)) return NB200_EINVAL;
	if(kept > KEPT_MAX || vocabulary > (1 << 30)) return NB200_ETOOBIG;
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
		|| !type_aligned(logits_diff, type) || !type_aligned(teacher_logits, teacher_type)
		|| !words_aligned(loss_diff, teacher_indices, log_sum)) return NB200_EINVAL;
	if(kept > 0 && (teacher_logits == nullptr || teacher_indices == nullptr)) return NB200_EINVAL;
	if(kept > KEPT_MAX || vocabulary > (1 << 30)) return NB200_ETOOBIG;
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
