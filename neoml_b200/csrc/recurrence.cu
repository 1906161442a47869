// A gated linear recurrence over [batch][length][channels], forward and backward.
//
//   a = sigmoid(forget), u = sigmoid(input), or 1 - a without input gates;   h_t = a_t h_{t-1} + u_t z_t
//   backward:  S_t = dh_t + a_{t+1} S_{t+1};  dz = S u,  d(forget) = S h_{t-1} a (1 - a)  [coupled: S (h_{t-1} - z) a (1 - a)],
//   d(input) = S z u (1 - u),  dh_0 = a_1 S_1
//
// Both are first-order linear recurrences, s' = A s + H, whose steps compose: (A2, H2) after (A1, H1) is (A2 A1, A2 H1 + H2).
// The work is bound by memory as long as every element is read once and both gates are formed once, so a chunk of the time
// axis is read into registers, folded there, joined with the chunks around it, and its states are written out of the
// same registers:
//   thread   one channel (two 16-bit channels) times STEPS steps: loads them all at once,
//            folds them to one (A, H)
//   block    its warps hold consecutive stretches of time for the same 32 or 64 channels; the folds meet in shared memory
//   cluster  up to 8 blocks hold consecutive stretches again; a cluster walks its channels' whole time axis, carrying the state
//            in a register.  Blocks send each other their folds by asynchronous stores that count on the receiver's
//            mbarrier: a cluster-wide barrier would wait for the results' stores to global memory too, every round
// The next round's loads are issued before this one is folded.
// The gates' pre-activations are the inputs: a gate of 0.999 rounded to bf16 is 1 and would never forget.
// The backward pass of fp32 takes h_{t-1} from the result.  In 16-bit types the result is rounded (half a step of it in d(forget), and an infinite
// one where a half ends), so the states are formed again in fp32: a pass over the inputs stores one in front of every eight steps, a quarter of an
// array's bytes, and a thread of the backward kernel goes through its own steps from there while the folds are under way (16 x 2048 x 2048
// bf16: 60 us and 132; by rounded states 141 without that pass, and gradients 1.77e-3 off instead of 1.66e-3).
#include "product16.cuh"
#include <cooperative_groups.h>
#include <cuda.h>

namespace nb200 {

namespace {

namespace cg = cooperative_groups;

constexpr int STEPS = 8;       // of a thread
constexpr int MAX_WARPS = 8;   // of a block
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_BATCH = 65535; // sequences are the grid's third dimension
constexpr int KERNEL_ID = 0x71; // in the status word: (KERNEL_ID << 8) | site

struct RecurrenceParams {
	const void *z, *f, *i;          // update, forget, input (null: coupled)
	const void *dh, *h;             // backward: gradient of the result, the result
	void *out, *df, *di;            // out: result, or gradient of the update
	const float* first;             // initial state [batch][channels], null: zeros; backward too
	const float* lastDiff;          // backward: gradient of the final state, null: zeros
	float* last;                    // final state, or gradient of the initial one; null: not wanted
	const int* lengths;             // null: all `length`
	long long zBatch, zRow, fBatch, fRow, iBatch, iRow, dhBatch, dhRow; // elements between sequences and steps
	int length, channels;
	int* status;
};

// The one or two channels of a thread.
template<int W> struct Num;
template<> struct Num<1> { float v; };
template<> struct Num<2> { float2 v; };
__device__ __forceinline__ Num<1> add(Num<1> a, Num<1> b) { return { a.v + b.v }; }
__device__ __forceinline__ Num<1> mul(Num<1> a, Num<1> b) { return { a.v * b.v }; }
__device__ __forceinline__ Num<1> fma(Num<1> a, Num<1> b, Num<1> c) { return { fmaf(a.v, b.v, c.v) }; }
__device__ __forceinline__ Num<2> add(Num<2> a, Num<2> b) { return { add2(a.v, b.v) }; }
__device__ __forceinline__ Num<2> mul(Num<2> a, Num<2> b) { return { mul2(a.v, b.v) }; }
__device__ __forceinline__ Num<2> fma(Num<2> a, Num<2> b, Num<2> c) { return { fma2(a.v, b.v, c.v) }; }
template<int W> __device__ __forceinline__ Num<W> all(float v)
{
	if constexpr(W == 1) return { v };
	else return { both(v) };
}
template<int W> __device__ __forceinline__ Num<W> pick(bool yes, Num<W> a, Num<W> b)
{
	if constexpr(W == 1) return { yes ? a.v : b.v };
	else return { make_float2(yes ? a.v.x : b.v.x, yes ? a.v.y : b.v.y) };
}

__device__ __forceinline__ float inverse_fast(float x)
{
	float y;
	asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}
__device__ __forceinline__ Num<1> exp2_of(Num<1> x) { return { exp2_fast(x.v) }; }
__device__ __forceinline__ Num<2> exp2_of(Num<2> x) { return { make_float2(exp2_fast(x.v.x), exp2_fast(x.v.y)) }; }
__device__ __forceinline__ Num<1> inverse_of(Num<1> x) { return { inverse_fast(x.v) }; }
__device__ __forceinline__ Num<2> inverse_of(Num<2> x) { return { make_float2(inverse_fast(x.v.x), inverse_fast(x.v.y)) }; }

// The channels of one step as they lie in memory: one register.  SPLIT: two 16-bit channels that are not one aligned word; `second`
// is 1, or 0 where the thread has the last channel alone.
template<typename T, bool SPLIT>
__device__ __forceinline__ uint32_t load_raw(const T* p, int second)
{
	if constexpr(!SPLIT) return *reinterpret_cast<const uint32_t*>(p);
	else return reinterpret_cast<const unsigned short*>(p)[0] | static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(p)[second]) << 16;
}
template<typename T, int W>
__device__ __forceinline__ Num<W> number(uint32_t raw)
{
	if constexpr(sizeof(T) == 4) return { __uint_as_float(raw) };
	else return { unpack2<T>(raw) };
}
template<typename T, int W, bool SPLIT>
__device__ __forceinline__ void store_raw(T* p, Num<W> v, int second)
{
	if constexpr(sizeof(T) == 4) {
		*p = v.v;
	} else if constexpr(!SPLIT) {
		*reinterpret_cast<uint32_t*>(p) = pack2<T>(v.v.x, v.v.y);
	} else {
		p[0] = from_float<T>(v.v.x);
		if(second != 0) p[1] = from_float<T>(v.v.y);
	}
}

// A pair of states in front of a stretch of steps, kept in 16-bit memory that the stretch's gradients take later: the upper halves of both in
// the stretch's first row, the lower halves in its second one.  Who reads them is the thread that writes the gradients there.
template<typename T, bool SPLIT>
__device__ __forceinline__ void store_parts(T* at, int row, Num<2> v, int second)
{
	const uint32_t x = __float_as_uint(v.v.x), y = __float_as_uint(v.v.y);
	const uint32_t parts[2] = { __byte_perm(x, y, 0x7632), __byte_perm(x, y, 0x5410) };
#pragma unroll
	for(int k = 0; k < 2; ++k) {
		unsigned short* const to = reinterpret_cast<unsigned short*>(at + static_cast<long long>(k) * row);
		if constexpr(SPLIT) {
			to[0] = static_cast<unsigned short>(parts[k]);
			if(second != 0) to[1] = static_cast<unsigned short>(parts[k] >> 16);
		} else {
			*reinterpret_cast<uint32_t*>(to) = parts[k];
		}
	}
}
template<typename T, bool SPLIT>
__device__ __forceinline__ uint2 load_parts(const T* at, int row, int second)
{
	return make_uint2(load_raw<T, SPLIT>(at, second), load_raw<T, SPLIT>(at + row, second));
}
template<int W>
__device__ __forceinline__ Num<W> from_parts(uint2 parts)
{
	if constexpr(W == 2) return { make_float2(__uint_as_float(__byte_perm(parts.y, parts.x, 0x5410)), __uint_as_float(__byte_perm(parts.y, parts.x, 0x7632))) };
	else return all<W>(0.f); // fp32 states are not kept in parts
}

template<int W>
struct Gate {
	Num<W> keep, take; // sigmoid(x), 1 - sigmoid(x)
};

constexpr float MINUS_LOG2E = -1.4426950408889634f;

// Both without cancellation: with e = 2^(-x log2 e), keep = 1 / (1 + e) and take = e keep.  In fp32, where e may overflow, of |x|,
// and exchanged for a negative x.  16-bit gates are held at -80 instead (not a number stays one): 1.8e-35 is no other gate than zero there.
template<typename T, int W>
__device__ __forceinline__ Gate<W> gate(uint32_t raw)
{
	if constexpr(sizeof(T) == 4) {
		const float x = __uint_as_float(raw);
		const float e = exp2_fast(fabsf(x) * MINUS_LOG2E);
		const float large = inverse_fast(1.f + e), small = e * large;
		return x >= 0.f ? Gate<W>{ { large }, { small } } : Gate<W>{ { small }, { large } };
	} else {
		using T2 = typename PairOf<T>::type;
		const uint32_t floor = pack2<T>(-80.f, -80.f);
		const T2 held = __hmax2_nan(*reinterpret_cast<const T2*>(&raw), *reinterpret_cast<const T2*>(&floor));
		const Num<W> e = exp2_of(mul(number<T, W>(*reinterpret_cast<const uint32_t*>(&held)), all<W>(MINUS_LOG2E)));
		const Num<W> keep = inverse_of(add(e, all<W>(1.f)));
		return { keep, mul(e, keep) };
	}
}
template<typename T, int W>
__device__ __forceinline__ Num<W> sigmoid(uint32_t raw)
{
	return inverse_of(add(exp2_of(mul(number<T, W>(raw), all<W>(MINUS_LOG2E))), all<W>(1.f))); // 2^infinity: zero
}

template<int W>
struct Fold {
	Num<W> a, h;
};

// What a block's threads share: their folds, and those of the cluster's blocks, each in two sets for alternating rounds; laid out at the
// head of the dynamic shared memory, alike in all blocks of the cluster.
template<int W>
struct Shared {
	Fold<W>* folds; // [2][warps][32], then [2][blocks][32]
	int warpCount, blockCount;
	uint64_t* arrived;  // [2]
	int* abortFlag;
	__device__ __forceinline__ Fold<W>& warp(int set, int k, int lane) const { return folds[(set * warpCount + k) * 32 + lane]; }
	__device__ __forceinline__ Fold<W>& block(int set, int k, int lane) const { return folds[(2 * warpCount + set * blockCount + k) * 32 + lane]; }
};
__host__ __device__ __forceinline__ constexpr int shared_bytes(int warps, int blocks, int w) // a multiple of 128
{
	return 2 * (warps + blocks) * 32 * 8 * w;
}

// Stores a fold in the shared memory of block `rank` of the cluster and counts its bytes on that block's barrier.
__device__ __forceinline__ void send(const Fold<1>& f, Fold<1>* at, uint64_t* bar, int rank)
{
	asm volatile("{\n\t.reg .b32 a, m;\n\t"
		"mapa.shared::cluster.u32 a, %0, %2;\n\t"
		"mapa.shared::cluster.u32 m, %1, %2;\n\t"
		"st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [a], {%3, %4}, [m];\n\t}"
		::"r"(smem_u32(at)), "r"(smem_u32(bar)), "r"(rank), "r"(__float_as_uint(f.a.v)), "r"(__float_as_uint(f.h.v)) : "memory");
}
__device__ __forceinline__ void send(const Fold<2>& f, Fold<2>* at, uint64_t* bar, int rank)
{
	asm volatile("{\n\t.reg .b32 a, m;\n\t"
		"mapa.shared::cluster.u32 a, %0, %2;\n\t"
		"mapa.shared::cluster.u32 m, %1, %2;\n\t"
		"st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [a], {%3, %4, %5, %6}, [m];\n\t}"
		::"r"(smem_u32(at)), "r"(smem_u32(bar)), "r"(rank), "r"(__float_as_uint(f.a.v.x)), "r"(__float_as_uint(f.a.v.y)),
		  "r"(__float_as_uint(f.h.v.x)), "r"(__float_as_uint(f.h.v.y)) : "memory");
}

template<int W>
__device__ __forceinline__ Shared<W> begin_sharing(uint8_t* room, uint64_t* arrived, int* abortFlag, int warps, int blocks)
{
	if(threadIdx.x == 0) {
		mbar_init(arrived, 1);
		mbar_init(arrived + 1, 1);
		mbar_init_fence();
		*abortFlag = 0;
	}
	if(blocks > 1) cg::this_cluster().sync(); // the others' shared memory and barriers exist from here on
	else __syncthreads();
	return { reinterpret_cast<Fold<W>*>(room), warps, blocks, arrived, abortFlag };
}

// A wait of the whole warp; once one of the block's has given up, the others do as soon as they would have to wait.  A block then sends and
// asks for nothing more, since its barriers' phases are no longer those of its rounds, but goes through them with what is there: every
// block has to reach the end.
__device__ __forceinline__ void wait_warp(uint64_t* bar, uint32_t parity, volatile int* abortFlag, int* status, int site)
{
	if(__all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || *abortFlag != 0) return;
	mbar_wait_bounded_warp(bar, parity, abortFlag, status, site);
}

// Joins the folds of a round: `mine` is this thread's stretch; the state before it is returned in `state`, and `carry` moves on by
// the whole round.  Stretches follow one another warp by warp, block by block.
//   A set of folds is written again two rounds later.  Within the block, the barrier of the round between keeps the writers
// behind the readers.  Between blocks: a block sends its fold of a round after its own barrier, when all its warps have read
// the set of the round before, and nobody sends the round after next without having received that fold.
// `meanwhile` is what can be done without the state, while the folds are under way.
template<int W, typename F>
__device__ __forceinline__ void join(const Shared<W>& s, const Fold<W>& mine, int round, int rank, int blocks, int warps, int* status,
	Num<W>& carry, Num<W>& state, F&& meanwhile)
{
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, set = round & 1;
	Fold<W> before = { all<W>(1.f), all<W>(0.f) };
	auto after = [](Fold<W>& f, const Fold<W>& next) {
		f.h = fma(next.a, f.h, next.h);
		f.a = mul(f.a, next.a);
	};
	if(warps > 1) {
		if(warp < warps - 1) s.warp(set, warp, lane) = mine;
		__syncthreads();
		for(int k = 0; k < warp; ++k) after(before, s.warp(set, k, lane));
	}
	if(warp == warps - 1) { // the block's fold, to every block of the cluster, this one too
		Fold<W> whole = before;
		after(whole, mine);
		if(*static_cast<volatile int*>(s.abortFlag) != 0) {
		} else if(blocks == 1) { // launched without a cluster: st.async is not an instruction of such a kernel
			s.block(set, 0, lane) = whole;
			__syncwarp();
			if(lane == 0) mbar_arrive(s.arrived + set);
		} else {
			if(lane == 0) mbar_arrive_expect_tx(s.arrived + set, static_cast<uint32_t>(blocks * 32 * sizeof(Fold<W>)));
			for(int k = 0; k < blocks; ++k) send(whole, &s.block(set, rank, lane), s.arrived + set, k);
		}
	}
	meanwhile();
	wait_warp(s.arrived + set, (round >> 1) & 1, s.abortFlag, status, (KERNEL_ID << 8) | 1);
	Num<W> start = carry;
	for(int k = 0; k < blocks; ++k) {
		if(k == rank) start = carry;
		const Fold<W> next = s.block(set, k, lane);
		carry = fma(next.a, carry, next.h);
	}
	state = fma(before.a, start, before.h);
}

// A state or its gradient, fp32; null: zeros.
template<int W>
__device__ __forceinline__ Num<W> load_state(const float* from, long long at, int second)
{
	if(from == nullptr) return all<W>(0.f);
	if constexpr(W == 1) return { from[at] };
	else return { make_float2(from[at], from[at + second]) };
}
template<int W>
__device__ __forceinline__ void store_state(float* to, long long at, Num<W> v, int second)
{
	if constexpr(W == 1) {
		to[at] = v.v;
	} else {
		to[at] = v.v.x;
		if(second != 0) to[at + 1] = v.v.y;
	}
}

__device__ __forceinline__ int sequence_length(const RecurrenceParams& p, int b)
{
	if(p.lengths == nullptr) return p.length;
	const int n = __ldg(p.lengths + b);
	return n < 0 ? 0 : n > p.length ? p.length : n;
}

// Where a block's part of a round lies in an operand.  DENSE operands (channels adjacent, steps `channels` apart) share one 32-bit
// offset per step, the same in every round, on a base that is uniform in the block: no address arithmetic per load.
template<typename T, bool DENSE>
struct Operand {
	const uint8_t* base; // step 0 of this block's sequence; DENSE: of the round
	long long row;       // bytes between steps
	__device__ __forceinline__ const T* at(uint32_t offset, int t, int c) const
	{
		return DENSE ? reinterpret_cast<const T*>(base + offset) : reinterpret_cast<const T*>(base + t * row) + c;
	}
};

// Runs f(integral constant) as true where every step of the thread's stretch exists, without a test per step.
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// The same pass over the inputs, but of the states only those in front of every STEPS-th step are stored, for the backward pass of 16-bit
// types (store_parts): stretches end at a sequence's end then, as they do there, and the first of them may begin in front of step 0.
template<bool STATES>
struct Stretches {
	int n;
	__device__ __forceinline__ int begin(int stride) const { return STATES ? n - (n + stride - 1) / stride * stride : 0; }
	__device__ __forceinline__ bool in(int t) const { return STATES ? t >= 0 && t < n : t < n; }
	__device__ __forceinline__ bool whole(int t, int steps) const { return (!STATES || t >= 0) && t + steps <= n; }
};

template<typename T, int W, bool INPUT, bool DENSE, bool SPLIT, bool STATES>
__global__ void __launch_bounds__(MAX_WARPS * 32, W == 1 ? 3 : 2) recurrence_forward_kernel(const RecurrenceParams p)
{
	extern __shared__ __align__(128) uint8_t sharedRoom[];
	__shared__ uint64_t arrived[2];
	__shared__ int abortFlag;
	const int blocks = gridDim.y, rank = blockIdx.y; // the blocks of a cluster
	const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
	const Shared<W> s = begin_sharing<W>(sharedRoom, arrived, &abortFlag, warps, blocks);
	const int b = blockIdx.z;
	const int own = (blockIdx.x * 32 + (threadIdx.x & 31)) * W;
	const bool on = own < p.channels;
	const int c = on ? own : 0; // lanes behind the last channel read what others read, and write nothing
	const int second = c + 1 < p.channels ? 1 : 0;
	const int n = sequence_length(p, b);
	const int span = warps * STEPS, stride = span * blocks;
	const Stretches<STATES> all_steps = { n };
	const int begin = all_steps.begin(stride), first = rank * span + warp * STEPS;
	const long long back = DENSE ? static_cast<long long>(begin) * p.channels * static_cast<long long>(sizeof(T)) : 0; // nothing in front of step 0 is read
	Operand<T, DENSE> z = { static_cast<const uint8_t*>(p.z) + b * p.zBatch * sizeof(T) + back, p.zRow * static_cast<long long>(sizeof(T)) };
	Operand<T, DENSE> f = { static_cast<const uint8_t*>(p.f) + b * p.fBatch * sizeof(T) + back, p.fRow * static_cast<long long>(sizeof(T)) };
	Operand<T, DENSE> i = { static_cast<const uint8_t*>(p.i) + b * p.iBatch * sizeof(T) + back, p.iRow * static_cast<long long>(sizeof(T)) };
	T* const out = static_cast<T*>(p.out) + static_cast<long long>(b) * p.length * p.channels;
	uint8_t* outRound = reinterpret_cast<uint8_t*>(out) + back;
	const long long roundBytes = static_cast<long long>(stride) * p.channels * sizeof(T);
	uint32_t offset[STEPS];
#pragma unroll
	for(int k = 0; k < STEPS; ++k) offset[k] = (static_cast<uint32_t>(first + k) * p.channels + c) * static_cast<uint32_t>(sizeof(T));
	const long long state0 = static_cast<long long>(b) * p.channels + c;
	Num<W> carry = load_state<W>(p.first, state0, second);

	uint32_t rz[STEPS], rf[STEPS], ri[STEPS];
	auto load = [&](int t, auto full) {
#pragma unroll
		for(int k = 0; k < STEPS; ++k) {
			const bool in = decltype(full)::value || all_steps.in(t + k);
			rz[k] = in ? load_raw<T, SPLIT>(z.at(offset[k], t + k, c), second) : 0u;
			rf[k] = in ? load_raw<T, SPLIT>(f.at(offset[k], t + k, c), second) : 0u;
			if constexpr(INPUT) ri[k] = in ? load_raw<T, SPLIT>(i.at(offset[k], t + k, c), second) : 0u;
		}
	};
	int round = 0, t = begin + first;
	if(all_steps.whole(t, STEPS)) load(t, Yes());
	else load(t, No());
	// the whole cluster agrees on n, and on the number of rounds
	for(; round * stride < n; ++round) {
		Num<W> a[STEPS], h[STEPS];
		Fold<W> mine = { all<W>(1.f), all<W>(0.f) };
		auto fold = [&](auto full) {
#pragma unroll
			for(int k = 0; k < STEPS; ++k) {
				const bool in = decltype(full)::value || all_steps.in(t + k);
				const Gate<W> forget = gate<T, W>(rf[k]);
				Num<W> take = forget.take;
				if constexpr(INPUT) take = sigmoid<T, W>(ri[k]);
				a[k] = pick<W>(in, forget.keep, all<W>(1.f));
				h[k] = pick<W>(in, mul(take, number<T, W>(rz[k])), all<W>(0.f));
				mine.h = fma(a[k], mine.h, h[k]);
				mine.a = mul(mine.a, a[k]);
			}
		};
		const bool whole = all_steps.whole(t, STEPS);
		if(whole) fold(Yes());
		else fold(No());
		if constexpr(DENSE) {
			z.base += roundBytes;
			f.base += roundBytes;
			if constexpr(INPUT) i.base += roundBytes;
		}
		if(all_steps.whole(t + stride, STEPS)) load(t + stride, Yes());
		else load(t + stride, No());
		Num<W> state;
		join<W>(s, mine, round, rank, blocks, warps, p.status, carry, state, [] {});
		auto apply = [&](auto full) {
#pragma unroll
			for(int k = 0; k < STEPS; ++k) {
				state = fma(a[k], state, h[k]);
				T* const to = DENSE ? reinterpret_cast<T*>(outRound + offset[k]) : out + static_cast<long long>(t + k) * p.channels + c;
				if(on && (decltype(full)::value || t + k < n)) store_raw<T, W, SPLIT>(to, state, second);
			}
		};
		if constexpr(STATES) {
			if(on && t > 0) store_parts<T, SPLIT>(DENSE ? reinterpret_cast<T*>(outRound + offset[0]) : out + static_cast<long long>(t) * p.channels + c, p.channels, state, second);
		} else {
			if(whole) apply(Yes());
			else apply(No());
		}
		outRound += roundBytes;
		t += stride;
	}
	// behind the sequence the results are zeros
	for(int k = n + rank * warps + warp; !STATES && k < p.length; k += blocks * warps) {
		if(on) store_raw<T, W, SPLIT>(out + static_cast<long long>(k) * p.channels + c, all<W>(0.f), second);
	}
	if(blocks > 1) cg::this_cluster().sync(); // nobody leaves while its shared memory may be written
	// behind it: the initial state, which all blocks read, may lie in the same place
	if(on && p.last != nullptr && rank == 0 && warp == 0) store_state<W>(p.last, state0, carry, second);
}

// Time runs backwards: step k of a stretch is t - k.
template<typename T, int W, bool INPUT, bool DENSE, bool SPLIT>
__global__ void __launch_bounds__(MAX_WARPS * 32, 2) recurrence_backward_kernel(const RecurrenceParams p)
{
	constexpr bool STORED = sizeof(T) == 4; // the result holds the states as they were
	extern __shared__ __align__(128) uint8_t sharedRoom[];
	__shared__ uint64_t arrived[2];
	__shared__ int abortFlag;
	const int blocks = gridDim.y, rank = blockIdx.y;
	const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
	const Shared<W> s = begin_sharing<W>(sharedRoom, arrived, &abortFlag, warps, blocks);
	const int b = blockIdx.z;
	const int own = (blockIdx.x * 32 + (threadIdx.x & 31)) * W;
	const bool on = own < p.channels;
	const int c = on ? own : 0;
	const int second = c + 1 < p.channels ? 1 : 0;
	const int n = sequence_length(p, b);
	const int span = warps * STEPS, stride = span * blocks;
	const int back = rank * span + warp * STEPS; // steps between the round's last one and this thread's first
	const long long roundBytes = static_cast<long long>(stride) * p.channels * sizeof(T);
	const long long sequence = static_cast<long long>(b) * p.length * p.channels;
	// DENSE: bases of the round, which ends behind step n - 1; nothing in front of step 0 is read
	const long long begin = DENSE ? static_cast<long long>(n - stride) * p.channels * static_cast<long long>(sizeof(T)) : 0;
	Operand<T, DENSE> z = { static_cast<const uint8_t*>(p.z) + b * p.zBatch * sizeof(T) + begin, p.zRow * static_cast<long long>(sizeof(T)) };
	Operand<T, DENSE> f = { static_cast<const uint8_t*>(p.f) + b * p.fBatch * sizeof(T) + begin, p.fRow * static_cast<long long>(sizeof(T)) };
	Operand<T, DENSE> i = { static_cast<const uint8_t*>(p.i) + b * p.iBatch * sizeof(T) + begin, p.iRow * static_cast<long long>(sizeof(T)) };
	Operand<T, DENSE> dh = { static_cast<const uint8_t*>(p.dh) + b * p.dhBatch * sizeof(T) + begin, p.dhRow * static_cast<long long>(sizeof(T)) };
	const long long denseRow = static_cast<long long>(p.channels) * sizeof(T);
	Operand<T, DENSE> h = { static_cast<const uint8_t*>(p.h) + sequence * sizeof(T) + begin - denseRow, denseRow }; // the step before
	T* const dz = static_cast<T*>(p.out) + sequence;
	T* const df = static_cast<T*>(p.df) + sequence;
	T* const di = INPUT ? static_cast<T*>(p.di) + sequence : nullptr;
	long long outRound = begin;
	uint32_t offset[STEPS];
#pragma unroll
	for(int k = 0; k < STEPS; ++k) offset[k] = (static_cast<uint32_t>(stride - 1 - back - k) * p.channels + c) * static_cast<uint32_t>(sizeof(T));
	const long long state0 = static_cast<long long>(b) * p.channels + c;
	Num<W> carry = load_state<W>(p.lastDiff, state0, second); // what step t + 1 hands back, a_{t+1} S_{t+1}
	const Num<W> first = load_state<W>(p.first, state0, second);
	// behind the sequence the gradients are zeros
	for(int k = n + rank * warps + warp; k < p.length; k += blocks * warps) {
		const long long at = static_cast<long long>(k) * p.channels + c;
		if(!on) break;
		store_raw<T, W, SPLIT>(dz + at, all<W>(0.f), second);
		store_raw<T, W, SPLIT>(df + at, all<W>(0.f), second);
		if constexpr(INPUT) store_raw<T, W, SPLIT>(di + at, all<W>(0.f), second);
	}
	// The gates and the gradients are wanted when a round begins, the rest only when its state has arrived: the former are
	// loaded a whole round ahead, the latter while the round before them ends.
	uint32_t rz[STEPS], rf[STEPS], ri[STEPS], rd[STEPS], nd[STEPS], rh[STORED ? STEPS : 1];
	uint2 parts = make_uint2(0u, 0u); // the state in front of the stretch
	auto load_gates = [&](int t, auto full) {
#pragma unroll
		for(int k = 0; k < STEPS; ++k) {
			const bool in = decltype(full)::value || t - k >= 0;
			rf[k] = in ? load_raw<T, SPLIT>(f.at(offset[k], t - k, c), second) : 0u;
			nd[k] = in ? load_raw<T, SPLIT>(dh.at(offset[k], t - k, c), second) : 0u;
		}
	};
	auto load_rest = [&](int t, long long round, auto full) {
		if constexpr(!STORED && decltype(full)::value) {
			parts = load_parts<T, SPLIT>(DENSE ? reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(dz) + round + offset[STEPS - 1])
				: dz + static_cast<long long>(t - STEPS + 1) * p.channels + c, p.channels, second);
		}
#pragma unroll
		for(int k = 0; k < STEPS; ++k) {
			const bool in = decltype(full)::value || t - k >= 0;
			rz[k] = in ? load_raw<T, SPLIT>(z.at(offset[k], t - k, c), second) : 0u;
			if constexpr(STORED) rh[k] = decltype(full)::value || t - k > 0 ? load_raw<T, SPLIT>(h.at(offset[k], t - k, c), second) : 0u;
			if constexpr(INPUT) ri[k] = in ? load_raw<T, SPLIT>(i.at(offset[k], t - k, c), second) : 0u;
		}
	};
	int round = 0, t = n - 1 - back;
	if(t - STEPS >= 0) {
		load_gates(t, Yes());
		load_rest(t, outRound, Yes());
	} else {
		load_gates(t, No());
		load_rest(t, outRound, No());
	}
	for(; round * stride < n; ++round) {
		Num<W> a[STEPS], u[STEPS];
		Fold<W> mine = { all<W>(1.f), all<W>(0.f) };
		auto fold = [&](auto full) {
#pragma unroll
			for(int k = 0; k < STEPS; ++k) {
				rd[k] = nd[k];
				const bool in = decltype(full)::value || t - k >= 0;
				const Gate<W> forget = gate<T, W>(rf[k]);
				a[k] = pick<W>(in, forget.keep, all<W>(1.f));
				u[k] = forget.take;
				// a (dh + s): this step's own part is a dh
				mine.h = mul(a[k], add(mine.h, number<T, W>(rd[k])));
				mine.a = mul(mine.a, a[k]);
			}
		};
		const bool whole = t - STEPS >= 0, nextWhole = t - stride - STEPS >= 0;
		if(whole) fold(Yes());
		else fold(No());
		if constexpr(DENSE) {
			f.base -= roundBytes;
			dh.base -= roundBytes;
		}
		if(nextWhole) load_gates(t - stride, Yes());
		else load_gates(t - stride, No());
		// d(forget) of a step: S times this, which takes the state in front of it
		Num<W> slope[STEPS];
		auto slopes = [&](auto full) {
			Num<W> running = first;
			if constexpr(!STORED && decltype(full)::value) running = from_parts<W>(parts);
#pragma unroll
			for(int k = STEPS - 1; k >= 0; --k) {
				const Num<W> value = number<T, W>(rz[k]);
				Num<W> before = running;
				if constexpr(STORED) {
					before = number<T, W>(rh[k]);
					if(!decltype(full)::value && t - k == 0) before = first;
				} else { // steps in front of the first one: a is one, the value zero
					Num<W> take = u[k];
					if constexpr(INPUT) take = sigmoid<T, W>(ri[k]);
					running = fma(a[k], before, mul(take, value));
				}
				slope[k] = mul(mul(a[k], u[k]), INPUT ? before : fma(value, all<W>(-1.f), before));
			}
		};
		Num<W> state;
		join<W>(s, mine, round, rank, blocks, warps, p.status, carry, state, [&] {
			if(whole) slopes(Yes());
			else slopes(No());
		});
		auto apply = [&](auto full) {
#pragma unroll
			for(int k = 0; k < STEPS; ++k) {
				const Num<W> S = add(state, number<T, W>(rd[k]));
				Num<W> oz, oi = S;
				if constexpr(INPUT) {
					const Gate<W> take = gate<T, W>(ri[k]);
					oz = mul(S, take.keep);
					oi = mul(mul(oz, number<T, W>(rz[k])), take.take);
				} else {
					oz = mul(S, u[k]);
				}
				const Num<W> of = mul(S, slope[k]);
				state = mul(a[k], S);
				if(on && (decltype(full)::value || t - k >= 0)) {
					const long long step = DENSE ? 0 : static_cast<long long>(t - k) * p.channels + c;
					store_raw<T, W, SPLIT>(DENSE ? reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(dz) + outRound + offset[k]) : dz + step, oz, second);
					store_raw<T, W, SPLIT>(DENSE ? reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(df) + outRound + offset[k]) : df + step, of, second);
					if constexpr(INPUT) {
						store_raw<T, W, SPLIT>(DENSE ? reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(di) + outRound + offset[k]) : di + step, oi, second);
					}
				}
			}
		};
		if(whole) apply(Yes());
		else apply(No());
		if constexpr(DENSE) {
			z.base -= roundBytes;
			h.base -= roundBytes;
			if constexpr(INPUT) i.base -= roundBytes;
		}
		if(nextWhole) load_rest(t - stride, outRound - roundBytes, Yes());
		else load_rest(t - stride, outRound - roundBytes, No());
		outRound -= roundBytes;
		t -= stride;
	}
	if(blocks > 1) cg::this_cluster().sync();
	if(on && p.last != nullptr && rank == 0 && warp == 0) store_state<W>(p.last, state0, carry, second);
}

// ---- the same fed by TMA ----------------------------------------------------------------------------------------------
// Long sequences whose rows begin on 16-byte boundaries: a warp's stretches come as boxes of S steps x 128 bytes into a ring of its
// own in shared memory, several rounds ahead, by one lane's instructions; steps and channels that do not exist come as zeros.  Loads into
// registers are one round ahead at most: the kernels above take 1.1 to 1.3 times as long (launch()'s comment).  A ring needs no
// barrier for free stages: its warp has read a stage when it asks for the next round in its place.

struct Maps {
	CUtensorMap z, f, i, dh, h;
};
__host__ __device__ constexpr int backward_arrays(bool input, bool stored) { return 3 + (stored ? 1 : 0) + (input ? 1 : 0); }

// One warp's ring: `arrays` boxes a stage.
template<int S>
struct Ring {
	static constexpr int BOX_BYTES = S * 128;
	uint8_t* stages;
	uint64_t* full;
	int* asked; // rounds asked for
	int arrays, depth;
	__device__ __forceinline__ const uint32_t* box(int round, int array) const
	{
		return reinterpret_cast<const uint32_t*>(stages + ((round % depth) * arrays + array) * BOX_BYTES);
	}
	__device__ __forceinline__ uint32_t begin(int round) const // by one lane
	{
		*asked = round + 1;
		mbar_arrive_expect_tx(full + round % depth, arrays * BOX_BYTES);
		return smem_u32(stages + (round % depth) * arrays * BOX_BYTES);
	}
	__device__ __forceinline__ void wait(int round, volatile int* abortFlag, int* status) const
	{
		wait_warp(full + round % depth, (round / depth) & 1, abortFlag, status, (KERNEL_ID << 8) | 2);
	}
	// Once a wait has given up: what was asked for lands before the shared memory goes (rounds that have landed come back at once).
	__device__ __forceinline__ void drain() const
	{
		__syncwarp();
		for(int round = max(*asked - depth, 0); round < *asked; ++round) {
			int ignored = 0;
			mbar_wait_bounded_warp(full + round % depth, (round / depth) & 1, &ignored, nullptr, 0);
		}
	}
};

template<int S, int DEPTH>
__device__ __forceinline__ Ring<S> make_ring(uint8_t* room, uint64_t (&bars)[MAX_WARPS][DEPTH], int (&asked)[MAX_WARPS], int arrays)
{
	const int warp = threadIdx.x >> 5;
	Ring<S> ring = { room + warp * DEPTH * arrays * Ring<S>::BOX_BYTES, bars[warp], asked + warp, arrays, DEPTH };
	if((threadIdx.x & 31) == 0) {
		asked[warp] = 0;
		for(int k = 0; k < DEPTH; ++k) mbar_init(ring.full + k, 1);
		mbar_init_fence();
	}
	return ring; // begin_sharing() is the barrier behind this
}

// The stage has been read by the whole warp: its next round may be asked for.
__device__ __forceinline__ void stage_read()
{
	__syncwarp();
	fence_proxy_async_smem();
}

template<typename T, int W, bool INPUT, int S, int DEPTH, bool STATES>
__global__ void __launch_bounds__(MAX_WARPS * 32, 2) recurrence_forward_stream_kernel(const RecurrenceParams p, const __grid_constant__ Maps maps)
{
	extern __shared__ __align__(128) uint8_t sharedRoom[];
	__shared__ uint64_t arrived[2];
	__shared__ int abortFlag;
	__shared__ uint64_t bars[MAX_WARPS][DEPTH];
	__shared__ int asked[MAX_WARPS];
	constexpr int ARRAYS = INPUT ? 3 : 2;
	const int blocks = gridDim.y, rank = blockIdx.y;
	const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	constexpr int BOX_BYTES = Ring<S>::BOX_BYTES;
	const Ring<S> ring = make_ring<S, DEPTH>(sharedRoom + shared_bytes(warps, blocks, W), bars, asked, ARRAYS);
	const Shared<W> s = begin_sharing<W>(sharedRoom, arrived, &abortFlag, warps, blocks);
	const int b = blockIdx.z;
	const int tile = blockIdx.x * 32 * W;
	const int c = tile + lane * W;
	const bool on = c < p.channels;
	const int n = sequence_length(p, b);
	const int span = warps * S, stride = span * blocks;
	const Stretches<STATES> all_steps = { n };
	const int first = all_steps.begin(stride) + rank * span + warp * S;
	T* const out = static_cast<T*>(p.out) + static_cast<long long>(b) * p.length * p.channels;
	uint8_t* outRound = reinterpret_cast<uint8_t*>(out) + static_cast<long long>(all_steps.begin(stride)) * p.channels * static_cast<long long>(sizeof(T));
	const long long roundBytes = static_cast<long long>(stride) * p.channels * sizeof(T);
	uint32_t offset[S];
#pragma unroll
	for(int k = 0; k < S; ++k) offset[k] = (static_cast<uint32_t>(rank * span + warp * S + k) * p.channels + c) * static_cast<uint32_t>(sizeof(T));
	const long long state0 = static_cast<long long>(b) * p.channels + c;
	Num<W> carry = all<W>(0.f);
	if(on) carry = load_state<W>(p.first, state0, 1);
	auto ask = [&](int round) {
		const int t = first + round * stride;
		if(t >= n || lane != 0 || *static_cast<volatile int*>(s.abortFlag) != 0) return; // (a box may lie in front of step 0: rounds that a warp leaves out are the last ones)
		const uint32_t at = ring.begin(round);
		uint64_t* const bar = ring.full + round % DEPTH;
		tma_load_3d(at, &maps.z, bar, tile, t, b);
		tma_load_3d(at + BOX_BYTES, &maps.f, bar, tile, t, b);
		if constexpr(INPUT) tma_load_3d(at + 2 * BOX_BYTES, &maps.i, bar, tile, t, b);
	};
	for(int k = 0; k < DEPTH; ++k) ask(k);
	int t = first;
	for(int round = 0; round * stride < n; ++round, t += stride) {
		Num<W> a[S], h[S];
		Fold<W> mine = { all<W>(1.f), all<W>(0.f) };
		auto fold = [&](auto full) {
			const uint32_t *z = ring.box(round, 0) + lane, *f = ring.box(round, 1) + lane, *i = ring.box(round, INPUT ? 2 : 0) + lane;
#pragma unroll
			for(int k = 0; k < S; ++k) {
				const bool in = decltype(full)::value || all_steps.in(t + k);
				const Gate<W> forget = gate<T, W>(f[k * 32]);
				Num<W> take = forget.take;
				if constexpr(INPUT) take = sigmoid<T, W>(i[k * 32]);
				a[k] = pick<W>(in, forget.keep, all<W>(1.f));
				h[k] = pick<W>(in, mul(take, number<T, W>(z[k * 32])), all<W>(0.f));
				mine.h = fma(a[k], mine.h, h[k]);
				mine.a = mul(mine.a, a[k]);
			}
		};
		const bool whole = all_steps.whole(t, S);
		if(t < n) ring.wait(round, s.abortFlag, p.status);
		if(whole) fold(Yes());
		else if(t < n) fold(No());
		stage_read();
		ask(round + DEPTH);
		Num<W> state;
		join<W>(s, mine, round, rank, blocks, warps, p.status, carry, state, [] {});
		auto apply = [&](auto full) {
#pragma unroll
			for(int k = 0; k < S; ++k) {
				state = fma(a[k], state, h[k]);
				if(on && (decltype(full)::value || t + k < n)) store_raw<T, W, false>(reinterpret_cast<T*>(outRound + offset[k]), state, 1);
			}
		};
		if constexpr(STATES) {
#pragma unroll
			for(int k = 0; k < S; ++k) {
				if(k % STEPS == 0 && on && t + k > 0) store_parts<T, false>(reinterpret_cast<T*>(outRound + offset[k]), p.channels, state, 1);
				state = fma(a[k], state, h[k]);
			}
		} else {
			if(whole) apply(Yes());
			else if(t < n) apply(No());
		}
		outRound += roundBytes;
	}
	if(*static_cast<volatile int*>(s.abortFlag) != 0) ring.drain();
	// behind the sequence the results are zeros
	for(int k = n + rank * warps + warp; !STATES && k < p.length; k += blocks * warps) {
		if(on) store_raw<T, W, false>(out + static_cast<long long>(k) * p.channels + c, all<W>(0.f), 1);
	}
	if(blocks > 1) cg::this_cluster().sync(); // nobody leaves while its shared memory may be written
	// behind it: the initial state, which all blocks read, may lie in the same place
	if(on && p.last != nullptr && rank == 0 && warp == 0) store_state<W>(p.last, state0, carry, 1);
}

template<typename T, int W, bool INPUT, int S, int DEPTH>
__global__ void __launch_bounds__(MAX_WARPS * 32, 2) recurrence_backward_stream_kernel(const RecurrenceParams p, const __grid_constant__ Maps maps)
{
	extern __shared__ __align__(128) uint8_t sharedRoom[];
	__shared__ uint64_t arrived[2];
	__shared__ int abortFlag;
	__shared__ uint64_t bars[MAX_WARPS][DEPTH];
	__shared__ int asked[MAX_WARPS];
	constexpr bool STORED = sizeof(T) == 4; // the result holds the states as they were
	constexpr int ARRAYS = backward_arrays(INPUT, STORED), INPUT_AT = ARRAYS - 1;
	static_assert(STORED || S % STEPS == 0, "a state in front of every stretch");
	const int blocks = gridDim.y, rank = blockIdx.y;
	const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	constexpr int BOX_BYTES = Ring<S>::BOX_BYTES;
	const Ring<S> ring = make_ring<S, DEPTH>(sharedRoom + shared_bytes(warps, blocks, W), bars, asked, ARRAYS);
	const Shared<W> s = begin_sharing<W>(sharedRoom, arrived, &abortFlag, warps, blocks);
	const int b = blockIdx.z;
	const int tile = blockIdx.x * 32 * W;
	const int c = tile + lane * W;
	const bool on = c < p.channels;
	const int n = sequence_length(p, b);
	const int span = warps * S, stride = span * blocks;
	const int back = rank * span + warp * S; // steps between the round's last one and this thread's first
	const long long roundBytes = static_cast<long long>(stride) * p.channels * sizeof(T);
	const long long sequence = static_cast<long long>(b) * p.length * p.channels;
	long long outRound = static_cast<long long>(n - stride) * p.channels * static_cast<long long>(sizeof(T));
	uint8_t* const dz = reinterpret_cast<uint8_t*>(static_cast<T*>(p.out) + sequence);
	uint8_t* const df = reinterpret_cast<uint8_t*>(static_cast<T*>(p.df) + sequence);
	uint8_t* const di = INPUT ? reinterpret_cast<uint8_t*>(static_cast<T*>(p.di) + sequence) : nullptr;
	uint32_t offset[S];
#pragma unroll
	for(int k = 0; k < S; ++k) offset[k] = (static_cast<uint32_t>(stride - 1 - back - k) * p.channels + c) * static_cast<uint32_t>(sizeof(T));
	const long long state0 = static_cast<long long>(b) * p.channels + c;
	Num<W> carry = all<W>(0.f), first = all<W>(0.f);
	if(on) {
		carry = load_state<W>(p.lastDiff, state0, 1);
		first = load_state<W>(p.first, state0, 1);
	}
	auto ask = [&](int round) {
		const int t = n - 1 - back - round * stride, from = t - S + 1; // a box may begin in front of step 0
		if(t < 0 || lane != 0 || *static_cast<volatile int*>(s.abortFlag) != 0) return;
		const uint32_t at = ring.begin(round);
		uint64_t* const bar = ring.full + round % DEPTH;
		tma_load_3d(at, &maps.f, bar, tile, from, b);
		tma_load_3d(at + BOX_BYTES, &maps.dh, bar, tile, from, b);
		tma_load_3d(at + 2 * BOX_BYTES, &maps.z, bar, tile, from, b);
		if constexpr(STORED) tma_load_3d(at + 3 * BOX_BYTES, &maps.h, bar, tile, from - 1, b); // the step before
		if constexpr(INPUT) tma_load_3d(at + INPUT_AT * BOX_BYTES, &maps.i, bar, tile, from, b);
	};
	for(int k = 0; k < DEPTH; ++k) ask(k);
	// behind the sequence the gradients are zeros
	for(int k = n + rank * warps + warp; k < p.length; k += blocks * warps) {
		const long long at = (static_cast<long long>(k) * p.channels + c) * static_cast<long long>(sizeof(T));
		if(!on) break;
		store_raw<T, W, false>(reinterpret_cast<T*>(dz + at), all<W>(0.f), 1);
		store_raw<T, W, false>(reinterpret_cast<T*>(df + at), all<W>(0.f), 1);
		if constexpr(INPUT) store_raw<T, W, false>(reinterpret_cast<T*>(di + at), all<W>(0.f), 1);
	}
	int t = n - 1 - back;
	uint2 parts = make_uint2(0u, 0u); // the state in front of the stretch, a round ahead
	auto load_next = [&](int t, long long round) {
		if constexpr(!STORED) {
			if(on && t - S >= 0) parts = load_parts<T, false>(reinterpret_cast<const T*>(dz + round + offset[S - 1]), p.channels, 1);
		}
	};
	load_next(t, outRound);
	for(int round = 0; round * stride < n; ++round, t -= stride) {
		Num<W> a[S], u[S];
		Fold<W> mine = { all<W>(1.f), all<W>(0.f) };
		const uint32_t *f = ring.box(round, 0) + lane, *d = ring.box(round, 1) + lane, *z = ring.box(round, 2) + lane,
			*h = ring.box(round, STORED ? 3 : 0) + lane, *i = ring.box(round, INPUT ? INPUT_AT : 0) + lane;
		auto fold = [&](auto full) {
#pragma unroll
			for(int k = 0; k < S; ++k) {
				const int row = (S - 1 - k) * 32;
				const bool in = decltype(full)::value || t - k >= 0;
				const Gate<W> forget = gate<T, W>(f[row]);
				a[k] = pick<W>(in, forget.keep, all<W>(1.f));
				u[k] = forget.take;
				mine.h = mul(a[k], add(mine.h, number<T, W>(d[row]))); // this step's own part is a dh
				mine.a = mul(mine.a, a[k]);
			}
		};
		const bool whole = t - S >= 0;
		if(t >= 0) ring.wait(round, s.abortFlag, p.status);
		if(whole) fold(Yes());
		else if(t >= 0) fold(No());
		// d(forget) of a step: S times this, which takes the state in front of it
		Num<W> slope[S];
		auto slopes = [&](auto full) {
			Num<W> running = first;
			if constexpr(!STORED && decltype(full)::value) running = from_parts<W>(parts);
#pragma unroll
			for(int k = S - 1; k >= 0; --k) {
				const int row = (S - 1 - k) * 32;
				const Num<W> value = number<T, W>(z[row]);
				Num<W> before = running;
				if constexpr(STORED) {
					before = number<T, W>(h[row]);
					if(!decltype(full)::value && t - k == 0) before = first;
				} else { // steps in front of the first one: a is one, the value zero
					Num<W> take = u[k];
					if constexpr(INPUT) take = sigmoid<T, W>(i[row]);
					running = fma(a[k], before, mul(take, value));
				}
				slope[k] = mul(mul(a[k], u[k]), INPUT ? before : fma(value, all<W>(-1.f), before));
			}
		};
		Num<W> state;
		join<W>(s, mine, round, rank, blocks, warps, p.status, carry, state, [&] {
			if(whole) slopes(Yes());
			else if(t >= 0) slopes(No());
			load_next(t - stride, outRound - roundBytes);
		});
		auto apply = [&](auto full) {
#pragma unroll
			for(int k = 0; k < S; ++k) {
				const int row = (S - 1 - k) * 32;
				const Num<W> S = add(state, number<T, W>(d[row]));
				Num<W> oz, oi = S;
				if constexpr(INPUT) {
					const Gate<W> take = gate<T, W>(i[row]);
					oz = mul(S, take.keep);
					oi = mul(mul(oz, number<T, W>(z[row])), take.take);
				} else {
					oz = mul(S, u[k]);
				}
				const Num<W> of = mul(S, slope[k]);
				state = mul(a[k], S);
				if(on && (decltype(full)::value || t - k >= 0)) {
					store_raw<T, W, false>(reinterpret_cast<T*>(dz + outRound + offset[k]), oz, 1);
					store_raw<T, W, false>(reinterpret_cast<T*>(df + outRound + offset[k]), of, 1);
					if constexpr(INPUT) store_raw<T, W, false>(reinterpret_cast<T*>(di + outRound + offset[k]), oi, 1);
				}
			}
		};
		if(whole) apply(Yes());
		else if(t >= 0) apply(No());
		stage_read();
		ask(round + DEPTH);
		outRound -= roundBytes;
	}
	if(*static_cast<volatile int*>(s.abortFlag) != 0) ring.drain();
	if(blocks > 1) cg::this_cluster().sync();
	if(on && p.last != nullptr && rank == 0 && warp == 0) store_state<W>(p.last, state0, carry, 1);
}

using Kernel = void (*)(const RecurrenceParams);

enum Pass {
	FORWARD,
	STATES,  // of 16-bit types, in front of BACKWARD: the states in front of every STEPS-th step
	BACKWARD
};

template<typename T, int W, bool SPLIT, Pass PASS>
Kernel kernel_of(bool input, bool dense)
{
	if(PASS == BACKWARD) {
		if(dense) return input ? recurrence_backward_kernel<T, W, true, true, SPLIT> : recurrence_backward_kernel<T, W, false, true, SPLIT>;
		return input ? recurrence_backward_kernel<T, W, true, false, SPLIT> : recurrence_backward_kernel<T, W, false, false, SPLIT>;
	}
	constexpr bool S = PASS == STATES;
	if(dense) return input ? recurrence_forward_kernel<T, W, true, true, SPLIT, S> : recurrence_forward_kernel<T, W, false, true, SPLIT, S>;
	return input ? recurrence_forward_kernel<T, W, true, false, SPLIT, S> : recurrence_forward_kernel<T, W, false, false, SPLIT, S>;
}

template<Pass PASS>
Kernel kernel_for(int type, bool pair, bool input, bool dense)
{
	if(type == NB200_TYPE_FP16) return pair ? kernel_of<__half, 2, false, PASS>(input, dense) : kernel_of<__half, 2, true, PASS>(input, dense);
	if(type == NB200_TYPE_BF16) return pair ? kernel_of<__nv_bfloat16, 2, false, PASS>(input, dense) : kernel_of<__nv_bfloat16, 2, true, PASS>(input, dense);
	if constexpr(PASS == STATES) return nullptr;
	else return kernel_of<float, 1, false, PASS>(input, dense);
}

// Rounds that a warp's loads are ahead of its work, by what fits beside one another in 16 or more warps' shared memory.
constexpr int FORWARD_STEPS = 16, FORWARD_DEPTH = 2, FORWARD_INPUT_DEPTH = 2, BACKWARD_STEPS = 8, BACKWARD_DEPTH = 2,
	BACKWARD_INPUT_STEPS = 8, BACKWARD_INPUT_STEPS_FP32 = 16, BACKWARD_INPUT_DEPTH = 2; // (16 steps of 16-bit gates and states spill: 570 us for 275)

using StreamKernel = void (*)(const RecurrenceParams, const Maps);

template<Pass PASS, typename T, int W>
StreamKernel stream_of(bool input)
{
	if(PASS == BACKWARD) return input ? recurrence_backward_stream_kernel<T, W, true, W == 1 ? BACKWARD_INPUT_STEPS_FP32 : BACKWARD_INPUT_STEPS, BACKWARD_INPUT_DEPTH>
		: recurrence_backward_stream_kernel<T, W, false, BACKWARD_STEPS, BACKWARD_DEPTH>;
	return input ? recurrence_forward_stream_kernel<T, W, true, FORWARD_STEPS, FORWARD_INPUT_DEPTH, PASS == STATES>
		: recurrence_forward_stream_kernel<T, W, false, FORWARD_STEPS, FORWARD_DEPTH, PASS == STATES>;
}
template<Pass PASS>
StreamKernel stream_for(int type, bool input)
{
	if(type == NB200_TYPE_FP16) return stream_of<PASS, __half, 2>(input);
	if(type == NB200_TYPE_BF16) return stream_of<PASS, __nv_bfloat16, 2>(input);
	if constexpr(PASS == STATES) return nullptr;
	else return stream_of<PASS, float, 1>(input);
}
// Maps of the operands; false where one of them does not lie as TMA takes it (or a step's distance does not fit 32 bits of a round's offsets).
bool make_maps(Maps& maps, int type, bool backward, const RecurrenceParams& p, int batch, int steps)
{
	const int size = type_size(type);
	const long long dense = p.channels;
	if(dense * size % 16 != 0 || dense * size * (MAX_CLUSTER + 1) * MAX_WARPS * FORWARD_STEPS >= (1ll << 32)) return false;
	auto one = [&](CUtensorMap& map, const void* base, long long batchStride, long long row) {
		return sequence_map(&map, base, type, p.channels, p.length, batch, row, batch > 1 ? batchStride : row * p.length, steps);
	};
	return one(maps.z, p.z, p.zBatch, p.zRow) && one(maps.f, p.f, p.fBatch, p.fRow) && (p.i == nullptr || one(maps.i, p.i, p.iBatch, p.iRow))
		&& (!backward || one(maps.dh, p.dh, p.dhBatch, p.dhRow)) && (!backward || size != 4 || one(maps.h, p.h, dense * p.length, dense));
}

// How many warps and blocks share a sequence's time axis: the fewest that fill three quarters of the warps that the SMs hold
// (16, or 24 in the kernels of fewer registers); up to four warps before more blocks, which exchange folds through the cluster.  Measured,
// forward + both backward passes by TMA: 16 x 2048 x 2048 bf16 75 + 192 us in blocks of four, 105 + 269 of two, 81 + 206 of eight, 81 + 210 in
// clusters of two; 64 x 100 x 4096 fp16 40 + 91 in blocks of two, 50 + 110 of four, 60 + 144 of eight.  Where there are few channels (2 x 16384 x 2048 bf16)
// clusters of eight blocks of four: 86 + 216, in clusters of four 120 + 300, without 373 + 958.  By loads into registers the three take 94 + 248,
// 43 + 112 and 105 + 289 in the same shapes.  fp32: 16 x 2048 x 2048 142 + 290 (0.87 and 0.85 of the copy rate), 24 x 1021 x 1024 with input
// gates 78 + 142.
int launch(int type, bool pair, Pass pass, RecurrenceParams p, int batch, cudaStream_t stream)
{
	const bool backward = pass == BACKWARD;
	const bool input = p.i != nullptr;
	const long long row = p.channels;
	const bool dense = row * type_size(type) * (MAX_CLUSTER + 1) * MAX_WARPS * STEPS < (1ll << 32)
		&& (p.length <= 1 || (p.zRow == row && p.fRow == row && (!input || p.iRow == row) && (!backward || p.dhRow == row)));
	const Kernel kernel = backward ? kernel_for<BACKWARD>(type, pair, input, dense) : pass == STATES ? kernel_for<STATES>(type, pair, input, dense)
		: kernel_for<FORWARD>(type, pair, input, dense);
	p.status = device_status_word();
	const int channelsPerLane = type == NB200_TYPE_FP32 ? 1 : 2;
	const int tiles = (p.channels + 32 * channelsPerLane - 1) / (32 * channelsPerLane);
	const int stretches = (p.length + STEPS - 1) / STEPS;
	const long long groups = static_cast<long long>(tiles) * batch;
	const long long wanted = static_cast<long long>(sm_count()) * (backward || channelsPerLane == 2 ? 12 : 18);
	int warps = stretches < 2 ? 1 : 2, blocks = 1;
	auto more = [&](int w, int n) { return groups * w * n < wanted && w * n < stretches; };
	while(warps < 4 && more(warps, blocks)) warps *= 2;
	while(blocks < MAX_CLUSTER && more(warps, blocks)) blocks *= 2;
	while(warps < MAX_WARPS && more(warps, blocks)) warps *= 2;
	Maps maps = {};
	StreamKernel stream_kernel = nullptr;
	int depth = 0;
	const int steps = !backward ? FORWARD_STEPS : !input ? BACKWARD_STEPS : type == NB200_TYPE_FP32 ? BACKWARD_INPUT_STEPS_FP32 : BACKWARD_INPUT_STEPS;
	// (their stores go by whole words; maps ask more of what is read)
	if((pair || channelsPerLane == 1) && p.length >= 2 * warps * blocks * steps && make_maps(maps, type, backward, p, batch, steps)) {
		stream_kernel = backward ? stream_for<BACKWARD>(type, input) : pass == STATES ? stream_for<STATES>(type, input) : stream_for<FORWARD>(type, input);
		depth = backward ? (input ? BACKWARD_INPUT_DEPTH : BACKWARD_DEPTH) : (input ? FORWARD_INPUT_DEPTH : FORWARD_DEPTH);
	}
	cudaLaunchConfig_t config = {};
	config.blockDim = dim3(warps * 32);
	config.gridDim = dim3(tiles, blocks, batch);
	config.dynamicSmemBytes = shared_bytes(warps, blocks, channelsPerLane);
	config.stream = stream;
	cudaLaunchAttribute attribute[1];
	attribute[0].id = cudaLaunchAttributeClusterDimension;
	attribute[0].val.clusterDim.x = 1;
	attribute[0].val.clusterDim.y = blocks;
	attribute[0].val.clusterDim.z = 1;
	config.attrs = attribute;
	config.numAttrs = blocks > 1 ? 1 : 0;
	if(stream_kernel != nullptr) {
		const int arrays = backward ? backward_arrays(input, type == NB200_TYPE_FP32) : 2 + (input ? 1 : 0);
		const int perWarp = depth * arrays * steps * 128;
		config.dynamicSmemBytes += static_cast<size_t>(warps) * perWarp;
		// the most that the kernel is ever launched with: another thread may be between this and its own launch
		cudaFuncSetAttribute(stream_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
			MAX_WARPS * perWarp + shared_bytes(MAX_WARPS, MAX_CLUSTER, channelsPerLane));
		cudaLaunchKernelEx(&config, stream_kernel, static_cast<const RecurrenceParams&>(p), static_cast<const Maps&>(maps));
	} else {
		cudaLaunchKernelEx(&config, kernel, static_cast<const RecurrenceParams&>(p));
	}
	count_launch();
	return check_launch();
}

// 16-bit channels go in pairs where every pair lies in one aligned word
struct Strided {
	const void* p;
	long long batch, row;
};
bool pairs_aligned(int type, int batch, int length, int channels, const Strided* s, int n)
{
	if(type == NB200_TYPE_FP32 || channels % 2 != 0) return false;
	for(int k = 0; k < n; ++k) {
		if(s[k].p == nullptr) continue;
		if((reinterpret_cast<uintptr_t>(s[k].p) & 3u) != 0) return false;
		if((batch > 1 && s[k].batch % 2 != 0) || (length > 1 && s[k].row % 2 != 0)) return false;
	}
	return true;
}

// Elements from an operand's first to behind its last.
long long extent(const nb200_recurrence_desc* d, long long batch, long long row)
{
	return (d->batch - 1) * batch + (d->length - 1) * row + d->channels;
}
bool apart(const void* a, long long aBytes, const void* b, long long bBytes)
{
	const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
	return a == nullptr || b == nullptr || (x < y ? y - x >= static_cast<uintptr_t>(aBytes) : x - y >= static_cast<uintptr_t>(bBytes));
}

bool desc_valid(int type, const nb200_recurrence_desc* d)
{
	if(d == nullptr || !type_valid(type) || d->batch < 0 || d->length < 0 || d->channels < 0) return false;
	const long long rows[] = { d->update_row, d->forget_row, d->input_row };
	const long long batches[] = { d->update_batch, d->forget_batch, d->input_batch };
	for(int k = 0; k < 3; ++k) {
		if(rows[k] < 0 || batches[k] < 0) return false;
	}
	return true;
}

} // namespace

} // namespace nb200

using namespace nb200;

extern "C" {

int nb200_gated_recurrence(void* stream, int type, const nb200_recurrence_desc* d, const void* update, const void* forget,
	const void* input, const float* initial_state, const int* lengths, void* result, float* final_state)
{
	if(!desc_valid(type, d)) return NB200_EINVAL;
	if(d->batch == 0 || d->channels == 0) return NB200_OK;
	if(d->length > 0 && (update == nullptr || forget == nullptr || result == nullptr)) return NB200_EINVAL;
	if(!type_aligned(update, type) || !type_aligned(forget, type) || !type_aligned(input, type) || !type_aligned(result, type)
		|| !words_aligned(initial_state, final_state, lengths)) return NB200_EINVAL;
	if(d->batch > MAX_BATCH || d->length > (1 << 30) || d->channels > (1 << 30)) return NB200_ETOOBIG;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	RecurrenceParams p = {};
	p.z = update; p.f = forget; p.i = input; p.out = result; p.first = initial_state; p.last = final_state; p.lengths = lengths;
	p.zBatch = d->update_batch; p.zRow = d->update_row; p.fBatch = d->forget_batch; p.fRow = d->forget_row;
	p.iBatch = d->input_batch; p.iRow = d->input_row;
	p.length = d->length; p.channels = d->channels;
	const Strided all[] = { { update, d->update_batch, d->update_row }, { forget, d->forget_batch, d->forget_row },
		{ input, d->input_batch, d->input_row }, { result, 0, 0 } };
	return launch(type, pairs_aligned(type, d->batch, d->length, d->channels, all, 4), FORWARD, p, d->batch, as_stream(stream));
}

int nb200_gated_recurrence_backward(void* stream, int type, const nb200_recurrence_desc* d, const void* result_diff,
	long long result_diff_batch, long long result_diff_row, const void* result, const void* update, const void* forget,
	const void* input, const float* initial_state, const float* final_state_diff, const int* lengths, void* update_diff,
	void* forget_diff, void* input_diff, float* initial_state_diff)
{
	if(!desc_valid(type, d) || result_diff_batch < 0 || result_diff_row < 0) return NB200_EINVAL;
	if(d->batch == 0 || d->channels == 0) return NB200_OK;
	if(d->length > 0 && (result_diff == nullptr || result == nullptr || update == nullptr || forget == nullptr
		|| update_diff == nullptr || forget_diff == nullptr)) return NB200_EINVAL;
	if(d->length > 0 && (input == nullptr) != (input_diff == nullptr)) return NB200_EINVAL;
	const void* const typed[] = { result_diff, result, update, forget, input, update_diff, forget_diff, input_diff };
	for(const void* t : typed) {
		if(!type_aligned(t, type)) return NB200_EINVAL;
	}
	if(!words_aligned(initial_state, final_state_diff, lengths, initial_state_diff)) return NB200_EINVAL;
	if(type != NB200_TYPE_FP32 && d->length > 0) { // update_diff holds states before it holds gradients
		const long long size = 2, own = extent(d, static_cast<long long>(d->length) * d->channels, d->channels) * size;
		if(!apart(update_diff, own, result_diff, extent(d, result_diff_batch, result_diff_row) * size)
			|| !apart(update_diff, own, update, extent(d, d->update_batch, d->update_row) * size)
			|| !apart(update_diff, own, forget, extent(d, d->forget_batch, d->forget_row) * size)
			|| !apart(update_diff, own, input, extent(d, d->input_batch, d->input_row) * size)) return NB200_EINVAL;
	}
	if(d->batch > MAX_BATCH || d->length > (1 << 30) || d->channels > (1 << 30)) return NB200_ETOOBIG;
	if(device_status_word() == nullptr) return NB200_ENODEVICE;
	RecurrenceParams p = {};
	p.z = update; p.f = forget; p.i = input; p.dh = result_diff; p.h = result;
	p.out = update_diff; p.df = forget_diff; p.di = input_diff;
	p.first = initial_state; p.lastDiff = final_state_diff; p.last = initial_state_diff; p.lengths = lengths;
	p.zBatch = d->update_batch; p.zRow = d->update_row; p.fBatch = d->forget_batch; p.fRow = d->forget_row;
	p.iBatch = d->input_batch; p.iRow = d->input_row; p.dhBatch = result_diff_batch; p.dhRow = result_diff_row;
	p.length = d->length; p.channels = d->channels;
	const Strided all[] = { { update, d->update_batch, d->update_row }, { forget, d->forget_batch, d->forget_row },
		{ input, d->input_batch, d->input_row }, { result_diff, result_diff_batch, result_diff_row }, { result, 0, 0 },
		{ update_diff, 0, 0 }, { forget_diff, 0, 0 }, { input_diff, 0, 0 } };
	const bool pair = pairs_aligned(type, d->batch, d->length, d->channels, all, 8);
	if(type != NB200_TYPE_FP32 && d->length > STEPS) { // the states in front of stretches, in update_diff's memory
		RecurrenceParams q = p;
		q.last = nullptr;
		const int rc = launch(type, pair, STATES, q, d->batch, as_stream(stream));
		if(rc != NB200_OK) return rc;
	}
	return launch(type, pair, BACKWARD, p, d->batch, as_stream(stream));
}

} // extern "C"
