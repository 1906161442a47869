// Element types of the row, sequence and loss kernels: fp32, fp16 and bf16 data in global memory, fp32 in registers.
// Conversions to 16 bits happen once, at the final store, to nearest even.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace nb200 {

inline int type_size(int type) { return type == NB200_TYPE_FP32 ? 4 : 2; }
inline bool type_valid(int type) { return type == NB200_TYPE_FP32 || type == NB200_TYPE_FP16 || type == NB200_TYPE_BF16; }
// every address of a row-addressed operand is a multiple of its element's size
inline bool type_aligned(const void* p, int type) { return (reinterpret_cast<uintptr_t>(p) & (type_size(type) - 1)) == 0; }
// and so is that of fp32 and int32 vectors; null is one that is not given
template<typename... P> bool words_aligned(const P*... p) { return ((reinterpret_cast<uintptr_t>(p) | ... | 0u) & 3u) == 0; }

#ifdef __CUDACC__

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template<typename T> __device__ __forceinline__ T from_float(float v);
template<> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template<> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template<> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two 16-bit values in one register, and back.
template<typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template<> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v)
{
	return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template<> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v)
{
	return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); // a bf16 is the upper half of a float
}
template<typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template<> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b)
{
	const __half2 h = __floats2half2_rn(a, b);
	return *reinterpret_cast<const uint32_t*>(&h);
}
template<> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b)
{
	const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
	return *reinterpret_cast<const uint32_t*>(&h);
}

template<typename T> struct PairOf;
template<> struct PairOf<__half> { using type = __half2; };
template<> struct PairOf<__nv_bfloat16> { using type = __nv_bfloat162; };

// 16 bytes as they lie in memory <-> the floats they hold (four or eight).
template<typename T> struct Unit16 {
	static constexpr int N = 16 / static_cast<int>(sizeof(T));
	static __device__ __forceinline__ void unpack(const uint4& r, float* v)
	{
		const uint32_t w[4] = { r.x, r.y, r.z, r.w };
#pragma unroll
		for(int i = 0; i < 4; ++i) {
			const float2 f = unpack2<T>(w[i]);
			v[2 * i] = f.x;
			v[2 * i + 1] = f.y;
		}
	}
	static __device__ __forceinline__ uint4 pack(const float* v)
	{
		return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
	}
};
template<> struct Unit16<float> {
	static constexpr int N = 4;
	static __device__ __forceinline__ void unpack(const uint4& r, float* v)
	{
		v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
	}
	static __device__ __forceinline__ uint4 pack(const float* v)
	{
		return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
	}
};

// ---- rows in 16-byte units of memory -----------------------------------------------------------------------------------
// A row is cut into the aligned 16-byte units that it touches, so that rows of any width and first address move at full
// rate: the units at its two ends hold elements of the neighbouring rows too, which the caller leaves out of what it
// computes.  V: elements of a unit, or 1 for units of single elements (operands that are aligned differently).
// A row and the matrix that it lies in.  A unit is addressed by the column of its element 0, negative at a row's head.
template<typename T, int V>
struct Row {
	const T* p;      // element 0 of the row
	const T* begin;  // of the matrix
	const T* end;
};

// A unit as it lies in memory, neighbouring rows' elements included (whole_floats leaves them out): what has just been asked
// for is not looked at here, so that loads stay under way.  EDGES false: rows that begin and end with whole units.
template<typename T, int V, bool EDGES = true>
__device__ __forceinline__ void load_unit(const Row<T, V>& row, int first, int width, uint4& raw)
{
	if constexpr(V == 1) {
		raw.x = 0u;
		if(first < width) {
			if constexpr(sizeof(T) == 4) raw.x = __float_as_uint(reinterpret_cast<const float*>(row.p)[first]);
			else raw.x = reinterpret_cast<const unsigned short*>(row.p)[first];
		}
	} else {
		const T* const at = row.p + first;
		raw = make_uint4(0u, 0u, 0u, 0u);
		if(first >= width) return;
		if(!EDGES || (at >= row.begin && at + V <= row.end)) {
			raw = *reinterpret_cast<const uint4*>(at);
		} else { // the first unit of the first row, the last one of the last
			float v[V];
#pragma unroll
			for(int j = 0; j < V; ++j) v[j] = first + j >= 0 && first + j < width ? to_float(at[j]) : 0.f;
			raw = Unit16<T>::pack(v);
		}
	}
}

template<typename T, int V>
__device__ __forceinline__ void unit_floats(const uint4& raw, float* v)
{
	if constexpr(V == 1) {
		if constexpr(sizeof(T) == 4) v[0] = __uint_as_float(raw.x);
		else v[0] = unpack2<T>(raw.x).x;
	} else {
		Unit16<T>::unpack(raw, v);
	}
}

template<typename T, int V, bool EDGES = true>
__device__ __forceinline__ void store_unit(T* row, int first, int width, const float* v)
{
	if constexpr(V == 1) {
		if(first < width) row[first] = from_float<T>(v[0]);
	} else if constexpr(!EDGES) {
		if(first < width) *reinterpret_cast<uint4*>(row + first) = Unit16<T>::pack(v);
	} else {
		if(first >= 0 && first + V <= width) {
			*reinterpret_cast<uint4*>(row + first) = Unit16<T>::pack(v);
		} else {
#pragma unroll
			for(int j = 0; j < V; ++j) {
				if(first + j >= 0 && first + j < width) row[first + j] = from_float<T>(v[j]);
			}
		}
	}
}

template<int V, bool EDGES = true>
__device__ __forceinline__ bool inside(int first, int j, int width)
{
	return V == 1 || !EDGES ? first < width : first + j >= 0 && first + j < width;
}

// the whole unit belongs to the row
template<int V, bool EDGES = true>
__device__ __forceinline__ bool whole(int first, int width)
{
	return V == 1 || !EDGES ? first < width : first >= 0 && first + V <= width;
}

// a unit's floats, with zeros for what is not the row's
template<typename T, int V, bool EDGES>
__device__ __forceinline__ void whole_floats(const uint4& raw, int first, int width, float* v)
{
	unit_floats<T, V>(raw, v);
	if(V > 1 && EDGES && !whole<V>(first, width)) {
#pragma unroll
		for(int j = 0; j < V; ++j) v[j] = inside<V>(first, j, width) ? v[j] : 0.f;
	}
}

// elements by which a row's first address lies behind a 16-byte boundary
template<typename T, int V>
__device__ __forceinline__ int row_offset(const T* row)
{
	return V == 1 ? 0 : static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
}

// Two fp32 operations in one instruction, each rounded like the scalar one.
__device__ __forceinline__ unsigned long long as_pair(float2 v)
{
	return *reinterpret_cast<unsigned long long*>(&v);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
	float2 r;
	asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(*reinterpret_cast<unsigned long long*>(&r)) : "l"(as_pair(a)), "l"(as_pair(b)));
	return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
	float2 r;
	asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(*reinterpret_cast<unsigned long long*>(&r)) : "l"(as_pair(a)), "l"(as_pair(b)));
	return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
	float2 r;
	asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(*reinterpret_cast<unsigned long long*>(&r)) : "l"(as_pair(a)), "l"(as_pair(b)), "l"(as_pair(c)));
	return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ float exp2_fast(float x)
{
	float y;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}

__device__ __forceinline__ float warp_sum_all(float v)
{
#pragma unroll
	for(int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
	return v;
}
__device__ __forceinline__ float warp_max_all(float v)
{
#pragma unroll
	for(int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
	return v;
}

#endif // __CUDACC__

} // namespace nb200
