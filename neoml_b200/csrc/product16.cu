// The 16-bit products behind the cross entropy over a vocabulary (product16.cuh): a persistent tcgen05 kernel.
//
//   warp 0      loads: tiles of A (128 x 64) and B (256 x 64) by TMA into a ring of four stages
//   warp 1      issues the MMAs (128 x 256 x 16) into one of two accumulators of 256 tensor-memory columns
//   warps 4-11  epilogue: two warps per lane quarter, 128 columns each, while the next tile is multiplied
// NARROW: tiles of 64 columns, eight stages, 32 columns per epilogue warp, for products that have few tiles and no K to split.
//
// Operands whose m or n is adjacent in memory need no transposition: the tensor core reads them MN-major.  A box of 64 adjacent
// indices x 64 k lands as 64 rows of 128 bytes; eight rows are a swizzle atom of 1024 bytes (stride byte offset), the next 64
// indices lie 8192 bytes further (leading byte offset).  Every wait is bounded (common.cuh).
//
// The tensor core's own additions cut off rather than round, each MMA a unit or two in the last place of the running sum: all of it in one
// direction where the sum has one sign (7.8e-6 of logits of 4096 positive products, 1.9e-4 of a gradient summed over 30000 entries), less where signs
// alternate (1.3e-6 after 384 MMAs, 3.5e-5 after 11250).  So the K loop is cut into chunks whose sums the epilogue warps add up in registers:
//   fp32        256 elements, the small products first, so that only the 16 MMAs of hi hi work on a sum of full size.  Gradients
//               of 1023 x 768 rows over 30011 entries are 3.7e-7 off then (1.3e-6 with chunks of 1024, 6.7e-7 of 512, fp32 arithmetic 5.7e-7), and
//               take as long: the additions hide behind six times the MMAs.
//   16 bits     512 for the statistics, whose results are fp32: log_sum 1.6e-7 off at any width (whole K 3.2e-7 at 1024, 1.3e-6 at 4096; chunks of
//               256 9e-8).  8192 x 2048 rows over 50257 entries take 1.06 ms (whole 1.02, chunks of 256 1.17).  1024 for gradients, which end as 16 bits: 1.6e-5
//               of the sum above, 1 to 2 % of the time (2048: 3e-5, within the noise; 512: 9e-6, 3 %).  None for dz, which is rounded to 16 bits
//               as it is formed, and none where K is no longer than a chunk.
#include "product16.cuh"

#include <cuda.h>
#include <mutex>

namespace nb200 {

namespace {

constexpr int BM = PRODUCT16_M, BK = PRODUCT16_K;
constexpr int RING_BYTES = 192 * 1024; // four stages, or eight narrow ones
constexpr int A_BYTES = BM * BK * 2;
constexpr int EPILOGUE_WARPS = 8;
constexpr int THREADS = (4 + EPILOGUE_WARPS) * 32;
constexpr int SMEM_BYTES = RING_BYTES + 1024 + 256;
constexpr int KERNEL_ID = 0x70;       // in the status word: (KERNEL_ID << 8) | site
constexpr float LOG2E = 1.4426950408889634f;
enum { SITE_LOAD = 1, SITE_MMA = 2, SITE_MMA_ACC = 3, SITE_EPILOGUE = 4 };

// The products of planes in the order of their MMAs, small ones first: 0 hi, 1 mid, 2 lo.
__device__ constexpr int PLANE_A[6] = { 2, 0, 1, 1, 0, 0 }, PLANE_B[6] = { 0, 2, 1, 0, 1, 0 };
// K blocks that are summed in tensor memory before the epilogue warps add them up in registers.
template<int EPILOGUE, bool FP32> constexpr int CHUNK = FP32 ? 256 / BK : EPILOGUE == PRODUCT16_STATS ? 512 / BK : 1024 / BK;

// MN-major operand of 16-bit elements: see the head of this file.
__device__ __forceinline__ uint64_t desc_across(uint32_t smemAddr)
{
	uint64_t d = 0;
	d |= static_cast<uint64_t>((smemAddr >> 4) & 0x3FFFu);
	d |= static_cast<uint64_t>(8192 >> 4) << 16;
	d |= static_cast<uint64_t>(1024 >> 4) << 32;
	d |= static_cast<uint64_t>(1) << 46;
	d |= static_cast<uint64_t>(2) << 61;
	return d;
}

__device__ __forceinline__ void umma_f16_ss(uint32_t tmemD, uint64_t descA, uint64_t descB, uint32_t idesc, uint32_t accumulate)
{
	asm volatile(
		"{\n\t.reg .pred p;\n\t"
		"setp.ne.b32 p, %4, 0;\n\t"
		"tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
		::"r"(tmemD), "l"(descA), "l"(descB), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void store32(void* p, const uint32_t* v) // 32 bytes, aligned
{
	asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
		::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void load32(const void* p, uint32_t* v)
{
	asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
		: "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p) : "memory");
}

struct Tile {
	int m0, n0, mTile, nTile, split, kBegin, kEnd;
};

template<int BN>
__device__ __forceinline__ Tile tile_of(const Product16Params& p, int tile)
{
	Tile t;
	const int perSplit = p.mTiles * p.nTiles;
	t.split = tile / perSplit;
	const int r = tile - t.split * perSplit;
	if(p.mFast) {
		t.nTile = r / p.mTiles;
		t.mTile = r - t.nTile * p.mTiles;
	} else {
		t.mTile = r / p.nTiles;
		t.nTile = r - t.mTile * p.nTiles;
	}
	t.m0 = t.mTile * BM;
	t.n0 = t.nTile * BN;
	t.kBegin = t.split * p.kBlocksPerSplit;
	t.kEnd = min(p.kBlocks, t.kBegin + p.kBlocksPerSplit);
	return t;
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int bf16)
{
	return bf16 ? pack2<__nv_bfloat16>(a, b) : pack2<__half>(a, b);
}

template<int EPILOGUE, bool A_ACROSS, bool B_ACROSS, bool FP32, bool NARROW, bool CHUNKED>
__global__ void __launch_bounds__(THREADS, 1) product16_kernel(const Product16Params p, const __grid_constant__ CUtensorMap mapA,
	const __grid_constant__ CUtensorMap mapB)
{
	constexpr int TERMS = FP32 ? 6 : 1, CHUNKS = CHUNK<EPILOGUE, FP32>;
	static_assert(CHUNKED || !FP32, "the terms of fp32 operands come chunk by chunk");
	constexpr int BN = NARROW ? PRODUCT16_NARROW : PRODUCT16_N, COLUMNS = BN / 2; // of a tile, and of an epilogue warp
	constexpr int STAGE_BYTES = A_BYTES + BN * BK * 2, STAGES = RING_BYTES / STAGE_BYTES;
	static_assert(STAGES * STAGE_BYTES == RING_BYTES && STAGE_BYTES % 1024 == 0, "stages fill the ring");
	enum { B_FULL = 0, B_EMPTY = STAGES, B_ACCFULL = 2 * STAGES, B_ACCEMPTY = 2 * STAGES + 2, B_DONE = 2 * STAGES + 4, BARS };
	extern __shared__ uint8_t smemRaw[];
	uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~static_cast<uintptr_t>(1023));
	uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + RING_BYTES);
	uint32_t* const tmemSlot = reinterpret_cast<uint32_t*>(bars + BARS);
	volatile int* const abortFlag = reinterpret_cast<volatile int*>(tmemSlot + 1);
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	const uint32_t smemBase = smem_u32(smem);
	if(threadIdx.x == 0) {
		for(int i = 0; i < STAGES; ++i) {
			mbar_init(bars + B_FULL + i, 1);
			mbar_init(bars + B_EMPTY + i, 1);
		}
		for(int i = 0; i < 2; ++i) {
			mbar_init(bars + B_ACCFULL + i, 1);
			mbar_init(bars + B_ACCEMPTY + i, EPILOGUE_WARPS);
		}
		mbar_init(bars + B_DONE, 1);
		mbar_init_fence();
		*abortFlag = 0;
		tma_prefetch_descriptor(&mapA);
		tma_prefetch_descriptor(&mapB);
	}
	if(warp == 2) {
		tmem_alloc(tmemSlot, 512);
		tmem_relinquish();
	}
	tc_fence_before_sync();
	__syncthreads();
	tc_fence_after_sync();
	const uint32_t tmemBase = *tmemSlot;
	const int tiles = p.mTiles * p.nTiles * p.splits;
	dependent_wait();

	if(warp == 0) {
		if(elect_one()) {
			int it = 0;
			bool ok = true;
			// rows of A that do not exist are left out of the box: what their place in the stage holds reaches no other row of the
			// accumulator.  (Leaving out boxes across that lie behind m or n as well, by a test each, made gradients of 1023 x 768 rows over
			// 30011 entries 2.5 % slower.)
			const uint32_t bytes = (A_ACROSS ? A_BYTES : p.boxA * BK * 2) + BN * BK * 2;
			auto load = [&](const Tile& t, int kb, int planeA, int planeB) {
				const int s = it % STAGES;
				if(it >= STAGES && !mbar_wait_bounded(bars + B_EMPTY + s, (it / STAGES - 1) & 1, abortFlag, p.status, (KERNEL_ID << 8) | SITE_LOAD)) return false;
				uint64_t* const full = bars + B_FULL + s;
				const uint32_t a = smemBase + s * STAGE_BYTES, b = a + A_BYTES;
				mbar_arrive_expect_tx(full, bytes);
				const int k = kb * BK;
				if constexpr(A_ACROSS) {
#pragma unroll
					for(int i = 0; i < BM / 64; ++i) tma_load_3d(a + i * 8192, &mapA, full, t.m0 + i * 64, k, planeA);
				} else {
					tma_load_3d(a, &mapA, full, k, t.m0, planeA);
				}
				if constexpr(B_ACROSS) {
#pragma unroll
					for(int i = 0; i < BN / 64; ++i) tma_load_3d(b + i * 8192, &mapB, full, t.n0 + i * 64, k, planeB);
				} else {
					tma_load_3d(b, &mapB, full, k, t.n0, planeB);
				}
				++it;
				return true;
			};
			for(int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
				const Tile t = tile_of<BN>(p, tile);
				const int chunk = CHUNKED ? CHUNKS : p.kBlocks;
				for(int k0 = t.kBegin; ok && k0 < t.kEnd; k0 += chunk) {
					const int k1 = min(t.kEnd, k0 + chunk);
					for(int term = 0; ok && term < TERMS; ++term) {
						for(int kb = k0; ok && kb < k1; ++kb) ok = load(t, kb, FP32 ? PLANE_A[term] : 0, FP32 ? PLANE_B[term] : 0);
					}
				}
			}
			if(!ok) { // let what is in flight land before the shared memory goes
				int ignored = 0;
				for(int i = it > STAGES ? it - STAGES : 0; i < it; ++i) {
					mbar_wait_bounded(bars + B_FULL + i % STAGES, (i / STAGES) & 1, &ignored, nullptr, 0);
				}
			}
		}
		__syncwarp();
	} else if(warp == 1) {
		if(elect_one()) {
			const uint32_t format = p.bf16 ? (1u << 7) | (1u << 10) : 0u;
			const uint32_t idesc = umma_idesc_f16(BM, BN) | format | (A_ACROSS ? 1u << 15 : 0u) | (B_ACROSS ? 1u << 16 : 0u);
			int it = 0, n = 0;
			bool ok = true;
			for(int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
				const Tile t = tile_of<BN>(p, tile);
				const int chunk = CHUNKED ? CHUNKS : p.kBlocks;
				int k0 = t.kBegin;
				do { // a part of K without steps takes its turn too
					const int acc = n & 1;
					if(n >= 2 && !mbar_wait_bounded(bars + B_ACCEMPTY + acc, (n / 2 - 1) & 1, abortFlag, p.status, (KERNEL_ID << 8) | SITE_MMA_ACC)) {
						ok = false;
						break;
					}
					tc_fence_after_sync();
					const uint32_t d = tmemBase + acc * BN;
					const int steps = (min(t.kEnd, k0 + chunk) - k0) * TERMS;
					for(int i = 0; i < steps; ++i, ++it) {
						const int s = it % STAGES;
						if(!mbar_wait_bounded(bars + B_FULL + s, (it / STAGES) & 1, abortFlag, p.status, (KERNEL_ID << 8) | SITE_MMA)) {
							ok = false;
							break;
						}
						tc_fence_after_sync();
						const uint32_t a = smemBase + s * STAGE_BYTES, b = a + A_BYTES;
#pragma unroll
						for(int k = 0; k < BK / 16; ++k) {
							const uint64_t da = A_ACROSS ? desc_across(a + k * 2048) : umma_desc_k128(a + k * 32);
							const uint64_t db = B_ACROSS ? desc_across(b + k * 2048) : umma_desc_k128(b + k * 32);
							umma_f16_ss(d, da, db, idesc, i > 0 || k > 0 ? 1u : 0u);
						}
						umma_commit(bars + B_EMPTY + s);
					}
					if(ok) umma_commit(bars + B_ACCFULL + acc);
					++n;
					k0 += chunk;
				} while(ok && k0 < t.kEnd);
			}
			if(*abortFlag != 0) { // nothing may still write tensor memory when it is freed
				int ignored = 0;
				umma_commit(bars + B_DONE);
				mbar_wait_bounded(bars + B_DONE, 0, &ignored, nullptr, 0);
			}
		}
		__syncwarp();
	} else if(warp >= 4) {
		const int quarter = warp & 3, half = (warp - 4) >> 2;
		int n = 0;
		bool ok = true;
		for(int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
			const Tile t = tile_of<BN>(p, tile);
			const int row = t.m0 + quarter * 32 + lane;
			const bool on = row < p.m;
			const int col0 = t.n0 + half * COLUMNS;
			const uint32_t tmemRow = tmemBase + (static_cast<uint32_t>(quarter * 32) << 16) + half * COLUMNS;
			int label = -1;
			float logSum2 = 0.f, by = 0.f;
			if(on && (EPILOGUE == PRODUCT16_STATS || EPILOGUE == PRODUCT16_DIFF)) {
				label = __ldg(p.labels + row);
				if(label < 0 || label >= p.columns) label = -1;
			}
			if(on && EPILOGUE == PRODUCT16_DIFF) {
				logSum2 = __ldg(p.logSum + row) * LOG2E;
				by = __fdiv_rn(__ldg(p.rowScale + row), __ldg(p.scale)) * __ldg(p.scale + 1);
				if(label < 0) by = 0.f;
			}
			if(EPILOGUE == PRODUCT16_STORE) by = __ldg(p.resultScale);
			const int own = label - p.firstColumn - col0; // the label's place in this thread's columns, if it is there
			float top = -INFINITY, sum = 0.f;
			// what becomes of 32 columns of the thread's row, from col0 + c
			auto finish = [&](int c, float (&r)[32]) __attribute__((always_inline)) {
				if constexpr(EPILOGUE == PRODUCT16_STATS) {
					const int left = p.columns - p.firstColumn - col0 - c; // valid ones of these 32
					if(left < 32) {
#pragma unroll
						for(int i = 0; i < 32; ++i) {
							if(i >= left) r[i] = -INFINITY;
						}
					}
					const uint32_t hot = own >= c && own < c + 32 ? 1u << (own - c) : 0u;
					if(__any_sync(0xffffffffu, hot != 0u)) {
						uint32_t value = 0u; // (written so that the row stays in registers)
#pragma unroll
						for(int i = 0; i < 32; ++i) value |= (hot >> i & 1u) != 0u ? __float_as_uint(r[i]) : 0u;
						if(hot != 0u && left > own - c) p.labelled[row] = __uint_as_float(value);
					}
					float most = r[0];
#pragma unroll
					for(int i = 1; i < 32; ++i) most = fmaxf(most, r[i]);
					const float newTop = fmaxf(top, most * LOG2E);
					const float reference = newTop == -INFINITY ? 0.f : newTop;
					float2 part[2] = { both(0.f), both(0.f) };
#pragma unroll
					for(int i = 0; i < 32; i += 2) {
						const float2 e = fma2(make_float2(r[i], r[i + 1]), both(LOG2E), both(-reference));
						part[(i >> 1) & 1] = add2(part[(i >> 1) & 1], make_float2(exp2_fast(e.x), exp2_fast(e.y)));
					}
					const float2 parts = add2(part[0], part[1]);
					sum = sum * exp2_fast(top - reference) + (parts.x + parts.y);
					top = newTop;
				} else if constexpr(EPILOGUE == PRODUCT16_DIFF) {
					const int left = p.columns - p.firstColumn - col0 - c;
#pragma unroll
					for(int i = 0; i < 32; i += 2) {
						const float2 e = fma2(make_float2(r[i], r[i + 1]), both(LOG2E), both(-logSum2));
						const float2 v = mul2(make_float2(exp2_fast(e.x), exp2_fast(e.y)), both(by));
						r[i] = v.x;
						r[i + 1] = v.y;
					}
					const uint32_t hot = own >= c && own < c + 32 ? 1u << (own - c) : 0u;
					if(__any_sync(0xffffffffu, hot != 0u)) {
#pragma unroll
						for(int i = 0; i < 32; ++i) r[i] -= (hot >> i & 1u) != 0u ? by : 0.f;
					}
					// a row without a target has no gradient, whatever its logits; columns behind the vocabulary are zeros,
					// which the products that read them count on
					if(by == 0.f || left < 32) {
#pragma unroll
						for(int i = 0; i < 32; ++i) {
							if(by == 0.f || i >= left) r[i] = 0.f;
						}
					}
					if(on) {
						uint16_t* const out = static_cast<uint16_t*>(p.out) + row * p.ldOut + col0 + c;
#pragma unroll
						for(int plane = 0; plane < (FP32 ? 3 : 1); ++plane) {
#pragma unroll
							for(int j = 0; j < 2; ++j) {
								uint32_t w[8];
#pragma unroll
								for(int i = 0; i < 8; ++i) {
									float &v0 = r[j * 16 + 2 * i], &v1 = r[j * 16 + 2 * i + 1];
									w[i] = FP32 ? pack2<__nv_bfloat16>(v0, v1) : pack16(v0, v1, p.bf16);
									if(FP32) { // the rest, for the next plane
										const float2 taken = unpack2<__nv_bfloat16>(w[i]);
										v0 -= taken.x;
										v1 -= taken.y;
									}
								}
								store32(out + plane * p.outPlane + j * 16, w);
							}
						}
					}
				} else if constexpr(EPILOGUE == PRODUCT16_SUM) {
					if(on) {
						float* const out = p.plane + (static_cast<long long>(t.split) * p.m + row) * p.ldPlane + col0 + c;
#pragma unroll
						for(int j = 0; j < 4; ++j) {
							if(col0 + c + j * 8 < p.n) { // ldPlane is a multiple of 8
								uint32_t w[8];
								if(p.accumulate) {
									load32(out + j * 8, w);
#pragma unroll
									for(int i = 0; i < 8; ++i) w[i] = __float_as_uint(r[j * 8 + i] + __uint_as_float(w[i]));
								} else {
#pragma unroll
									for(int i = 0; i < 8; ++i) w[i] = __float_as_uint(r[j * 8 + i]);
								}
								store32(out + j * 8, w);
							}
						}
					}
				} else if constexpr(FP32) {
					if(on) {
						float* const out = static_cast<float*>(p.out) + row * p.ldOut + col0 + c;
						const bool aligned = (p.ldOut & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0;
#pragma unroll
						for(int j = 0; j < 8; ++j) {
							const int left = p.n - (col0 + c + j * 4);
							if(aligned && left >= 4) {
								*reinterpret_cast<float4*>(out + j * 4) = make_float4(r[j * 4] * by, r[j * 4 + 1] * by, r[j * 4 + 2] * by, r[j * 4 + 3] * by);
							} else {
#pragma unroll
								for(int i = 0; i < 4; ++i) {
									if(i < left) out[j * 4 + i] = r[j * 4 + i] * by;
								}
							}
						}
					}
				} else {
					if(on) {
						uint16_t* const out = static_cast<uint16_t*>(p.out) + row * p.ldOut + col0 + c;
						// whole sectors where rows allow it: a thread's row is 32 bytes at a time
						const bool sectors = (p.ldOut & 15) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0;
						const bool aligned = (p.ldOut & 7) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0;
#pragma unroll
						for(int j = 0; j < 2; ++j) {
							uint32_t w[8];
#pragma unroll
							for(int i = 0; i < 8; ++i) w[i] = pack16(r[j * 16 + 2 * i] * by, r[j * 16 + 2 * i + 1] * by, p.bf16);
							const int left = p.n - (col0 + c + j * 16);
							if(sectors && left >= 16) {
								store32(out + j * 16, w);
							} else {
#pragma unroll
								for(int h = 0; h < 2; ++h) {
									if(aligned && left >= 8 * h + 8) {
										*reinterpret_cast<uint4*>(out + j * 16 + h * 8) = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
									} else {
#pragma unroll
										for(int i = 8 * h; i < 8 * h + 8; ++i) {
											if(i < left) out[j * 16 + i] = static_cast<uint16_t>(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu);
										}
									}
								}
							}
						}
					}
				}
			};
			const bool empty = t.kBegin >= t.kEnd; // a part of K without steps: nothing was multiplied
			if constexpr(CHUNKED) {
				float total[COLUMNS / 32][32];
				int k0 = t.kBegin;
				do {
					const int acc = n & 1;
					ok = mbar_wait_bounded_warp(bars + B_ACCFULL + acc, (n >> 1) & 1, abortFlag, p.status, (KERNEL_ID << 8) | SITE_EPILOGUE);
					if(!ok) break;
					tc_fence_after_sync();
#pragma unroll
					for(int c = 0; c < COLUMNS / 32; ++c) {
						uint32_t r[32];
						tmem_ld32_issue(tmemRow + acc * BN + c * 32, r);
						tmem_ld_wait();
#pragma unroll
						for(int i = 0; i < 32; ++i) total[c][i] = (k0 == t.kBegin ? 0.f : total[c][i]) + (empty ? 0.f : __uint_as_float(r[i]));
					}
					tc_fence_before_sync();
					if(lane == 0) mbar_arrive(bars + B_ACCEMPTY + acc);
					++n;
					k0 += CHUNKS;
				} while(k0 < t.kEnd);
				if(!ok) break;
#pragma unroll
				for(int c = 0; c < COLUMNS / 32; ++c) finish(c * 32, total[c]);
			} else {
				const int acc = n & 1;
				ok = mbar_wait_bounded_warp(bars + B_ACCFULL + acc, (n >> 1) & 1, abortFlag, p.status, (KERNEL_ID << 8) | SITE_EPILOGUE);
				if(!ok) break;
				++n;
				tc_fence_after_sync();
#pragma unroll 1
				for(int c = 0; c < COLUMNS; c += 32) {
					uint32_t r[32];
					tmem_ld32_issue(tmemRow + acc * BN + c, r);
					tmem_ld_wait();
					if(c == COLUMNS - 32) { // the accumulator is free
						tc_fence_before_sync();
						if(lane == 0) mbar_arrive(bars + B_ACCEMPTY + acc);
					}
					float v[32];
#pragma unroll
					for(int i = 0; i < 32; ++i) v[i] = EPILOGUE == PRODUCT16_SUM && empty ? 0.f : __uint_as_float(r[i]);
					finish(c, v);
				}
			}
			if(EPILOGUE == PRODUCT16_STATS && on) {
				p.partial[static_cast<long long>(t.nTile * 2 + half) * p.m + row] = make_float2(top, sum);
			}
		}
	}
	tc_fence_before_sync();
	__syncthreads();
	if(warp == 2) tmem_dealloc(tmemBase, 512);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
	const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder()
{
	static EncodeTiledFn found = nullptr;
	static std::once_flag once;
	std::call_once(once, [] {
		void* fn = nullptr;
		cudaDriverEntryPointQueryResult q;
		if(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) {
			found = reinterpret_cast<EncodeTiledFn>(fn);
		}
		cudaGetLastError();
	});
	return found;
}

using Kernel = void (*)(const Product16Params, const CUtensorMap, const CUtensorMap);

template<int EPILOGUE, bool A_ACROSS, bool B_ACROSS, bool NARROW>
Kernel kernel_for(const Product16Params& p)
{
	if(p.fp32) return product16_kernel<EPILOGUE, A_ACROSS, B_ACROSS, true, NARROW, true>;
	if constexpr(EPILOGUE != PRODUCT16_DIFF) { // (whose exponentials are rounded to the operands' type)
		if(p.kBlocksPerSplit > CHUNK<EPILOGUE, false>) return product16_kernel<EPILOGUE, A_ACROSS, B_ACROSS, false, NARROW, true>;
	}
	return product16_kernel<EPILOGUE, A_ACROSS, B_ACROSS, false, NARROW, false>;
}
template<int EPILOGUE>
Kernel rows_kernel(const Product16Params& p)
{
	return p.narrow ? kernel_for<EPILOGUE, false, false, true>(p) : kernel_for<EPILOGUE, false, false, false>(p);
}

} // namespace

bool product16_map(void* map, const void* base, bool bf16, long long inner, long long rows, long long rowSize, int boxRows, long long planeSize)
{
	const EncodeTiledFn encode = encoder();
	if(encode == nullptr || !aligned16(base) || rowSize % 8 != 0 || planeSize % 8 != 0 || rowSize * 2 >= (1ll << 40) || planeSize * 2 >= (1ll << 40)) return false;
	const cuuint64_t dims[3] = { static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows), planeSize > 0 ? 3u : 1u };
	const cuuint64_t strides[2] = { static_cast<cuuint64_t>(rowSize) * 2, static_cast<cuuint64_t>(planeSize > 0 ? planeSize : rowSize) * 2 };
	const cuuint32_t box[3] = { 64, static_cast<cuuint32_t>(boxRows), 1 };
	const cuuint32_t steps[3] = { 1, 1, 1 };
	return encode(static_cast<CUtensorMap*>(map), bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
		const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
		CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool sequence_map(void* map, const void* base, int type, long long channels, long long length, long long batch, long long row,
	long long batchStride, int steps)
{
	const EncodeTiledFn encode = encoder();
	const long long size = type_size(type);
	if(encode == nullptr || !aligned16(base) || row <= 0 || batchStride <= 0 || row * size % 16 != 0 || batchStride * size % 16 != 0
		|| row * size >= (1ll << 40) || batchStride * size >= (1ll << 40)) return false;
	const cuuint64_t dims[3] = { static_cast<cuuint64_t>(channels), static_cast<cuuint64_t>(length), static_cast<cuuint64_t>(batch) };
	const cuuint64_t strides[2] = { static_cast<cuuint64_t>(row * size), static_cast<cuuint64_t>(batchStride * size) };
	const cuuint32_t box[3] = { static_cast<cuuint32_t>(128 / size), static_cast<cuuint32_t>(steps), 1 };
	const cuuint32_t each[3] = { 1, 1, 1 };
	return encode(static_cast<CUtensorMap*>(map), type == NB200_TYPE_FP32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == NB200_TYPE_FP16
		? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, each,
		CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int product16(Product16Epilogue epilogue, bool aAcross, bool bAcross, const Product16Params& p, const void* mapA, const void* mapB,
	cudaStream_t stream)
{
	Kernel kernel = nullptr;
	if(epilogue == PRODUCT16_STATS && !aAcross && !bAcross) kernel = rows_kernel<PRODUCT16_STATS>(p);
	else if(epilogue == PRODUCT16_DIFF && !aAcross && !bAcross) kernel = rows_kernel<PRODUCT16_DIFF>(p);
	else if(epilogue == PRODUCT16_SUM && !aAcross && bAcross && !p.narrow) kernel = kernel_for<PRODUCT16_SUM, false, true, false>(p);
	else if(epilogue == PRODUCT16_SUM && aAcross && bAcross && !p.narrow) kernel = kernel_for<PRODUCT16_SUM, true, true, false>(p);
	else if(epilogue == PRODUCT16_STORE && aAcross && bAcross && !p.narrow) kernel = kernel_for<PRODUCT16_STORE, true, true, false>(p);
	else return NB200_EINVAL;
	const long long tiles = static_cast<long long>(p.mTiles) * p.nTiles * p.splits;
	if(tiles > 0x7fffffffLL - 1024) return NB200_ETOOBIG;
	if(tiles == 0) return NB200_OK;
	if(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) return check_launch();
	const int grid = tiles < sm_count() ? static_cast<int>(tiles) : sm_count();
	launch_dependent(true, kernel, dim3(grid), dim3(THREADS), SMEM_BYTES, stream, p, *static_cast<const CUtensorMap*>(mapA),
		*static_cast<const CUtensorMap*>(mapB));
	count_launch();
	return check_launch();
}

} // namespace nb200
