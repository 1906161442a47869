// Products of 16-bit matrices on the tensor core (fp16 or bf16 in, fp32 accumulators), with the epilogues of the cross entropy over a
// vocabulary (vocabulary_loss.cu).  D[m][n] = sum_k A[m][k] B[n][k]; either operand may lie with its k adjacent (rows of k) or with
// its m or n adjacent (rows per k, as a gradient's product meets what the forward pass stored).
//
// fp32 operands come as three bf16 matrices each ("planes"), x = hi + mid + lo with eight bits of x in each: all 24.  Of the nine
// products of planes six are formed (hi hi, hi mid, mid hi, mid mid, hi lo, lo hi); what is left out is below 2^-26 of the product of
// the largest.  bf16 rather than fp16 parts, since softmax gradients reach from 1 to far below what a half holds.
#pragma once
#include "types16.cuh"

namespace nb200 {

enum Product16Epilogue {
	PRODUCT16_STATS, // per row and half a tile of columns: maximum and sum of exponentials, and the labelled column's value
	PRODUCT16_DIFF,  // gradient by the logits, 16-bit or three planes: coefficient[row] * (softmax - [column is the label])
	PRODUCT16_SUM,   // fp32 planes, one per part of K; added to what is there where `accumulate` is set
	PRODUCT16_STORE  // result times *resultScale, of the operands' type
};

struct Product16Params {
	int m, n;            // rows and columns of the result
	int mTiles, nTiles, splits;
	int kBlocks, kBlocksPerSplit;
	int narrow;          // tiles of PRODUCT16_NARROW columns, B's box likewise: STATS and DIFF
	int boxA;            // rows of A's box where A lies in rows: product16_box_a(m)
	int mFast;           // consecutive tiles go down the rows (A stays near) rather than along the columns
	int bf16;            // operands are bf16 rather than fp16
	int fp32;            // operands are three bf16 planes
	int* status;
	// STATS
	float2* partial;     // [2 * nTiles][m]: maximum in units of log 2, sum of 2^(x - maximum)
	float* labelled;     // [m]
	// STATS, DIFF
	const int* labels;   // [m]
	int firstColumn;     // the column that column 0 of this result stands for
	int columns;         // of all: columns behind are left out
	// DIFF
	const float* logSum; // [m]
	const float* rowScale; // [m], over scale[0] and times scale[1]
	const float* scale;
	// DIFF, STORE
	void* out;           // STORE: 16-bit or fp32
	long long ldOut;
	long long outPlane;  // DIFF with planes: elements between them
	// STORE
	const float* resultScale;
	// SUM
	float* plane;        // [splits][m][ldPlane]
	long long ldPlane;   // a multiple of 8
	int accumulate;
};

// Enqueues the product.  mapA and mapB are the operands' tensor maps (product16_map).
int product16(Product16Epilogue epilogue, bool aAcross, bool bAcross, const Product16Params& p, const void* mapA, const void* mapB,
	cudaStream_t stream);
// Map of a matrix of 16-bit elements, `inner` adjacent ones in each of `rows` rows; boxes of 64 x boxRows land as 128-byte rows
// with the 128-byte swizzle.  planeSize > 0: three such matrices that many elements apart.  False where TMA cannot describe it (base
// or rows off a 16-byte boundary).
bool product16_map(void* map, const void* base, bool bf16, long long inner, long long rows, long long rowSize, int boxRows,
	long long planeSize = 0);

// Map of [batch][length][channels] in the operator types: boxes of `steps` steps x 128 bytes of channels, dense.  False as above, and where
// a stride is zero.
bool sequence_map(void* map, const void* base, int type, long long channels, long long length, long long batch, long long row,
	long long batchStride, int steps);

constexpr int PRODUCT16_M = 128, PRODUCT16_N = 256, PRODUCT16_NARROW = 64, PRODUCT16_K = 64; // of a tile
// boxRows of the operands' maps: across, and in rows; of B in rows the tile's columns
constexpr int PRODUCT16_BOX_ACROSS = 64;
inline int product16_box_a(int m) { return m >= PRODUCT16_M ? PRODUCT16_M : (m + 7) / 8 * 8; } // no more rows than there are

} // namespace nb200
