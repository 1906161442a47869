// The cross entropy over a vocabulary for a few rows of fp32 (vocabulary_few.cu), behind the entry points of vocabulary_loss.cu.
#pragma once
#include "types16.cuh"

namespace nb200 {

constexpr int FEW_ROWS = 8;             // at most
constexpr int FEW_FORWARD_ROWS = 32;    // and of the forward pass
constexpr int FEW_TILE = 64;            // vocabulary entries of a tile
constexpr int FEW_MOST_ENTRIES = 1024;  // of a block

struct FewParams {
	const float *hidden, *weights;
	long long hiddenRow, weightsRow;
	int rows, width, vocabulary;
	int perBlock;           // entries of a block: few_entries()
	const int* labels;
	float2* partial;        // forward: [few_blocks()][rows], maximum in units of log 2 and sum
	float* labelled;        // forward: [rows]
	const float *logSum, *lossDiff; // backward
	float* weightsDiff;     // backward; null: not wanted
	long long weightsDiffRow;
	float* hiddenPart;      // backward: [few_blocks()][rows][width]; null: hidden_diff is not wanted
};

int few_entries(int rows, int vocabulary);
int few_blocks(int rows, int vocabulary);
int few_forward(const FewParams& p, cudaStream_t stream);
int few_backward(const FewParams& p, float* hiddenDiff, long long hiddenDiffRow, cudaStream_t stream);

} // namespace nb200
