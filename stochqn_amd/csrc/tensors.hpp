// tensors.hpp -- first-order steps over the tensors of a model: what the host side (tensors.cpp) hands to the kernels (tensors.hip).
// Everything here takes DEVICE pointers and enqueues work on a stream; nothing synchronises, allocates or copies, so that a call
// can be captured into a graph.
#pragma once
#include <hip/hip_runtime.h>
#include <cstddef>
#include <cstdint>

namespace sqn {

constexpr int kStateBlock = 128;     // elements that share the scale of an 8-bit moment; every tensor's state starts at a multiple of it
// Elements a workgroup of 256 threads takes at a time, their loads issued together.  Measured: the step with 32-bit moments at 1e8 f32
// elements 482 us with tiles of 2048, 473 with 4096, 535 with 8192, at 1.28e9 bf16 + f32 elements 6.99, 6.50 and 7.72 ms; with 8-bit moments at 1.28e9 bf16
// elements 2.58 ms with 4096, 2.40 with 8192 (16384 spill: 14.9); the norm of those 396, 392, 395 us and 379 with 16384, of 7.7e6 elements 12.6, 9.6, 9.3
// and 10.3 us.
constexpr int kTileSmall = 2048;     // short lists: both sides measured at the rule (tensors.cpp: shape_of)
constexpr int kTile32 = 4096;        // moments in 32 bits
constexpr int kTile8 = 8192;         // in 8 bits
constexpr int kTileNormMid = 8192;   // the norm
constexpr int kTileNorm = 16384;
constexpr int kEntries = 112;        // tensors per launch: the table travels in the kernel's arguments (32 B each, 4 KB in all)
constexpr int kFewEntries = 12;      // ... of a short list: 3.6 KB less for the host to hand over, 0.1 - 0.3 us of a call (12 tensors: 5.7 against 5.8 us, their norm 8.6
                                     // against 8.8); the GPU's time is the same (5.16 and 5.15 us a step), with 40 entries too

enum TensorType { T_F32 = 0, T_BF16 = 1, T_F16 = 2 };
inline size_t type_size(int t) { return t == T_F32 ? 4 : 2; }

// One tensor as a kernel sees it.  `info`: elements (56 bits), the parameter's type (2 bits), the gradient's (2), "no weight decay" (1).
struct TensorEntry {
	void* param;
	const void* grad;
	uint64_t info;
	uint32_t tile0;              // first tile of this launch that is the tensor's (tiles of LaunchShape::tile elements)
	uint32_t block0;             // first block of kStateBlock elements of its state, counted from AdamwArgs::block_base
};
constexpr uint64_t kCountMask = (1ull << 56) - 1;
inline uint64_t entry_info(size_t count, int ptype, int gtype, bool no_decay)
{
	return (uint64_t) count | (uint64_t) ptype << 56 | (uint64_t) gtype << 58 | (uint64_t) no_decay << 60;
}

// How a list is cut up: one rule for every call on it, by its sizes alone.
struct LaunchShape {
	int tile;                    // elements of a tile
	int grid;                    // most workgroups
};

// Workgroups arrive at one of these counters, the last of each at count[1]: arrivals at one address take 6.5 ns each, one after the other.
constexpr int kGates = 16, kGateStride = 256;            // bytes

struct AdamwArgs {
	int entries;                 // of the table that are in use
	uint32_t tiles;
	uint64_t block_base;
	float* master;               // f32 weights of the 16-bit tensors, or NULL
	void *m, *v;                 // f32[state] or codes [state]
	uint8_t *m_scale, *v_scale;  // [state / kStateBlock], 8-bit moments only
	long long* count;            // [0] steps taken, [1] arrivals (zero between steps)
	char* gates;                 // kGates counters (zero between steps)
	const float* grad_scale;     // what every gradient is multiplied with; NULL = 1
	const float* step_size_dev;  // NULL: step_size
	double step_size, beta1, beta2, weight_decay;
	float eps;
	uint64_t seed;
	int last;                    // the launch that counts the step
	int stochastic;              // bf16 parameters without f32 weights beside them are rounded stochastically
};

struct NormArgs {
	int entries;
	uint32_t tiles;
	double* part;                // one partial sum of squares per workgroup of this launch
	double grad_scale, max_norm;
	float* out;                  // not NULL: this workgroup, the only one, finishes
};

template <class Args, int N> struct Table {
	Args a;
	TensorEntry entry[N];
};
static_assert(sizeof(Table<AdamwArgs, kEntries>) <= 4096, "kernel arguments");

void launch_adamw(hipStream_t st, int bits, int tile, int grid, const Table<AdamwArgs, kEntries>& t);
void launch_norm(hipStream_t st, int tile, int grid, const Table<NormArgs, kEntries>& t);      // TensorEntry::param unused
// part[0] <- the sum of part[1 .. count] (in a fixed order); with `out` also the verdict
void launch_norm_sum(hipStream_t st, double* part, int count, double grad_scale, double max_norm, float* out);
// the verdict of a sum of squares that is final: out[0] the norm, out[1] the coefficient
void launch_norm_verdict(hipStream_t st, const double* sum, double grad_scale, double max_norm, float* out);

}  // namespace sqn
