// tensors.hip -- the AdamW step over many tensors at once and the norm over all their gradients.
//
// For every element, with the step's number t counted from 1 and all arithmetic in f32:
//   g <- grad_scale * g;   m <- b1 m + (1 - b1) g;   v <- b2 v + (1 - b2) g^2
//   w <- w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Every array is read once and written once; nothing is reused, so HBM bounds the step: 28 B per element with f32 weights and
// moments, 10 B with bf16 weights and 8-bit moments.  m and v are formed by separate products and sums (no fma), so that they -- and
// with them the 8-bit codes -- do not depend on what a compiler contracts.
#include "tensors.hpp"

namespace sqn {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));        // parameters and gradients: aligned to their elements only
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kLane = 8;                                                     // elements per lane and tile
static_assert(kTile == kThreads * kLane, "a tile is eight elements per lane");

__device__ inline float bits_float(uint32_t b) { return __builtin_bit_cast(float, b); }
__device__ inline uint32_t float_bits(float f) { return __builtin_bit_cast(uint32_t, f); }

__device__ inline float widen16(uint32_t h, int type)
{
	return type == T_BF16 ? bits_float(h << 16) : (float) __builtin_bit_cast(_Float16, (uint16_t) h);
}
__device__ inline uint32_t narrow16(float f, int type)
{
	return type == T_BF16 ? (uint32_t) __builtin_bit_cast(uint16_t, (__bf16) f) : (uint32_t) __builtin_bit_cast(uint16_t, (_Float16) f);
}

// elements i .. i+7 of a tensor of n; what lies behind its end reads as zero
__device__ inline void load8(const void* base, uint64_t i, uint64_t n, int type, float (&x)[kLane])
{
	if (i + kLane <= n) {
		if (type == T_F32) {
			const f32x4u* p = reinterpret_cast<const f32x4u*>(static_cast<const float*>(base) + i);
			const f32x4u a = p[0], b = p[1];
#pragma unroll
			for (int j = 0; j < 4; j++) { x[j] = a[j]; x[4 + j] = b[j]; }
		} else {
			const u32x4u a = *reinterpret_cast<const u32x4u*>(static_cast<const uint16_t*>(base) + i);
#pragma unroll
			for (int j = 0; j < 4; j++) { x[2 * j] = widen16(a[j] & 0xffff, type); x[2 * j + 1] = widen16(a[j] >> 16, type); }
		}
	} else {
#pragma unroll
		for (int j = 0; j < kLane; j++) {
			x[j] = 0;
			if (i + j < n) x[j] = type == T_F32 ? static_cast<const float*>(base)[i + j] : widen16(static_cast<const uint16_t*>(base)[i + j], type);
		}
	}
}

__device__ inline void store8(float* base, uint64_t i, uint64_t n, const float (&x)[kLane])
{
	if (i + kLane <= n) {
		f32x4u* p = reinterpret_cast<f32x4u*>(base + i);
		p[0] = f32x4u{x[0], x[1], x[2], x[3]};
		p[1] = f32x4u{x[4], x[5], x[6], x[7]};
	} else {
#pragma unroll
		for (int j = 0; j < kLane; j++)
			if (i + j < n) base[i + j] = x[j];
	}
}

__device__ inline void store8(uint16_t* base, uint64_t i, uint64_t n, const uint32_t (&h)[kLane])
{
	if (i + kLane <= n) {
		*reinterpret_cast<u32x4u*>(base + i) = u32x4u{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
	} else {
#pragma unroll
		for (int j = 0; j < kLane; j++)
			if (i + j < n) base[i + j] = (uint16_t) h[j];
	}
}

// the entry of the launch's table that tile `tile` belongs to (uniform over the workgroup)
template <class Args> __device__ inline int entry_of(const Args& a, uint32_t tile)
{
	int lo = 0, hi = a.entries;
	while (hi - lo > 1) {
		const int mid = (lo + hi) >> 1;
		if (a.entry[mid].tile0 <= tile) lo = mid; else hi = mid;
	}
	return lo;
}

// ---- stochastic rounding ---------------------------------------------------------------------------------------------------------
// The moments are running averages: at b2 = 0.999 a step moves v by about a thousandth, while half a step of e5m2 is an eighth -- with
// rounding to nearest v would never move again.  Rounded up with the probability of the rest, the mean stays exact.  The words come
// from a counter-based generator (the finaliser of the library's synthetic inputs): group q of eight elements, step t.  Element j
// of the group takes the low half (m) and the high half (v) advanced by j golden steps: each uniform by itself, evenly spread over
// the eight, independent between groups and steps.
constexpr uint64_t kGolden = 0x9E3779B97F4A7C15ull, kStepKey = 0xD1B54A32D192ED03ull;
constexpr uint32_t kLaneStep = 0x9E3779B9u;

__device__ inline uint64_t finalise(uint64_t z)
{
	z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
	z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
	return z ^ (z >> 31);
}

// ---- what is the same for every element of a step ---------------------------------------------------------------------------------
struct Step {
	float scale, b1, b2, a1, a2, decay, rate, root, eps;
	uint64_t key;
	bool stochastic;
};

__device__ inline Step step_of(const AdamwArgs& a, long long t)
{
	double p1 = 1, p2 = 1, q1 = a.beta1, q2 = a.beta2;       // b^t by squaring, in f64: 1 - b2^t loses ten bits at t = 1
	for (unsigned long long k = (unsigned long long) t; k; k >>= 1) {
		if (k & 1) { p1 *= q1; p2 *= q2; }
		q1 *= q1;
		q2 *= q2;
	}
	const double lr = a.step_size_dev ? (double) *a.step_size_dev : a.step_size;
	Step s;
	s.b1 = (float) a.beta1;
	s.b2 = (float) a.beta2;
	s.a1 = (float) (1 - a.beta1);
	s.a2 = (float) (1 - a.beta2);
	s.decay = (float) (1 - lr * a.weight_decay);
	s.rate = (float) (lr / (1 - p1));
	s.root = (float) (1 / sqrt(1 - p2));
	s.eps = a.eps;
	s.key = finalise(a.seed ^ (uint64_t) t * kStepKey);
	s.stochastic = a.stochastic != 0;
	return s;
}

// moments and weight of one element
__device__ inline void update(const Step& s, float decay, float g, float& m, float& v, float& w)
{
	m = m * s.b1 + g * s.a1;
	v = v * s.b2 + (g * g) * s.a2;
	w = fmaf(-s.rate, m / fmaf(sqrtf(v), s.root, s.eps), w * decay);
}

// the new weights go out: f32 as they are, 16 bits rounded (to nearest, or stochastically by the low half of the first word: bf16 is
// the upper half of f32, so the word's 16 bits are added to the lower half and cut off with it)
__device__ inline void put_weights(const AdamwArgs& a, const Step& s, void* param, uint64_t i, uint64_t n, int ptype, float* master, float (&w)[kLane], uint32_t word)
{
	if (ptype == T_F32) { store8(static_cast<float*>(param), i, n, w); return; }
	uint32_t h[kLane];
	if (master) store8(master, i, n, w);
	if (!master && s.stochastic) {
#pragma unroll
		for (int j = 0; j < kLane; j++) {
			const uint32_t b = float_bits(w[j]);
			h[j] = ((b & 0x7f800000u) == 0x7f800000u ? (b | (b << 16 ? 0x400000u : 0)) : b + ((word + j * kLaneStep) & 0xffff)) >> 16;
		}
	} else {
#pragma unroll
		for (int j = 0; j < kLane; j++) h[j] = narrow16(w[j], ptype);
	}
	store8(static_cast<uint16_t*>(param), i, n, h);
}

// ---- moments in 8 bits -------------------------------------------------------------------------------------------------------------
// A block of 128 elements shares a scale 2^k (a byte, the exponent's 8 bits): the largest |m| lies at 2^7 .. 2^8 of it, the largest v at
// 2^14 .. 2^15, so that rounding up stays inside e4m3 (448) and e5m2 (57344).  A power of two costs no precision in a floating
// format and makes every product with it exact.  16 lanes hold a block, eight elements each.
__device__ inline float scale_float(uint32_t byte)          // 255: the block is not finite, every value of it reads as NaN
{
	return bits_float(byte << 23 | (byte == 255 ? 0x400000u : 0));
}

__device__ inline uint32_t block_max(uint32_t x)             // over the 16 lanes of a block
{
#pragma unroll
	for (int d = 1; d < 16; d <<= 1) x = max(x, (uint32_t) __shfl_xor((int) x, d, 16));
	return x;
}

// byte of the scale for a block whose largest magnitude has the bits `top`; `at`: the power of two of the scale that it is brought to
__device__ inline uint32_t scale_byte(uint32_t top, int at)
{
	const int e = (int) (top >> 23) - at;
	return top >= 0x7f800000u ? 255u : (uint32_t) (e > 1 ? e : 1);
}

template <bool SECOND> __device__ inline u32x2 encode8(const float (&x)[kLane], uint32_t byte, uint32_t word)
{
	const float inv = byte == 255 ? 0.0f : bits_float((254u - byte) << 23);
	u32x2 out = {0, 0};
#pragma unroll
	for (int j = 0; j < kLane; j++) {
		float y = x[j] * inv;
		const int r = (int) (word + j * kLaneStep);
		// a second moment above zero stays above zero (the least code, 2^-16): m / (sqrt(0) + eps) would be a jump
		if (SECOND) y = x[j] > 0 ? fmaxf(y, 0x1p-16f) : y;
		const int c = SECOND ? __builtin_amdgcn_cvt_sr_bf8_f32(y, r, 0, 0) : __builtin_amdgcn_cvt_sr_fp8_f32(y, r, 0, 0);
		out[j >> 2] |= (uint32_t) (c & 0xff) << (8 * (j & 3));
	}
	return out;
}

template <bool SECOND> __device__ inline void decode8(u32x2 c, float scale, float (&x)[kLane])
{
#pragma unroll
	for (int j = 0; j < kLane; j += 2) {
		const int w = (int) (c[j >> 2] >> (8 * (j & 2)));
		const auto p = SECOND ? __builtin_amdgcn_cvt_pk_f32_bf8(w, false) : __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
		x[j] = p[0] * scale;
		x[j + 1] = p[1] * scale;
	}
}

template <int BITS> __global__ __launch_bounds__(kThreads) void k_adamw(const AdamwArgs a)
{
	// a scale that is not finite: the step is rejected as a whole, nothing changes and nothing is counted
	const float scale = a.grad_scale ? *a.grad_scale : 1.0f;
	if (!(fabsf(scale) <= 3.402823466e38f)) return;
	const long long t = a.count[0] + 1;
	Step s = step_of(a, t);
	s.scale = scale;
	for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
		const int k = entry_of(a, tile);
		const TensorEntry& e = a.entry[k];
		const uint64_t n = e.info & kCountMask;
		const int ptype = (int) (e.info >> 56) & 3, gtype = (int) (e.info >> 58) & 3;
		const float decay = (e.info >> 60) & 1 ? 1.0f : s.decay;
		const uint64_t i = (uint64_t) (tile - e.tile0) * kTile + threadIdx.x * kLane;
		const uint64_t state = (a.block_base + e.block0) * kStateBlock;
		float* master = a.master && ptype != T_F32 ? a.master + state : nullptr;
		uint64_t word = 0;
		if (BITS == 8 || s.stochastic) word = finalise(s.key + ((state + i) >> 3) * kGolden);
		float g[kLane], w[kLane], m[kLane], v[kLane];
		if (BITS == 32) {
			if (i >= n) continue;
			const f32x4* pm = reinterpret_cast<const f32x4*>(static_cast<float*>(a.m) + state + i);
			const f32x4* pv = reinterpret_cast<const f32x4*>(static_cast<float*>(a.v) + state + i);
			load8(e.grad, i, n, gtype, g);
			load8(master ? master : e.param, i, n, master ? T_F32 : ptype, w);
			const f32x4 m0 = pm[0], m1 = pm[1], v0 = pv[0], v1 = pv[1];
#pragma unroll
			for (int j = 0; j < 4; j++) { m[j] = m0[j]; m[4 + j] = m1[j]; v[j] = v0[j]; v[4 + j] = v1[j]; }
#pragma unroll
			for (int j = 0; j < kLane; j++) update(s, decay, g[j] * s.scale, m[j], v[j], w[j]);
			store8(static_cast<float*>(a.m) + state, i, n, m);
			store8(static_cast<float*>(a.v) + state, i, n, v);
		} else {
			if ((i & ~(uint64_t) (kStateBlock - 1)) >= n) continue;      // whole blocks of 16 lanes leave together
			const uint64_t b = (state + i) / kStateBlock;
			u32x2* cm = reinterpret_cast<u32x2*>(static_cast<uint8_t*>(a.m) + state + i);
			u32x2* cv = reinterpret_cast<u32x2*>(static_cast<uint8_t*>(a.v) + state + i);
			load8(e.grad, i, n, gtype, g);
			load8(master ? master : e.param, i, n, master ? T_F32 : ptype, w);
			decode8<false>(*cm, scale_float(a.m_scale[b]), m);
			decode8<true>(*cv, scale_float(a.v_scale[b]), v);
			uint32_t tm = 0, tv = 0;                                    // bits of magnitudes order like the magnitudes, infinity and NaN last
#pragma unroll
			for (int j = 0; j < kLane; j++) {
				update(s, decay, g[j] * s.scale, m[j], v[j], w[j]);
				tm = max(tm, float_bits(m[j]) & 0x7fffffffu);
				tv = max(tv, float_bits(v[j]) & 0x7fffffffu);
			}
			const uint32_t bm = scale_byte(block_max(tm), 7), bv = scale_byte(block_max(tv), 14);
			*cm = encode8<false>(m, bm, (uint32_t) word);
			*cv = encode8<true>(v, bv, (uint32_t) (word >> 32));
			if ((threadIdx.x & 15) == 0) { a.m_scale[b] = (uint8_t) bm; a.v_scale[b] = (uint8_t) bv; }
			if (i >= n) continue;
		}
		put_weights(a, s, e.param, i, n, ptype, master, w, (uint32_t) word);
	}
	// the last workgroup to arrive counts the step: by then every other one has read the counter
	if (a.last && threadIdx.x == 0) {
		unsigned long long* arrived = reinterpret_cast<unsigned long long*>(a.count + 1);
		if (__hip_atomic_fetch_add(arrived, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1) {
			__hip_atomic_store(arrived, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
			a.count[0] = t;
		}
	}
}

// ---- the norm ------------------------------------------------------------------------------------------------------------------------
// Squares are summed in f64: f32 gradients reach 3e38, whose square is past f32, and 1e9 of them add up.  The order is fixed by the sizes
// alone -- lane, wave, workgroup, then the partial sums by one workgroup -- so that the same gradients give the same bits.
__device__ inline double block_sum(double x)
{
	__shared__ double wave[kThreads / 64];
#pragma unroll
	for (int d = 32; d; d >>= 1) x += __shfl_down(x, d);
	if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = x;
	__syncthreads();
	return wave[0] + wave[1] + wave[2] + wave[3];
}

// a norm that is not finite leaves NaN as the coefficient: the step that takes it is rejected
__device__ inline void verdict(double sum, double grad_scale, double max_norm, float* out)
{
	const double norm = sqrt(sum) * fabs(grad_scale);
	const bool finite = norm <= 1.7976931348623157e308;
	out[0] = (float) norm;
	out[1] = !finite ? __builtin_nanf("") : (float) (norm > max_norm ? grad_scale * (max_norm / norm) : grad_scale);
}

__global__ __launch_bounds__(kThreads) void k_norm(const NormArgs a)
{
	double sum = 0;
	for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
		const TensorEntry& e = a.entry[entry_of(a, tile)];
		const uint64_t n = e.info & kCountMask;
		const uint64_t i = (uint64_t) (tile - e.tile0) * kTile + threadIdx.x * kLane;
		if (i >= n) continue;
		float g[kLane];
		load8(e.grad, i, n, (int) (e.info >> 58) & 3, g);
#pragma unroll
		for (int j = 0; j < kLane; j++) sum = fma((double) g[j], (double) g[j], sum);
	}
	sum = block_sum(sum);
	if (threadIdx.x) return;
	if (a.out) verdict(sum, a.grad_scale, a.max_norm, a.out);
	else a.part[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kThreads) void k_norm_sum(double* part, int count, double grad_scale, double max_norm, float* out)
{
	double sum = 0;
	for (int i = threadIdx.x; i < count; i += kThreads) sum += part[1 + i];
	sum = block_sum(sum);
	if (threadIdx.x) return;
	part[0] = sum;
	if (out) verdict(sum, grad_scale, max_norm, out);
}

__global__ void k_norm_verdict(const double* sum, double grad_scale, double max_norm, float* out) { verdict(*sum, grad_scale, max_norm, out); }

}  // namespace

void launch_adamw(hipStream_t st, int bits, int grid, const AdamwArgs& a)
{
	if (bits == 8) k_adamw<8><<<grid, kThreads, 0, st>>>(a);
	else k_adamw<32><<<grid, kThreads, 0, st>>>(a);
}
void launch_norm(hipStream_t st, int grid, const NormArgs& a) { k_norm<<<grid, kThreads, 0, st>>>(a); }
void launch_norm_sum(hipStream_t st, double* part, int count, double grad_scale, double max_norm, float* out)
{
	k_norm_sum<<<1, kThreads, 0, st>>>(part, count, grad_scale, max_norm, out);
}
void launch_norm_verdict(hipStream_t st, const double* sum, double grad_scale, double max_norm, float* out)
{
	k_norm_verdict<<<1, 1, 0, st>>>(sum, grad_scale, max_norm, out);
}

}  // namespace sqn
