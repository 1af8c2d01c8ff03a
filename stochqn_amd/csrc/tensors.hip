// tensors.hip -- the AdamW step over many tensors at once and the norm over all their gradients.
//
// For every element, with the step's number t counted from 1 and all arithmetic in f32:
//   g <- grad_scale * g;   m <- b1 m + (1 - b1) g;   v <- b2 v + (1 - b2) g^2
//   w <- w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Every array is read once and written once; nothing is reused, so HBM bounds the step: 28 B per element with f32 weights and
// moments, 10 B with bf16 weights and 8-bit moments.  Reached (MI355X): 1e8 f32 elements 474 us = 5.9 TB/s, where four read and three
// write streams without arithmetic reach 5.4 - 5.77 and a copy 4.8; with 8-bit moments 304 us = 5.3 TB/s; 1.28e9 bf16 elements with
// 8-bit moments 2.41 ms = 5.3 TB/s (the same streams without arithmetic: 2.33 - 2.53 ms), with f32 weights beside them and 32-bit
// moments 6.52 ms = 5.5 TB/s.  Counted traffic is 1.00 - 1.04 of those bytes.  24 vector instructions per element (8 bits) are
// below a third of the time.  All accesses stream (non-temporal: 8 % at 1e8).  m and v are formed by separate products and sums (no fma), so that they -- and
// with them the 8-bit codes -- do not depend on what a compiler contracts.
#include "tensors.hpp"

namespace sqn {
namespace {

constexpr int kThreads = 256;

// Tensors are aligned to their elements only, the arrays of the state to 16 bytes; global memory takes wide accesses at any address.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <class T, int ALIGN> struct Aligned;
template <int ALIGN> struct Aligned<u32x4, ALIGN> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Aligned<u32x4, 16> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(16))); };
template <> struct Aligned<u32x4, 4> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4))); };
template <int ALIGN> struct Aligned<u32x2, ALIGN> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Aligned<u32x2, 8> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(8))); };

template <int ALIGN, class T> __device__ inline void fetch(const void* p, T& x)
{
	x = __builtin_nontemporal_load(static_cast<const typename Aligned<T, ALIGN>::type*>(p));
}
template <int ALIGN, class T> __device__ inline void put(void* p, T x)
{
	__builtin_nontemporal_store((typename Aligned<T, ALIGN>::type) x, static_cast<typename Aligned<T, ALIGN>::type*>(p));
}

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

// What is known of a tensor where a tile of it is taken: nothing, or that the whole tile lies in it and how wide its elements are.
enum Kind { ANY, WIDE, HALF };

// V elements of a tensor on their way.  Every load has registers of its own: where two branches load into the same ones the compiler copies,
// and waits for each load before it issues the next (1e8 f32 elements with 32-bit moments: 487 us so, 474 like this).
template <int V> struct Raw;
template <> struct Raw<8> { u32x4 a, b; };                                   // f32: a, b; 16 bits: a
template <> struct Raw<4> { u32x4 a; u32x2 b; };                             // f32: a; 16 bits: b

// elements i .. i+V-1 of a tensor of n, if all of them exist
template <int V, Kind K = ANY> __device__ inline void load(const void* base, uint64_t i, uint64_t n, int type, Raw<V>& x)
{
	if (K == ANY && i + V > n) return;
	const bool wide = K == ANY ? type == T_F32 : K == WIDE;
	const char* at = static_cast<const char*>(base) + (i << (wide ? 2 : 1));
	if constexpr (V == 8) {
		fetch<2>(at, x.a);
		if (wide) fetch<4>(at + 16, x.b);
	} else {
		if (wide) fetch<4>(at, x.a);
		if (!wide) fetch<2>(at, x.b);
	}
}
// ... as f32.  Where a tensor ends inside of them they are loaded here, one by one; what lies behind its end is zero.
template <int V, Kind K = ANY> __device__ inline void widen(const Raw<V>& r, const void* base, uint64_t i, uint64_t n, int type, float (&x)[V])
{
	if (K == ANY && i + V > n) {
#pragma unroll
		for (int j = 0; j < V; j++) {
			x[j] = 0;
			if (i + j < n) x[j] = type == T_F32 ? static_cast<const float*>(base)[i + j] : widen16(static_cast<const uint16_t*>(base)[i + j], type);
		}
	} else if (K == ANY ? type == T_F32 : K == WIDE) {
#pragma unroll
		for (int j = 0; j < V; j++) x[j] = bits_float(j < 4 ? r.a[j] : r.b[j & 3]);
	} else {
		uint32_t h[V / 2];
#pragma unroll
		for (int j = 0; j < V / 2; j++) {
			if constexpr (V == 8) h[j] = r.a[j];
			else h[j] = r.b[j];
		}
		if (type == T_BF16) {
#pragma unroll
			for (int j = 0; j < V; j += 2) { x[j] = bits_float(h[j / 2] << 16); x[j + 1] = bits_float(h[j / 2] & 0xffff0000u); }
		} else {
#pragma unroll
			for (int j = 0; j < V; j += 2) { x[j] = widen16(h[j / 2] & 0xffff, T_F16); x[j + 1] = widen16(h[j / 2] >> 16, T_F16); }
		}
	}
}
template <int V, int ALIGN> __device__ inline void store32(float* base, uint64_t i, uint64_t n, const float (&x)[V])
{
	if (i + V <= n) {
#pragma unroll
		for (int j = 0; j < V; j += 4) put<ALIGN>(base + i + j, u32x4{float_bits(x[j]), float_bits(x[j + 1]), float_bits(x[j + 2]), float_bits(x[j + 3])});
	} else {
#pragma unroll
		for (int j = 0; j < V; j++)
			if (i + j < n) base[i + j] = x[j];
	}
}
template <int V> __device__ inline void store16(uint16_t* base, uint64_t i, uint64_t n, const uint32_t (&h)[V / 2])
{
	if (i + V <= n) {
		if constexpr (V == 8) put<2>(base + i, u32x4{h[0], h[1], h[2], h[3]});
		else put<2>(base + i, u32x2{h[0], h[1]});
	} else {
#pragma unroll
		for (int j = 0; j < V; j++)
			if (i + j < n) base[i + j] = (uint16_t) (h[j / 2] >> 16 * (j & 1));
	}
}

// the tensor that a workgroup is at: found by bisection once, then followed (its tiles come in rising order)
template <class T> struct Cursor {
	const T& t;
	int k;
	uint32_t next;
	__device__ Cursor(const T& table, uint32_t tile) : t(table)
	{
		int lo = 0, hi = t.a.entries;
		while (hi - lo > 1) {
			const int mid = (lo + hi) >> 1;
			if (t.entry[mid].tile0 <= tile) lo = mid; else hi = mid;
		}
		k = lo;
		next = end();
	}
	__device__ uint32_t end() const { return k + 1 < t.a.entries ? t.entry[k + 1].tile0 : 0xffffffffu; }
	__device__ const TensorEntry& at(uint32_t tile)
	{
		while (tile >= next) { k++; next = end(); }
		return t.entry[k];
	}
};

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
	bool go, stochastic, careful;
};

__device__ inline Step step_of(const AdamwArgs& a, long long t, float scale, double lr)
{
	Step s{};
	// A scale or a step size that is not finite, here or as the f32 numbers formed below: the step is rejected as a whole, nothing changes and
	// nothing is counted.  Every wave of every launch of the step decides alike: by the same scalars and the same count.
	s.scale = scale;
	s.go = __builtin_isfinite(s.scale) && __builtin_isfinite(lr);
	if (!s.go) return s;
	double p1 = 1, p2 = 1, q1 = a.beta1, q2 = a.beta2;       // b^t by squaring, in f64: 1 - b2^t loses ten bits at t = 1
	for (unsigned long long k = (unsigned long long) t; k; k >>= 1) {
		if (k & 1) { p1 *= q1; p2 *= q2; }
		q1 *= q1;
		q2 *= q2;
	}
	s.b1 = (float) a.beta1;
	s.b2 = (float) a.beta2;
	s.a1 = (float) (1 - a.beta1);
	s.a2 = (float) (1 - a.beta2);
	s.decay = (float) (1 - lr * a.weight_decay);
	// Reciprocal and reciprocal root: the hardware's, good to about 2^-23, and one Newton step, which squares that error; the results are
	// rounded to f32.  Division and root in full cost every wave some 40 f64 instructions more: 21.6 against 20.8 us at 7.7e6 elements
	// with 8-bit moments, 5.8 against 5.0 us for the smallest call.
	const double d1 = 1 - p1, d2 = 1 - p2;
	double y1 = __builtin_amdgcn_rcp(d1), y2 = __builtin_amdgcn_rsq(d2);
	y1 = fma(fma(-d1, y1, 1.0), y1, y1);
	y2 = fma(fma(-d2 * y2, y2, 1.0), 0.5 * y2, y2);
	s.rate = (float) (lr * y1);
	s.go = __builtin_isfinite(s.rate) && __builtin_isfinite(s.decay);
	s.root = (float) y2;
	s.eps = a.eps;
	s.key = finalise(a.seed ^ (uint64_t) t * kStepKey);
	s.stochastic = a.stochastic != 0;
	s.careful = s.root * 0x1p-63f > s.eps * 0x1p-25f;
	return s;
}

// Moments and weight of one element.  The hardware's root and reciprocal are within an ulp (1.6 and 1.5 times 2^-24, measured over all
// exponents), far below the weight's own rounding, and a quarter of the instructions of the exact ones.  The root takes subnormals for
// zero: their true roots are below 2^-63, nothing beside eps unless eps is tiny (`careful`).
__device__ inline void update(const Step& s, float decay, float g, float& m, float& v, float& w)
{
	m = m * s.b1 + g * s.a1;
	v = v * s.b2 + (g * g) * s.a2;
	float q = __builtin_amdgcn_sqrtf(v);
	if (s.careful && v < 0x1p-64f) q = __builtin_amdgcn_sqrtf(v * 0x1p64f) * 0x1p-32f;
	w = fmaf(-s.rate, m * __builtin_amdgcn_rcpf(fmaf(q, s.root, s.eps)), w * decay);
}

// the new weights go out: f32 as they are, 16 bits rounded (to nearest, or stochastically by the low half of the first word: bf16 is
// the upper half of f32, so the word's 16 bits are added to the lower half and cut off with it)
template <int V> __device__ inline void put_weights(const Step& s, void* param, uint64_t i, uint64_t n, int ptype, float* master, const float (&w)[V], uint32_t word)
{
	if (ptype == T_F32) { store32<V, 4>(static_cast<float*>(param), i, n, w); return; }
	if (master) store32<V, 16>(master, i, n, w);
	uint32_t h[V / 2];
	if (ptype == T_F16) {
#pragma unroll
		for (int j = 0; j < V; j += 2) h[j / 2] = narrow16(w[j], T_F16) | narrow16(w[j + 1], T_F16) << 16;
	} else if (s.stochastic) {
		uint32_t b[V];
#pragma unroll
		for (int j = 0; j < V; j++) b[j] = float_bits(w[j]) + (__builtin_isfinite(w[j]) ? (word + j * kLaneStep) & 0xffff : 0u);
#pragma unroll
		for (int j = 0; j < V; j += 2) h[j / 2] = __builtin_amdgcn_perm(b[j + 1], b[j], 0x07060302u);
	} else {
#pragma unroll
		for (int j = 0; j < V; j += 2) h[j / 2] = narrow16(w[j], T_BF16) | narrow16(w[j + 1], T_BF16) << 16;
	}
	store16<V>(static_cast<uint16_t*>(param), i, n, h);
}

// ---- moments in 8 bits -------------------------------------------------------------------------------------------------------------
// A block of 128 elements shares a scale 2^k (a byte, the exponent's 8 bits): the largest |m| lies at 2^7 .. 2^8 of it, the largest v at
// 2^14 .. 2^15, so that rounding up stays inside e4m3 (448) and e5m2 (57344).  A power of two costs no precision in a floating
// format and makes every product with it exact.  16 lanes hold a block, eight elements each.
// The conversions of gfx950 take the scale as an f32 of which they use the exponent: byte << 23, and 255 reads as NaN.
__device__ inline float scale_float(uint32_t byte) { return bits_float(byte << 23); }

template <class F> __device__ inline uint32_t row_reduce(uint32_t x, F f)            // over the 16 lanes of a block
{
	x = f(x, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, 0x128, 0xf, 0xf, false));     // rotated within the row by 8, 4, 2, 1
	x = f(x, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, 0x124, 0xf, 0xf, false));
	x = f(x, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, 0x122, 0xf, 0xf, false));
	x = f(x, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, 0x121, 0xf, 0xf, false));
	return x;
}

// byte of the scale for a block whose largest magnitude has the bits `top`; `at`: the power of two of the scale that it is brought to
__device__ inline uint32_t scale_byte(uint32_t top, int at)
{
	const int e = (int) (top >> 23) - at;
	return top >= 0x7f800000u ? 255u : (uint32_t) (e > 1 ? e : 1);
}

constexpr int kLane = 8;                                                     // elements of a block per lane

template <bool SECOND> __device__ inline void encode(const float (&x)[kLane], uint32_t byte, uint32_t word, u32x2& c)
{
	const float scale = scale_float(byte);
	// a second moment above zero stays above zero (the least code, 2^-16): m / (sqrt(0) + eps) would be a jump
	const float least = 0x1p-16f * scale;
	int out[2] = {0, 0};
	const auto one = [&](int j) {
		const float y = SECOND ? (x[j] > 0 ? fmaxf(x[j], least) : x[j]) : x[j];
		return y;
	};
#define TS_ENC(j, sel) out[(j) >> 2] = SECOND ? __builtin_amdgcn_cvt_scalef32_sr_bf8_f32(out[(j) >> 2], one(j), word + (j) * kLaneStep, scale, sel) \
	: __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(out[(j) >> 2], one(j), word + (j) * kLaneStep, scale, sel)
	TS_ENC(0, 0); TS_ENC(1, 1); TS_ENC(2, 2); TS_ENC(3, 3);
	TS_ENC(4, 0); TS_ENC(5, 1); TS_ENC(6, 2); TS_ENC(7, 3);
#undef TS_ENC
	c = u32x2{(uint32_t) out[0], (uint32_t) out[1]};
}

template <bool SECOND> __device__ inline void decode(u32x2 c, float scale, float (&x)[kLane])
{
#pragma unroll
	for (int k = 0; k < 2; k++) {
		const auto p = SECOND ? __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(c[k], scale, false) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[k], scale, false);
		const auto q = SECOND ? __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(c[k], scale, true) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[k], scale, true);
		x[4 * k] = p[0]; x[4 * k + 1] = p[1]; x[4 * k + 2] = q[0]; x[4 * k + 3] = q[1];
	}
}

// ---- the kernels -------------------------------------------------------------------------------------------------------------------
struct Place {                                                               // a tensor as the lanes see it
	void* param;
	const void* grad;
	uint64_t n, state;
	float* master;
	int ptype, gtype;
	bool decays;
	__device__ int wtype() const { return master ? (int) T_F32 : ptype; }
	__device__ const void* weights() const { return master ? master : param; }
};
__device__ inline Place place_of(const AdamwArgs& a, const TensorEntry& e)
{
	Place p;
	p.param = e.param;
	p.grad = e.grad;
	p.n = e.info & kCountMask;
	p.ptype = (int) (e.info >> 56) & 3;
	p.gtype = (int) (e.info >> 58) & 3;
	p.decays = !((e.info >> 60) & 1);
	p.state = (a.block_base + e.block0) * kStateBlock;
	p.master = a.master && p.ptype != T_F32 ? a.master + p.state : nullptr;
	return p;
}

__device__ inline uint64_t word_of(const Step& s, uint64_t element) { return finalise(s.key + (element >> 3) * kGolden); }

// A tile with moments in 32 bits: four elements per lane (16 B of every f32 array), U such groups in flight.
template <int TILE> struct Tile32 {
	static constexpr int V = 4, U = TILE / kThreads / V;
	Raw<V> g[U], w[U];
	u32x4 m[U], v[U];
	__device__ static uint64_t at(uint64_t first, int u) { return first + (u * kThreads + threadIdx.x) * V; }
	__device__ void load(const AdamwArgs& a, const Place& p, uint64_t first)
	{
#pragma unroll
		for (int u = 0; u < U; u++) {
			const uint64_t i = at(first, u);
			if (i >= p.n) continue;
			sqn::load<V>(p.grad, i, p.n, p.gtype, g[u]);
			sqn::load<V>(p.weights(), i, p.n, p.wtype(), w[u]);
			fetch<16>(static_cast<float*>(a.m) + p.state + i, m[u]);
			fetch<16>(static_cast<float*>(a.v) + p.state + i, v[u]);
		}
	}
	__device__ void work(const AdamwArgs& a, const Step& s, const Place& p, uint64_t first)
	{
		const float decay = p.decays ? s.decay : 1.0f;
#pragma unroll
		for (int u = 0; u < U; u++) {
			const uint64_t i = at(first, u);
			if (i >= p.n) continue;
			float fg[V], fw[V], fm[V], fv[V];
			widen<V>(g[u], p.grad, i, p.n, p.gtype, fg);
			widen<V>(w[u], p.weights(), i, p.n, p.wtype(), fw);
			uint32_t word = 0;
			if (s.stochastic) word = (uint32_t) word_of(s, p.state + i) + (uint32_t) (i & 7) * kLaneStep;
#pragma unroll
			for (int j = 0; j < V; j++) {
				fm[j] = bits_float(m[u][j]);
				fv[j] = bits_float(v[u][j]);
				update(s, decay, fg[j] * s.scale, fm[j], fv[j], fw[j]);
			}
			store32<V, 16>(static_cast<float*>(a.m) + p.state, i, p.n, fm);
			store32<V, 16>(static_cast<float*>(a.v) + p.state, i, p.n, fv);
			put_weights<V>(s, p.param, i, p.n, p.ptype, p.master, fw, word);
		}
	}
};

// A tile with moments in 8 bits: eight elements per lane, so that 16 lanes are a block; U such groups in flight.
template <int TILE> struct Tile8 {
	static constexpr int V = kLane, U = TILE / kThreads / V;
	Raw<V> g[U], w[U];
	u32x2 m[U], v[U];
	uint8_t ms[U], vs[U];
	__device__ static uint64_t at(uint64_t first, int u) { return first + (u * kThreads + threadIdx.x) * V; }
	__device__ static bool outside(uint64_t i, uint64_t n) { return (i & ~(uint64_t) (kStateBlock - 1)) >= n; }   // the same for the 16 lanes of a block
	__device__ void load(const AdamwArgs& a, const Place& p, uint64_t first)
	{
#pragma unroll
		for (int u = 0; u < U; u++) {
			const uint64_t i = at(first, u);
			if (outside(i, p.n)) continue;
			ms[u] = a.m_scale[(p.state + i) / kStateBlock];
			vs[u] = a.v_scale[(p.state + i) / kStateBlock];
			sqn::load<V>(p.grad, i, p.n, p.gtype, g[u]);
			sqn::load<V>(p.weights(), i, p.n, p.wtype(), w[u]);
			fetch<V>(static_cast<uint8_t*>(a.m) + p.state + i, m[u]);
			fetch<V>(static_cast<uint8_t*>(a.v) + p.state + i, v[u]);
		}
	}
	__device__ void work(const AdamwArgs& a, const Step& s, const Place& p, uint64_t first)
	{
		const float decay = p.decays ? s.decay : 1.0f;
		const auto larger = [](uint32_t x, uint32_t y) { return max(x, y); };
#pragma unroll
		for (int u = 0; u < U; u++) {
			const uint64_t i = at(first, u);
			if (outside(i, p.n)) continue;
			float fg[V], fw[V], fm[V], fv[V];
			widen<V>(g[u], p.grad, i, p.n, p.gtype, fg);
			widen<V>(w[u], p.weights(), i, p.n, p.wtype(), fw);
			decode<false>(m[u], scale_float(ms[u]), fm);
			decode<true>(v[u], scale_float(vs[u]), fv);
			const uint64_t word = word_of(s, p.state + i);
			// Bits of magnitudes order like the magnitudes, infinity and NaN last.  The first moment's maximum passes over NaN; but
			// where m is NaN so is v, of the same element.
			float tm = 0;
			uint32_t tv = 0;
#pragma unroll
			for (int j = 0; j < V; j++) {
				update(s, decay, fg[j] * s.scale, fm[j], fv[j], fw[j]);
				tm = fmaxf(tm, fabsf(fm[j]));
				tv = max(tv, float_bits(fv[j]) & 0x7fffffffu);
			}
			tv = row_reduce(tv, larger);
			if (tv >= 0x7f800000u) {
#pragma unroll
				for (int j = 0; j < V; j++)
					if (fm[j] != fm[j]) tm = __builtin_inff();
			}
			const uint32_t om = scale_byte(row_reduce(float_bits(tm), larger), 7), ov = scale_byte(tv, 14);
			u32x2 c;
			encode<false>(fm, om, (uint32_t) word, c);
			put<V>(static_cast<uint8_t*>(a.m) + p.state + i, c);
			encode<true>(fv, ov, (uint32_t) (word >> 32), c);
			put<V>(static_cast<uint8_t*>(a.v) + p.state + i, c);
			if ((threadIdx.x & 15) == 0) {
				a.m_scale[(p.state + i) / kStateBlock] = (uint8_t) om;
				a.v_scale[(p.state + i) / kStateBlock] = (uint8_t) ov;
			}
			if (i < p.n) put_weights<V>(s, p.param, i, p.n, p.ptype, p.master, fw, (uint32_t) word);
		}
	}
};

// Every wave reads the step counter and forms the step's numbers itself, while its first tile is on the way.  One thread of a workgroup arrives
// for its four waves, behind a barrier: only there have all of them read the counter (their stores wait for what they made of it).  The last
// workgroup to arrive counts the step.  (A kernel in front that did both cost 3.5 us a step; arrivals at one counter cost 6 us at 1000 workgroups.)  One launch of one workgroup takes 2.8 - 3.4 us.
template <template <int> class Tile, int TILE, int N> __global__ __launch_bounds__(kThreads) void k_adamw(const Table<AdamwArgs, N> table)
{
	const AdamwArgs& a = table.a;
	Cursor<Table<AdamwArgs, N>> cursor(table, blockIdx.x);
	const long long count = a.count[0] + 1;                 // read in front of every store: scalar loads
	const float scale = a.grad_scale ? *a.grad_scale : 1.0f;
	const double lr = a.step_size_dev ? (double) *a.step_size_dev : a.step_size;
	Tile<TILE> t;
	Place p{};
	uint64_t first = 0;
	const auto load = [&](uint32_t tile) {
		const TensorEntry& e = cursor.at(tile);
		p = place_of(a, e);
		first = (uint64_t) (tile - e.tile0) * TILE;
		t.load(a, p, first);
	};
	uint32_t tile = blockIdx.x;
	if (tile < a.tiles) load(tile);
	const Step s = step_of(a, count, scale, lr);
	if (!s.go) return;
	while (tile < a.tiles) {
		t.work(a, s, p, first);
		tile += gridDim.x;
		if (tile < a.tiles) load(tile);
	}
	if (!a.last) return;
	__syncthreads();
	if (threadIdx.x) return;
	const uint32_t gate = blockIdx.x % kGates, through = gridDim.x < kGates ? gridDim.x : kGates;
	uint32_t* arrived = reinterpret_cast<uint32_t*>(a.gates + gate * kGateStride);
	if (gridDim.x > 1) {
		if (__hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != (gridDim.x - gate - 1) / kGates) return;
		__hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
		unsigned long long* all = reinterpret_cast<unsigned long long*>(a.count + 1);
		if (__hip_atomic_fetch_add(all, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != through - 1) return;
		__hip_atomic_store(all, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
	}
	a.count[0] = count;
}

// ---- the norm ------------------------------------------------------------------------------------------------------------------------
// Bound by reading: 1.28e9 bf16 elements in 379 us = 6.75 TB/s, what the card reads at; below 1e7 elements by its two launches.  Tiles that
// lie in their tensor as a whole take code without a branch between its loads (1e8 f32 elements: 67.7 us, 72 with branches).
// Squares are summed in f64: f32 gradients reach 3e38, whose square is past f32, and 1e9 of them add up.  The order is fixed by the sizes
// alone -- lane, wave, workgroup, then the partial sums by one workgroup -- so that the same gradients give the same bits.
template <int THREADS> __device__ inline double block_sum(double x)
{
	__shared__ double wave[THREADS / 64];
#pragma unroll
	for (int d = 32; d; d >>= 1) x += __shfl_down(x, d);
	if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = x;
	__syncthreads();
	x = wave[0];
#pragma unroll
	for (int k = 1; k < THREADS / 64; k++) x += wave[k];
	return x;
}

// A norm that is not finite leaves NaN as the coefficient: the step that takes it is rejected.  Finite is what the caller sees, in f32.
__device__ inline void verdict(double sum, double grad_scale, double max_norm, float* out)
{
	const double norm = sqrt(sum) * fabs(grad_scale);
	out[0] = (float) norm;
	out[1] = !__builtin_isfinite((float) norm) ? __builtin_nanf("") : (float) (norm > max_norm ? grad_scale * (max_norm / norm) : grad_scale);
}

template <int TILE, Kind K> __device__ inline double squares(const void* grad, uint64_t first, uint64_t n, int type, double sum)
{
	constexpr int V = 8, U = TILE / kThreads / V;
	Raw<V> r[U];
#pragma unroll
	for (int u = 0; u < U; u++) load<V, K>(grad, first + (u * kThreads + threadIdx.x) * V, n, type, r[u]);
#pragma unroll
	for (int u = 0; u < U; u++) {
		const uint64_t i = first + (u * kThreads + threadIdx.x) * V;
		if (K == ANY && i >= n) continue;
		float g[V];
		widen<V, K>(r[u], grad, i, n, type, g);
#pragma unroll
		for (int j = 0; j < V; j++) sum = fma((double) g[j], (double) g[j], sum);
	}
	return sum;
}

template <int TILE, int N> __global__ __launch_bounds__(kThreads) void k_norm(const Table<NormArgs, N> table)
{
	const NormArgs& a = table.a;
	double sum = 0;
	Cursor<Table<NormArgs, N>> cursor(table, blockIdx.x);
	for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
		const TensorEntry& e = cursor.at(tile);
		const uint64_t n = e.info & kCountMask, first = (uint64_t) (tile - e.tile0) * TILE;
		const int type = (int) (e.info >> 58) & 3;
		if (first + TILE > n) sum = squares<TILE, ANY>(e.grad, first, n, type, sum);
		else if (type == T_F32) sum = squares<TILE, WIDE>(e.grad, first, n, type, sum);
		else sum = squares<TILE, HALF>(e.grad, first, n, type, sum);
	}
	sum = block_sum<kThreads>(sum);
	if (threadIdx.x) return;
	if (a.out) verdict(sum, a.grad_scale, a.max_norm, a.out);
	else a.part[blockIdx.x] = sum;
}

constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void k_norm_sum(double* part, int count, double grad_scale, double max_norm, float* out)
{
	double sum = 0;
	for (int i = threadIdx.x; i < count; i += kSumThreads) sum += part[1 + i];
	sum = block_sum<kSumThreads>(sum);
	if (threadIdx.x) return;
	part[0] = sum;
	if (out) verdict(sum, grad_scale, max_norm, out);
}

__global__ void k_norm_verdict(const double* sum, double grad_scale, double max_norm, float* out) { verdict(*sum, grad_scale, max_norm, out); }

}  // namespace

// a short list travels in a short table
template <class Args> static Table<Args, kFewEntries> few(const Table<Args, kEntries>& t)
{
	Table<Args, kFewEntries> f;
	f.a = t.a;
	for (int k = 0; k < t.a.entries; k++) f.entry[k] = t.entry[k];
	return f;
}

template <template <int> class Tile, int LARGE> static void launch_tiles(hipStream_t st, int tile, int grid, const Table<AdamwArgs, kEntries>& t)
{
	if (tile != kTileSmall) k_adamw<Tile, LARGE, kEntries><<<grid, kThreads, 0, st>>>(t);
	else if (t.a.entries > kFewEntries) k_adamw<Tile, kTileSmall, kEntries><<<grid, kThreads, 0, st>>>(t);
	else k_adamw<Tile, kTileSmall, kFewEntries><<<grid, kThreads, 0, st>>>(few(t));
}
void launch_adamw(hipStream_t st, int bits, int tile, int grid, const Table<AdamwArgs, kEntries>& t)
{
	if (bits == 8) launch_tiles<Tile8, kTile8>(st, tile, grid, t);
	else launch_tiles<Tile32, kTile32>(st, tile, grid, t);
}
void launch_norm(hipStream_t st, int tile, int grid, const Table<NormArgs, kEntries>& t)
{
	if (tile == kTileNorm) k_norm<kTileNorm, kEntries><<<grid, kThreads, 0, st>>>(t);
	else if (tile == kTileNormMid) k_norm<kTileNormMid, kEntries><<<grid, kThreads, 0, st>>>(t);
	else if (t.a.entries > kFewEntries) k_norm<kTileSmall, kEntries><<<grid, kThreads, 0, st>>>(t);
	else k_norm<kTileSmall, kFewEntries><<<grid, kThreads, 0, st>>>(few(t));
}
void launch_norm_sum(hipStream_t st, double* part, int count, double grad_scale, double max_norm, float* out)
{
	k_norm_sum<<<1, kSumThreads, 0, st>>>(part, count, grad_scale, max_norm, out);
}
void launch_norm_verdict(hipStream_t st, const double* sum, double grad_scale, double max_norm, float* out)
{
	k_norm_verdict<<<1, 1, 0, st>>>(sum, grad_scale, max_norm, out);
}

}  // namespace sqn
