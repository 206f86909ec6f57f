// layer_math.h — element types, activations and 8-bit checkpoints of the layer kernels (linear.hip, layer_norm.hip,
// checkpoint8.hip).  Device code only.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "ngp_internal.h"

namespace ngp {

typedef _Float16 f16;
typedef __bf16 bf16;

template <class T>
__device__ __forceinline__ float widen(T v) { return (float)v; }
template <class T>
__device__ __forceinline__ T narrow(float v) { return (T)v; }  // to nearest, ties to even

// A value of NGP_ACT_* and its derivative.  exp is the hardware's 2^x (v_exp_f32, ~1 ulp) of x log2(e) rounded once:
// relative error below 2^-23 (1 + |x|), against the half step 2^-12 / 2^-9 of the 16-bit results.
__device__ __forceinline__ float act_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float act_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// The normal distribution by a polynomial each, fitted for the least largest error (one exponential and no division, half the
// cost of a rational form of the tail: a 256 x 256 tile's 65536 gelus are a quarter of its time at K = 2048):
//  * the tail Phi(-a) = 2^L(a) for 0 <= a <= 8, degree 8: relative error 5.3e-6, 1.1e-5 with fp32 rounding.  Past 8 nothing
//    is left of it (6e-16).
//  * the gelu's slope at -a, Phi(-a) - a phi(a) = exp(-a^2 / 2) S(a), degree 9: off by 2.6e-7, 3.7e-7 with fp32 rounding (it
//    enters sums over all rows, which are held in fp32), and by less than 6e-8 past a = 6, where S(6) stands for S(a).
__device__ __forceinline__ float gelu_value(float z) {  // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
	const float a = fminf(fabsf(z), 8.0f);
	float l = 7.427881287228275e-08f;
	l = __builtin_fmaf(l, a, -3.655154276605529e-06f);
	l = __builtin_fmaf(l, a, 7.957170578537543e-05f);
	l = __builtin_fmaf(l, a, -0.001021958827187808f);
	l = __builtin_fmaf(l, a, 0.008762096122482587f);
	l = __builtin_fmaf(l, a, -0.05433718947457587f);
	l = __builtin_fmaf(l, a, -0.45819584686337644f);
	l = __builtin_fmaf(l, a, -1.1513217395138415f);
	l = __builtin_fmaf(l, a, -0.9999923663359365f);
	// max(z, 0) that keeps a NaN, in halves: z + |z| overflows from 2^127 on
	return __builtin_fmaf(-a, __builtin_amdgcn_exp2f(l), __builtin_fmaf(0.5f, fabsf(z), 0.5f * z));
}
__device__ __forceinline__ float gelu_slope(float z) {
	const float a = fminf(fabsf(z), 6.0f), bell = __builtin_amdgcn_exp2f(z * z * -0.7213475204444817f);  // -log2(e) / 2
	float s = -8.063526421414195e-06f;
	s = __builtin_fmaf(s, a, 0.00015194949927050064f);
	s = __builtin_fmaf(s, a, -0.0012712149702726438f);
	s = __builtin_fmaf(s, a, 0.006383002906360614f);
	s = __builtin_fmaf(s, a, -0.02223130768127502f);
	s = __builtin_fmaf(s, a, 0.05949735447645309f);
	s = __builtin_fmaf(s, a, -0.1317733057963848f);
	s = __builtin_fmaf(s, a, 0.24975246260495018f);
	s = __builtin_fmaf(s, a, -0.797864929825654f);
	s = __builtin_fmaf(s, a, 0.49999974472528175f);
	s *= bell;
	return z < 0.0f ? s : 1.0f - s;  // the slopes at z and -z add up to 1
}

__device__ __forceinline__ float act_value(int act, float z) {
	switch (act) {
		case NGP_ACT_RELU: return z <= 0.0f ? 0.0f : z;  // a NaN stays one
		case NGP_ACT_LOGISTIC: return act_rcp(1.0f + act_exp(-z));
		case NGP_ACT_EXPONENTIAL: return act_exp(z);
		case NGP_ACT_GELU: return gelu_value(z);
		case NGP_ACT_SILU: return z * act_rcp(1.0f + act_exp(-z));
		default: return z;
	}
}

__device__ __forceinline__ float act_slope(int act, float z) {
	switch (act) {
		case NGP_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
		case NGP_ACT_LOGISTIC: {
			const float s = act_rcp(1.0f + act_exp(-z));
			return s * act_rcp(1.0f + act_exp(z));  // 1 - s without the cancellation
		}
		case NGP_ACT_EXPONENTIAL: return act_exp(z);
		case NGP_ACT_GELU: return gelu_slope(z);
		case NGP_ACT_SILU: {
			const float s = act_rcp(1.0f + act_exp(-z));
			return s * __builtin_fmaf(z, 1.0f - s, 1.0f);
		}
		default: return 1.0f;
	}
}

// Eight neighbouring values at once: one branch on the activation, not eight.
__device__ __forceinline__ void act_values(int act, float (&v)[8]) {
	switch (act) {
		case NGP_ACT_RELU: for (float& x : v) x = act_value(NGP_ACT_RELU, x); break;
		case NGP_ACT_LOGISTIC: for (float& x : v) x = act_value(NGP_ACT_LOGISTIC, x); break;
		case NGP_ACT_EXPONENTIAL: for (float& x : v) x = act_value(NGP_ACT_EXPONENTIAL, x); break;
		case NGP_ACT_GELU: for (float& x : v) x = act_value(NGP_ACT_GELU, x); break;
		case NGP_ACT_SILU: for (float& x : v) x = act_value(NGP_ACT_SILU, x); break;
		default: break;
	}
}
__device__ __forceinline__ void act_slopes(int act, float (&v)[8]) {
	switch (act) {
		case NGP_ACT_RELU: for (float& x : v) x = act_slope(NGP_ACT_RELU, x); break;
		case NGP_ACT_LOGISTIC: for (float& x : v) x = act_slope(NGP_ACT_LOGISTIC, x); break;
		case NGP_ACT_EXPONENTIAL: for (float& x : v) x = act_slope(NGP_ACT_EXPONENTIAL, x); break;
		case NGP_ACT_GELU: for (float& x : v) x = act_slope(NGP_ACT_GELU, x); break;
		case NGP_ACT_SILU: for (float& x : v) x = act_slope(NGP_ACT_SILU, x); break;
		default: for (float& x : v) x = 1.0f; break;
	}
}

// Eight neighbouring elements of a row that has `left` of them left, at p: one wide access wherever the row starts (global
// memory takes 16 bytes at any address), element by element only at a row's end.
template <class T>
using v8 = T __attribute__((ext_vector_type(8), aligned(sizeof(T))));
template <class T>
__device__ __forceinline__ v8<T> load8_raw(const T* p, uint32_t left) {
	if (left >= 8) return *reinterpret_cast<const v8<T>*>(p);
	v8<T> x;
#pragma unroll
	for (int k = 0; k < 8; ++k) x[k] = (uint32_t)k < left ? p[k] : narrow<T>(0.0f);
	return x;
}
template <class T>
__device__ __forceinline__ void load8(const T* p, uint32_t left, float (&v)[8]) {
	const v8<T> x = load8_raw(p, left);
#pragma unroll
	for (int k = 0; k < 8; ++k) v[k] = widen(x[k]);
}
template <class T>
__device__ __forceinline__ void store8(T* p, uint32_t left, const float (&v)[8]) {
	v8<T> x;
#pragma unroll
	for (int k = 0; k < 8; ++k) x[k] = narrow<T>(v[k]);
	if (left >= 8) {
		*reinterpret_cast<v8<T>*>(p) = x;
	} else {
#pragma unroll
		for (int k = 0; k < 8; ++k)
			if ((uint32_t)k < left) p[k] = x[k];
	}
}

// ---- 8-bit checkpoints (ngp_checkpoint8) ----------------------------------------------------------------------
// A block's scale byte from the largest magnitude's bit pattern (patterns of non-negative floats order as the floats do,
// infinities and NaNs above all finite ones: their exponent field is 255, which marks the block).
template <class T>
__device__ __forceinline__ uint32_t checkpoint_scale(uint32_t max_bits) {
	const uint32_t e = max_bits >> 23;
	return std::is_same_v<T, f16> ? (e < 109u ? 109u : e) : e;
}
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// ldexp keeps the power of two exact over the whole range (133 - scale reaches past the largest float's exponent)
__device__ __forceinline__ float checkpoint_value(int q, uint32_t scale) {
	return scale == 255u ? __uint_as_float(0x7fc00000u) : ldexpf((float)q, (int)scale - 133);
}

// Eight neighbouring values of one block (the first at a multiple of 8) to and from a checkpoint's row.  Adding 1.5 2^23
// rounds to the nearest integer, ties to even, and leaves it in the sum's low bits.
typedef uint32_t q8 __attribute__((ext_vector_type(2), aligned(1)));
__device__ __forceinline__ void checkpoint_store8(int8_t* q, uint32_t left, uint32_t scale, const float (&v)[8]) {
	const int power = 133 - (int)scale;
	uint32_t w[2];
#pragma unroll
	for (int h = 0; h < 2; ++h) {
		uint32_t b[4];
#pragma unroll
		for (int k = 0; k < 4; ++k)
			b[k] = __float_as_uint(__builtin_amdgcn_fmed3f(ldexpf(v[4 * h + k], power), -127.0f, 127.0f) + 12582912.0f);
		// bytes 0 of two, then of all four
		const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
		w[h] = scale == 255u ? 0u : lo | hi;
	}
	if (left >= 8) {
		*reinterpret_cast<q8*>(q) = q8{w[0], w[1]};
	} else {
#pragma unroll
		for (int k = 0; k < 8; ++k)
			if ((uint32_t)k < left) q[k] = (int8_t)(w[k / 4] >> (8 * (k % 4)));
	}
}
__device__ __forceinline__ q8 checkpoint_load8_raw(const int8_t* q, uint32_t left) {
	if (left >= 8) return *reinterpret_cast<const q8*>(q);
	uint32_t w[2] = {0, 0};
#pragma unroll
	for (int k = 0; k < 8; ++k)
		if ((uint32_t)k < left) w[k / 4] |= (uint32_t)(uint8_t)q[k] << (8 * (k % 4));
	return q8{w[0], w[1]};
}
__device__ __forceinline__ void checkpoint_widen8(q8 w, uint32_t scale, float (&v)[8]) {
#pragma unroll
	for (int k = 0; k < 8; ++k) v[k] = checkpoint_value((int8_t)((k < 4 ? w.x : w.y) >> (8 * (k % 4))), scale);
}

// The largest of four neighbouring lanes' (lanes 4 k .. 4 k + 3).
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
	x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
	return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true));  // quad_perm 2 3 0 1
}

// Where a thread of a workgroup of 256 is among rows of `eighths` items, and how it steps by the whole grid without dividing
// again.
struct Walk {
	size_t i, di;
	uint32_t e, de, eighths;
	__device__ __forceinline__ explicit Walk(uint32_t eighths, uint32_t block = blockIdx.x, uint32_t blocks = gridDim.x) : eighths(eighths) {
		const size_t t = (size_t)block * 256u + threadIdx.x;
		const uint32_t step = blocks * 256u;
		i = t / eighths;
		e = (uint32_t)(t % eighths);
		di = step / eighths;
		de = step % eighths;
	}
	__device__ __forceinline__ void next() {
		i += di;
		e += de;
		if (e >= eighths) e -= eighths, ++i;
	}
};

// Activations as a backward pass finds them: [rows][stride] of T, or a checkpoint (v null), or absent (both null).
template <class T>
struct Kept {
	const T* v = nullptr;
	size_t stride = 0;
	const int8_t* q = nullptr;
	const uint8_t* scale = nullptr;
	size_t q_stride = 0, scale_stride = 0;
	struct Raw {  // eight neighbouring values as they lie: of T, or eight q in the first words and their scale
		uint32_t w[sizeof(T) * 2];
		uint32_t scale;
	};
	__device__ __forceinline__ Raw raw8_values(size_t i, uint32_t j, uint32_t left) const {
		Raw r = {};
		const v8<T> x = load8_raw(v + i * stride + j, left);
		__builtin_memcpy(r.w, &x, sizeof(r.w));
		return r;
	}
	__device__ __forceinline__ Raw raw8_checkpoint(size_t i, uint32_t j, uint32_t left) const {
		Raw r = {};
		const q8 x = checkpoint_load8_raw(q + i * q_stride + j, left);
		r.w[0] = x[0];
		r.w[1] = x[1];
		r.scale = scale[i * scale_stride + (j >> 5)];
		return r;
	}
	__device__ __forceinline__ Raw raw8(size_t i, uint32_t j, uint32_t left) const {
		return v ? raw8_values(i, j, left) : raw8_checkpoint(i, j, left);
	}
	__device__ __forceinline__ void widen8_values(const Raw& r, float (&x)[8]) const {
		v8<T> y;
		__builtin_memcpy(&y, r.w, sizeof(r.w));
#pragma unroll
		for (int k = 0; k < 8; ++k) x[k] = widen(y[k]);
	}
	__device__ __forceinline__ void widen8(const Raw& r, float (&x)[8]) const {
		if (v) {
			widen8_values(r, x);
		} else {
			checkpoint_widen8(q8{r.w[0], r.w[1]}, r.scale, x);
		}
	}
	template <bool VALUES>
	__device__ __forceinline__ void at8_of(size_t i, uint32_t j, uint32_t left, float (&x)[8]) const {
		if constexpr (VALUES) {
			load8(v + i * stride + j, left, x);
		} else {
			const q8 w = checkpoint_load8_raw(q + i * q_stride + j, left);
			checkpoint_widen8(w, scale[i * scale_stride + (j >> 5)], x);
		}
	}
	__device__ __forceinline__ void at8(size_t i, uint32_t j, uint32_t left, float (&x)[8]) const { widen8(raw8(i, j, left), x); }
};

template <class T>
inline Kept<T> kept(const void* v, uint32_t stride, const ngp_checkpoint8& c) {
	return Kept<T>{static_cast<const T*>(v), stride, c.q, c.scale, c.q_stride, c.scale_stride};
}

// put(j, the sum of part[0 .. shares)[j]) for j < columns, in a fixed order: 16 columns per workgroup by as many shares at a
// time as there are threads for, four reads on their way; a wave's four shares meet by lane exchange, the waves in LDS.
template <int THREADS, class Put>
__device__ __forceinline__ void column_sums(const float* __restrict__ part, uint32_t shares, size_t columns, const Put& put, uint32_t block) {
	constexpr uint32_t LINES = THREADS / 16;
	const uint32_t c = threadIdx.x % 16u, line = threadIdx.x / 16u;
	const size_t j = (size_t)block * 16u + c;
	float sum[4] = {};
	if (j < columns)
		for (uint32_t k = line; k < shares; k += 4u * LINES)
#pragma unroll
			for (uint32_t u = 0; u < 4; ++u)
				if (k + LINES * u < shares) sum[u] += part[(size_t)(k + LINES * u) * columns + j];
	float v = (sum[0] + sum[1]) + (sum[2] + sum[3]);
	v += __shfl_xor(v, 16);
	v += __shfl_xor(v, 32);
	__shared__ float s[THREADS / 64][16];
	if (threadIdx.x % 64u < 16u) s[threadIdx.x / 64u][c] = v;
	__syncthreads();
	if (line || j >= columns) return;
	v = 0.0f;
	for (int w = 0; w < THREADS / 64; ++w) v += s[w][c];
	put(j, v);
}

template <class Put>
__global__ void __launch_bounds__(1024) k_column_sums(const float* __restrict__ part, uint32_t shares, size_t columns, Put put) {
	column_sums<1024>(part, shares, columns, put, blockIdx.x);
}

template <class Put>
inline void launch_column_sums(const float* part, uint32_t shares, size_t columns, const Put& put, hipStream_t s) {
	k_column_sums<Put><<<(uint32_t)((columns + 15) / 16), 1024, 0, s>>>(part, shares, columns, put);
	NGP_HIP_CHECK(hipGetLastError());
}

// The first `width` columns' sums to out0, the others to out1; either may be null.
struct PutSums {
	float *out0, *out1;
	uint32_t width;
	bool accumulate;
	__device__ __forceinline__ void operator()(size_t j, float v) const {
		float* out = j < width ? out0 : out1;
		const size_t o = j < width ? j : j - width;
		if (out) out[o] = accumulate ? out[o] + v : v;
	}
};

}  // namespace ngp
