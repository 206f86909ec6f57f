// layer_norm.hip — layer norm forward and backward for rows of any width.
#include "layer_math.h"
#include "ngp_internal.h"

namespace ngp {

constexpr uint32_t NORM_BLOCK = 256;

__device__ __forceinline__ float block_sum(float v) {
	__shared__ float part[NORM_BLOCK / 64];
	for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
	__syncthreads();
	if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = v;
	__syncthreads();
	float s = 0.0f;
	for (uint32_t w = 0; w < NORM_BLOCK / 64; ++w) s += part[w];
	return s;
}

// One workgroup per row: the mean, then the mean square of what is left (no cancellation), then the row.
template <class T>
__global__ void __launch_bounds__(NORM_BLOCK) k_norm_forward(ngp_layer_norm_args a) {
	const size_t i = blockIdx.x;
	const T* x = static_cast<const T*>(a.x) + i * a.x_stride;
	T* y = static_cast<T*>(a.y) + i * a.y_stride;
	float s = 0.0f;
	for (uint32_t j = threadIdx.x; j < a.width; j += NORM_BLOCK) s += widen(x[j]);
	const float mean = block_sum(s) / (float)a.width;
	s = 0.0f;
	for (uint32_t j = threadIdx.x; j < a.width; j += NORM_BLOCK) {
		const float d = widen(x[j]) - mean;
		s += d * d;
	}
	const float rstd = 1.0f / sqrtf(block_sum(s) / (float)a.width + a.epsilon);
	if (threadIdx.x == 0) {
		if (a.mean) a.mean[i] = mean;
		if (a.rstd) a.rstd[i] = rstd;
	}
	for (uint32_t j0 = threadIdx.x & ~31u; j0 < a.width; j0 += NORM_BLOCK) {  // a half wave per 32 features
		const uint32_t j = j0 + (threadIdx.x & 31u);
		const bool in = j < a.width;
		const float v = in ? (widen(x[j]) - mean) * rstd * (a.gamma ? a.gamma[j] : 1.0f) + (a.beta ? a.beta[j] : 0.0f) : 0.0f;
		if (in) y[j] = narrow<T>(v);
		if (a.y8.q) {
			uint32_t top = magnitude_bits(v);
			for (int d = 16; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 32));
			const uint32_t scale = checkpoint_scale<T>(top);
			if (in) a.y8.q[i * a.y8.q_stride + j] = (int8_t)checkpoint_q(v, scale);
			if ((threadIdx.x & 31u) == 0) a.y8.scale[i * a.y8.scale_stride + j / 32u] = (uint8_t)scale;
		}
	}
}

template <class T>
__device__ __forceinline__ float at(const Kept<T>& x, size_t i, uint32_t j) {
	return x.v ? widen(x.v[i * x.stride + j]) : checkpoint_value(x.q[i * x.q_stride + j], x.scale[i * x.scale_stride + (j >> 5)]);
}

template <class T>
__global__ void __launch_bounds__(NORM_BLOCK) k_norm_backward_rows(ngp_layer_norm_backward_args a) {
	const size_t i = blockIdx.x;
	const Kept<T> x = {static_cast<const T*>(a.x), a.x_stride, a.x8.q, a.x8.scale, a.x8.q_stride, a.x8.scale_stride};
	const T* dy = static_cast<const T*>(a.dy) + i * a.dy_stride;
	const float mean = a.mean[i], rstd = a.rstd[i];
	float s0 = 0.0f, s1 = 0.0f;
	for (uint32_t j = threadIdx.x; j < a.width; j += NORM_BLOCK) {
		const float g = widen(dy[j]) * (a.gamma ? a.gamma[j] : 1.0f);
		s0 += g;
		s1 += g * ((at(x, i, j) - mean) * rstd);
	}
	s0 = block_sum(s0) / (float)a.width;
	s1 = block_sum(s1) / (float)a.width;
	for (uint32_t j = threadIdx.x; j < a.width; j += NORM_BLOCK) {
		const float g = widen(dy[j]) * (a.gamma ? a.gamma[j] : 1.0f);
		float d = rstd * (g - s0 - (at(x, i, j) - mean) * rstd * s1);
		if (a.dx_add) d += widen(static_cast<const T*>(a.dx_add)[i * a.dx_add_stride + j]);
		static_cast<T*>(a.dx)[i * a.dx_stride + j] = narrow<T>(d);
	}
}

// 64 columns x a share of the rows per workgroup, summed over the shares afterwards in their order.
template <class T>
__global__ void __launch_bounds__(NORM_BLOCK) k_norm_backward_columns(ngp_layer_norm_backward_args a, uint32_t rows_each,
                                                                      float* __restrict__ part) {
	const Kept<T> x = {static_cast<const T*>(a.x), a.x_stride, a.x8.q, a.x8.scale, a.x8.q_stride, a.x8.scale_stride};
	const uint32_t j = blockIdx.x * 64u + (threadIdx.x & 63u), w = threadIdx.x >> 6;
	const size_t begin = (size_t)blockIdx.y * rows_each, end = min(begin + rows_each, (size_t)a.n);
	float g = 0.0f, b = 0.0f;
	if (j < a.width) {
		for (size_t i = begin + w; i < end; i += NORM_BLOCK / 64) {
			const float d = widen(static_cast<const T*>(a.dy)[i * a.dy_stride + j]);
			g += d * ((at(x, i, j) - a.mean[i]) * a.rstd[i]);
			b += d;
		}
	}
	__shared__ float sg[NORM_BLOCK], sb[NORM_BLOCK];
	sg[threadIdx.x] = g;
	sb[threadIdx.x] = b;
	__syncthreads();
	if (w == 0 && j < a.width) {
		const uint32_t t = threadIdx.x;
		part[((size_t)blockIdx.y * 2 + 0) * a.width + j] = (sg[t] + sg[t + 64]) + (sg[t + 128] + sg[t + 192]);
		part[((size_t)blockIdx.y * 2 + 1) * a.width + j] = (sb[t] + sb[t + 64]) + (sb[t + 128] + sb[t + 192]);
	}
}

__global__ void k_norm_backward_sum(const float* __restrict__ part, uint32_t shares, uint32_t width, float* dgamma,
                                    float* dbeta, int accumulate) {
	const uint32_t j = blockIdx.x * 256u + threadIdx.x;
	if (j >= width) return;
	float g = 0.0f, b = 0.0f;
	for (uint32_t s = 0; s < shares; ++s) {
		g += part[((size_t)s * 2 + 0) * width + j];
		b += part[((size_t)s * 2 + 1) * width + j];
	}
	if (dgamma) dgamma[j] = accumulate ? dgamma[j] + g : g;
	if (dbeta) dbeta[j] = accumulate ? dbeta[j] + b : b;
}

static uint32_t norm_shares(uint32_t n) { return std::max(1u, std::min(256u, n / 64u)); }

size_t layer_norm_backward_workspace(const ngp_layer_norm_backward_args& a) {
	return a.dgamma || a.dbeta ? (size_t)norm_shares(a.n) * 2 * a.width * sizeof(float) : 0;
}

template <class T>
static void norm_backward(const ngp_layer_norm_backward_args& a, hipStream_t s) {
	if (a.dgamma || a.dbeta) {  // before dx: a row of dx may take the place of dx_add's, never of what these sums read
		const uint32_t shares = norm_shares(a.n), each = (a.n + shares - 1) / shares;
		float* part = static_cast<float*>(a.workspace);
		k_norm_backward_columns<T><<<dim3((a.width + 63) / 64, shares), NORM_BLOCK, 0, s>>>(a, each, part);
		NGP_HIP_CHECK(hipGetLastError());
		k_norm_backward_sum<<<(a.width + 255) / 256, 256, 0, s>>>(part, shares, a.width, a.dgamma, a.dbeta, a.accumulate);
		NGP_HIP_CHECK(hipGetLastError());
	}
	if (a.dx && a.n) {
		k_norm_backward_rows<T><<<a.n, NORM_BLOCK, 0, s>>>(a);
		NGP_HIP_CHECK(hipGetLastError());
	}
}

void run_layer_norm_forward(const ngp_layer_norm_args& a, hipStream_t s) {
	if (!a.n) return;
	if (a.type == NGP_TYPE_F32) k_norm_forward<float><<<a.n, NORM_BLOCK, 0, s>>>(a);
	else if (a.type == NGP_TYPE_F16) k_norm_forward<f16><<<a.n, NORM_BLOCK, 0, s>>>(a);
	else k_norm_forward<bf16><<<a.n, NORM_BLOCK, 0, s>>>(a);
	NGP_HIP_CHECK(hipGetLastError());
}

void run_layer_norm_backward(const ngp_layer_norm_backward_args& a, hipStream_t s) {
	if (a.type == NGP_TYPE_F32) norm_backward<float>(a, s);
	else if (a.type == NGP_TYPE_F16) norm_backward<f16>(a, s);
	else norm_backward<bf16>(a, s);
}

}  // namespace ngp
