// layer_norm.hip — layer norm forward and backward for rows of any width.
//
// Both are bound by memory: forward reads x and writes y (and 33/32 bytes per value of its checkpoint), backward reads dy,
// x (or its checkpoint) and the other branch's gradient and writes dx.  So every value is read once and stays in registers:
// a row belongs to a group of G threads (4 .. 1024, a power of two), each of which holds up to C chunks of eight
// neighbouring features, chunk c of thread g at features 8 (c G + g).  Groups of up to a wave sum with lane exchanges
// alone, larger ones through LDS.  (Only fp32 rows over 32768 values, eight chunks in each of 1024 threads, are more than a
// thread's 128 registers hold: 6 of them spill.)
#include <algorithm>

#include "layer_math.h"
#include "ngp_internal.h"

namespace ngp {

// Sums over a group, the same bits in all its threads.  `part` (N floats per wave of the workgroup) is used in turn with
// another such piece of LDS (the caller's two), so that one barrier does.
template <int N>
__device__ __forceinline__ void group_sums(float (&v)[N], uint32_t G, float* part) {
	for (uint32_t d = 1; d < min(G, 64u); d *= 2)
#pragma unroll
		for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], d);
	if (G <= 64u) return;
	const uint32_t waves = G / 64u;
	if (threadIdx.x % 64u == 0)
#pragma unroll
		for (int k = 0; k < N; ++k) part[threadIdx.x / 64u * N + k] = v[k];
	__syncthreads();
	part += threadIdx.x / G * waves * N;
#pragma unroll
	for (int k = 0; k < N; ++k) {
		v[k] = part[k];
		for (uint32_t w = 1; w < waves; ++w) v[k] += part[w * N + k];
	}
}

constexpr uint32_t NORM_THREADS = 256;     // a workgroup's, unless a row's group is larger
constexpr uint32_t NORM_GRID = 1u << 20;  // workgroups at most side by side (a grid has fewer than 2^32 threads that way)

// The mean, then the mean square of what is left of it (no cancellation), then the row.
template <class T, int C>
__global__ void __launch_bounds__(1024) k_norm_forward(ngp_layer_norm_args a, uint32_t G) {
	__shared__ float part[2][16];
	const uint32_t g = threadIdx.x % G;
	const size_t i = ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * (blockDim.x / G) + threadIdx.x / G;
	const bool here = i < a.n;
	const T* x = static_cast<const T*>(a.x) + i * a.x_stride;
	v8<T> raw[C];
	uint32_t left[C];
	float s[1] = {0.0f};
#pragma unroll
	for (int c = 0; c < C; ++c) {
		const uint32_t j = (c * G + g) * 8u;
		left[c] = here && j < a.width ? a.width - j : 0u;
		raw[c] = load8_raw(x + j, left[c]);
	}
#pragma unroll
	for (int c = 0; c < C; ++c)
#pragma unroll
		for (int k = 0; k < 8; ++k) s[0] += widen(raw[c][k]);  // zeros past the row
	group_sums(s, G, part[0]);
	const float mean = s[0] / (float)a.width;
	s[0] = 0.0f;
#pragma unroll
	for (int c = 0; c < C; ++c)
#pragma unroll
		for (int k = 0; k < 8; ++k) {
			const float d = widen(raw[c][k]) - mean;
			s[0] += (uint32_t)k < left[c] ? d * d : 0.0f;
		}
	group_sums(s, G, part[1]);
	const float rstd = 1.0f / sqrtf(s[0] / (float)a.width + a.epsilon);
	if (here && g == 0) {
		if (a.mean) a.mean[i] = mean;
		if (a.rstd) a.rstd[i] = rstd;
	}
#pragma unroll
	for (int c = 0; c < C; ++c) {
		const uint32_t j = (c * G + g) * 8u;
		float v[8], gamma[8], beta[8];
#pragma unroll
		for (int k = 0; k < 8; ++k) gamma[k] = 1.0f, beta[k] = 0.0f;
		if (left[c] && a.gamma) load8(a.gamma + j, left[c], gamma);
		if (left[c] && a.beta) load8(a.beta + j, left[c], beta);
#pragma unroll
		for (int k = 0; k < 8; ++k) v[k] = (widen(raw[c][k]) - mean) * rstd * gamma[k] + beta[k];
		if (left[c]) store8(static_cast<T*>(a.y) + i * a.y_stride + j, left[c], v);
		if (!a.y8.q) continue;
		uint32_t top = 0;
#pragma unroll
		for (int k = 0; k < 8; ++k) top = max(top, (uint32_t)k < left[c] ? magnitude_bits(v[k]) : 0u);
		const uint32_t scale = checkpoint_scale<T>(quad_max(top));
		if (!left[c]) continue;
		checkpoint_store8(a.y8.q + i * a.y8.q_stride + j, left[c], scale, v);
		if (j % 32u == 0) a.y8.scale[i * a.y8.scale_stride + j / 32u] = (uint8_t)scale;
	}
}

// A workgroup takes every gridDim.x-th set of rows.  SUMS: it keeps its threads' columns of dgamma and dbeta in registers
// meanwhile and leaves their sums over its rows in part_out[blockIdx.x][2][width].
template <class T, int C, int THREADS, bool SUMS>
__global__ void __launch_bounds__(THREADS, THREADS > 256 ? 1 : 3) k_norm_backward(ngp_layer_norm_backward_args a, uint32_t G, float* __restrict__ part_out) {
	extern __shared__ float lds[];  // two shares of 32 floats, then the columns of the groups
	const Kept<T> x{static_cast<const T*>(a.x), a.x_stride, a.x8.q, a.x8.scale, a.x8.q_stride, a.x8.scale_stride};
	const uint32_t g = threadIdx.x % G, group = threadIdx.x / G, groups = THREADS / G;
	uint32_t left[C];
	float gamma[C][8], dg[SUMS ? C : 1][8] = {}, db[SUMS ? C : 1][8] = {};
#pragma unroll
	for (int c = 0; c < C; ++c) {
		const uint32_t j = (c * G + g) * 8u;
		left[c] = j < a.width ? a.width - j : 0u;
#pragma unroll
		for (int k = 0; k < 8; ++k) gamma[c][k] = 1.0f;
		if (left[c] && a.gamma) load8(a.gamma + j, left[c], gamma[c]);
	}
	uint32_t turn = 0;
	for (size_t i0 = (size_t)blockIdx.x * groups; i0 < a.n; i0 += (size_t)gridDim.x * groups, turn ^= 32u) {
		const size_t i = i0 + group;
		const bool here = i < a.n;
		v8<T> dy[C], add[C];
		typename Kept<T>::Raw raw[C];
#pragma unroll
		for (int c = 0; c < C; ++c) {
			const uint32_t j = (c * G + g) * 8u, l = here ? left[c] : 0u;
			dy[c] = load8_raw(static_cast<const T*>(a.dy) + i * a.dy_stride + j, l);
			raw[c] = {};
			if (l) raw[c] = x.raw8(i, j, l);
			add[c] = {};
			if (a.dx_add) add[c] = load8_raw(static_cast<const T*>(a.dx_add) + i * a.dx_add_stride + j, l);
		}
		const float mean = here ? a.mean[i] : 0.0f, rstd = here ? a.rstd[i] : 0.0f;
		float s[2] = {0.0f, 0.0f};
#pragma unroll
		for (int c = 0; c < C; ++c) {
			float xv[8];
			x.widen8(raw[c], xv);
#pragma unroll
			for (int k = 0; k < 8; ++k) {
				// past the row d and x are 0: 0 times -mean is 0, where times rstd it might be infinite, so that is left for the sum
				const float d = widen(dy[c][k]), centred = xv[k] - mean, e = d * gamma[c][k];
				s[0] += e;
				s[1] += e * centred;
				if constexpr (SUMS) dg[c][k] += d * (centred * rstd), db[c][k] += d;
			}
		}
		if (!a.dx) continue;
		s[1] *= rstd;
		group_sums(s, G, lds + turn);
		const float m0 = s[0] / (float)a.width, m1 = s[1] / (float)a.width;
#pragma unroll
		for (int c = 0; c < C; ++c) {
			float v[8], xv[8];
			x.widen8(raw[c], xv);
#pragma unroll
			for (int k = 0; k < 8; ++k)
				v[k] = rstd * (widen(dy[c][k]) * gamma[c][k] - m0 - (xv[k] - mean) * rstd * m1) + widen(add[c][k]);
			if (here && left[c]) store8(static_cast<T*>(a.dx) + i * a.dx_stride + (c * G + g) * 8u, left[c], v);
		}
	}
	if constexpr (!SUMS) return;
	float* columns = lds + 64;
	float* out = part_out + (size_t)blockIdx.x * 2u * a.width;
#pragma unroll
	for (int c = 0; c < C; ++c)
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			float v[8];
#pragma unroll
			for (int k = 0; k < 8; ++k) v[k] = h ? db[SUMS ? c : 0][k] : dg[SUMS ? c : 0][k];
			if (groups > 1) {  // the groups' sums in their order
				__syncthreads();
#pragma unroll
				for (int k = 0; k < 8; ++k) columns[k * THREADS + threadIdx.x] = v[k];
				__syncthreads();
				if (group == 0)
					for (uint32_t o = 1; o < groups; ++o)
#pragma unroll
						for (int k = 0; k < 8; ++k) v[k] += columns[k * THREADS + o * G + g];
			}
			if (group == 0 && left[c]) store8(out + (size_t)h * a.width + (c * G + g) * 8u, left[c], v);
		}
}

// Rows too wide for that (over NORM_IN_PASS): dx by a workgroup of 1024 per row that reads it twice, the second time from
// its caches, ...
template <class T>
__global__ void __launch_bounds__(1024) k_norm_backward_rows(ngp_layer_norm_backward_args a) {
	__shared__ float part[2][32];
	const Kept<T> x{static_cast<const T*>(a.x), a.x_stride, a.x8.q, a.x8.scale, a.x8.q_stride, a.x8.scale_stride};
	uint32_t turn = 0;
	for (size_t i = blockIdx.x; i < a.n; i += gridDim.x, turn ^= 1u) {
		const T* dy = static_cast<const T*>(a.dy) + i * a.dy_stride;
		const float mean = a.mean[i], rstd = a.rstd[i];
		auto chunk = [&](uint32_t j, float (&e)[8], float (&centred)[8]) {  // dy gamma and x - mean: 0 and -mean past the row
			const uint32_t left = a.width - j;
			float gamma[8];
#pragma unroll
			for (int k = 0; k < 8; ++k) gamma[k] = 1.0f;
			if (a.gamma) load8(a.gamma + j, left, gamma);
			load8(dy + j, left, e);
			x.at8(i, j, left, centred);
#pragma unroll
			for (int k = 0; k < 8; ++k) e[k] *= gamma[k], centred[k] -= mean;
		};
		float s[2] = {0.0f, 0.0f}, e[8], centred[8];
		for (uint32_t j = threadIdx.x * 8u; j < a.width; j += 8192u) {
			chunk(j, e, centred);
#pragma unroll
			for (int k = 0; k < 8; ++k) s[0] += e[k], s[1] += e[k] * centred[k];
		}
		s[1] *= rstd;
		group_sums(s, 1024u, part[turn]);
		s[0] /= (float)a.width;
		s[1] /= (float)a.width;
		for (uint32_t j = threadIdx.x * 8u; j < a.width; j += 8192u) {
			chunk(j, e, centred);
			float add[8] = {};
			if (a.dx_add) load8(static_cast<const T*>(a.dx_add) + i * a.dx_add_stride + j, a.width - j, add);
#pragma unroll
			for (int k = 0; k < 8; ++k) e[k] = rstd * (e[k] - s[0] - centred[k] * rstd * s[1]) + add[k];
			store8(static_cast<T*>(a.dx) + i * a.dx_stride + j, a.width - j, e);
		}
	}
}

// ... and dgamma and dbeta in a pass of their own: 64 x 8 columns by a share of the rows per workgroup, four rows at a time.
template <class T>
__global__ void __launch_bounds__(256) k_norm_backward_columns(ngp_layer_norm_backward_args a, size_t rows_each, float* __restrict__ part_out) {
	const Kept<T> x{static_cast<const T*>(a.x), a.x_stride, a.x8.q, a.x8.scale, a.x8.q_stride, a.x8.scale_stride};
	const uint32_t g = threadIdx.x % 64u, j = (blockIdx.x * 64u + g) * 8u, left = j < a.width ? a.width - j : 0u;
	const size_t begin = blockIdx.y * rows_each, end = min(begin + rows_each, (size_t)a.n);
	float v[2][8] = {};
	if (left)
		for (size_t i = begin + threadIdx.x / 64u; i < end; i += 4) {
			float d[8], xv[8];
			load8(static_cast<const T*>(a.dy) + i * a.dy_stride + j, left, d);
			x.at8(i, j, left, xv);
			const float mean = a.mean[i], rstd = a.rstd[i];
#pragma unroll
			for (int k = 0; k < 8; ++k) v[0][k] += d[k] * ((xv[k] - mean) * rstd), v[1][k] += d[k];
		}
	__shared__ float lds[8][256];
	for (int h = 0; h < 2; ++h) {
		__syncthreads();
#pragma unroll
		for (int k = 0; k < 8; ++k) lds[k][threadIdx.x] = v[h][k];
		__syncthreads();
		if (threadIdx.x >= 64u || !left) continue;
		float s[8];
#pragma unroll
		for (int k = 0; k < 8; ++k) s[k] = (lds[k][g] + lds[k][g + 64]) + (lds[k][g + 128] + lds[k][g + 192]);
		store8(part_out + ((size_t)blockIdx.y * 2u + h) * a.width + j, left, s);
	}
}

// A row's group: with many rows the smallest that holds the row in `most` chunks per thread (a wave's exchanges cost less
// than barriers); with fewer rows than fill the GPU's 1024 SIMDs twice the largest that leaves every thread a chunk.
struct NormShape {
	uint32_t G, chunks, threads;
};
static NormShape norm_shape(uint32_t n, uint32_t width, uint32_t most) {
	NormShape s{4, 1, NORM_THREADS};
	const uint32_t eighths = (width + 7) / 8;
	while (s.G < 64 && s.G < eighths) s.G *= 2;
	while (s.G < 1024 && s.G * (n < 2048 ? 1u : most) < eighths) s.G *= 2;
	while (s.G * s.chunks < eighths) s.chunks *= 2;
	s.threads = std::max(s.G, NORM_THREADS);
	return s;
}

template <class T>
static void norm_forward(const ngp_layer_norm_args& a, hipStream_t s) {
	const NormShape p = norm_shape(a.n, a.width, sizeof(T) == 4 ? 4 : 8);
	const uint32_t rows = p.threads / p.G, sets = (a.n + rows - 1) / rows;
	const dim3 grid(std::min(sets, NORM_GRID), (sets + NORM_GRID - 1) / NORM_GRID);
	auto kernel = p.chunks == 1 ? k_norm_forward<T, 1> : p.chunks == 2 ? k_norm_forward<T, 2> : p.chunks == 4 ? k_norm_forward<T, 4> : k_norm_forward<T, 8>;
	kernel<<<grid, p.threads, 0, s>>>(a, p.G);
	NGP_HIP_CHECK(hipGetLastError());
}

// Backward: a quarter of the chunks, since a thread keeps two sums per column.  As many workgroups per CU as their registers
// allow, three of 256 or (rows over 4096) one of 512, go through the rows in turns (65536 rows of 2048 fp16, in turn on one
// card: 214..217 us, with two per CU 232..241, with two and four chunks per thread 313..319).
constexpr uint32_t NORM_IN_PASS = 512 * 2 * 8;
struct NormBackwardPlan {
	NormShape shape;
	bool sums, in_pass;  // dgamma or dbeta wanted; by k_norm_backward
	uint32_t grid, parts;
};
static NormBackwardPlan backward_plan(const ngp_layer_norm_backward_args& a) {
	NormBackwardPlan p{norm_shape(a.n, a.width, 2), a.dgamma || a.dbeta, a.width <= NORM_IN_PASS, 0, 0};
	while (p.in_pass && p.shape.G > (a.width <= 4096 ? 256u : 512u)) p.shape.G /= 2, p.shape.chunks *= 2;
	p.shape.threads = std::max(p.shape.G, NORM_THREADS);
	const uint32_t rows = std::max(1u, p.shape.threads / p.shape.G), most = p.shape.threads > 256 ? 256 : 768;
	const uint32_t sets = std::max(1u, (a.n + rows - 1) / rows), turns = (sets + most - 1) / most;
	p.grid = (sets + turns - 1) / turns;
	p.parts = p.in_pass ? p.grid : std::max(1u, std::min(256u, a.n / 16u));
	return p;
}

size_t layer_norm_backward_workspace(const ngp_layer_norm_backward_args& a) {
	const NormBackwardPlan p = backward_plan(a);
	return p.sums ? (size_t)p.parts * 2 * a.width * sizeof(float) : 0;
}

template <class T, int C>
static void launch_backward(const ngp_layer_norm_backward_args& a, const NormBackwardPlan& p, float* part, hipStream_t s) {
	const uint32_t threads = p.shape.threads;
	auto kernel = threads > 256 ? (part ? k_norm_backward<T, C, 512, true> : k_norm_backward<T, C, 512, false>)
	                            : (part ? k_norm_backward<T, C, 256, true> : k_norm_backward<T, C, 256, false>);
	kernel<<<p.grid, threads, (64 + (p.shape.G < threads ? 8 * threads : 0)) * sizeof(float), s>>>(a, p.shape.G, part);
	NGP_HIP_CHECK(hipGetLastError());
}

template <class T>
static void norm_backward(const ngp_layer_norm_backward_args& a, hipStream_t s) {
	const NormBackwardPlan p = backward_plan(a);
	float* part = p.sums ? static_cast<float*>(a.workspace) : nullptr;
	if (p.in_pass && (part || (a.dx && a.n))) {
		if (p.shape.chunks == 1) launch_backward<T, 1>(a, p, part, s);
		else launch_backward<T, 2>(a, p, part, s);
	}
	if (!p.in_pass && part) {
		const size_t each = ((size_t)a.n + p.parts - 1) / p.parts;
		k_norm_backward_columns<T><<<dim3((a.width + 511) / 512, p.parts), 256, 0, s>>>(a, each, part);
		NGP_HIP_CHECK(hipGetLastError());
	}
	if (!p.in_pass && a.dx && a.n) {
		k_norm_backward_rows<T><<<std::min(a.n, NORM_GRID), 1024, 0, s>>>(a);
		NGP_HIP_CHECK(hipGetLastError());
	}
	if (part) launch_column_sums(part, p.parts, 2 * a.width, PutSums{a.dgamma, a.dbeta, a.width, a.accumulate != 0}, s);
}

void run_layer_norm_forward(const ngp_layer_norm_args& a, hipStream_t s) {
	if (!a.n) return;
	if (a.type == NGP_TYPE_F32) norm_forward<float>(a, s);
	else if (a.type == NGP_TYPE_F16) norm_forward<f16>(a, s);
	else norm_forward<bf16>(a, s);
}

void run_layer_norm_backward(const ngp_layer_norm_backward_args& a, hipStream_t s) {
	if (a.type == NGP_TYPE_F32) norm_backward<float>(a, s);
	else if (a.type == NGP_TYPE_F16) norm_backward<f16>(a, s);
	else norm_backward<bf16>(a, s);
}

}  // namespace ngp
