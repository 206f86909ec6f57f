// linear.hip — linear layers of any width: forward with bias, activation, residual and kept pre-activation; backward.
//
//   forward   z = x W^T + b, y = act(z) + r
//   backward  dz = dy act'(z), dx = (dz W) act_x'(p), dW = dz^T act_x(p), db = sum of dz
#include "layer_math.h"
#include "ngp_internal.h"

namespace ngp {

// What a product C[m][n] does with its fp32 sums.
template <class T>
struct ForwardOut {
	const float* bias;
	int act;
	const T* residual;
	T* y;
	T* z;
	ngp_checkpoint8 z8;
	size_t residual_stride, y_stride, z_stride;
	__device__ __forceinline__ float finish(size_t i, uint32_t j, float z_) const {
		const float v = z_ + (bias ? bias[j] : 0.0f);
		if (z) z[i * z_stride + j] = narrow<T>(v);
		float r = act_value(act, v);
		if (residual) r += widen(residual[i * residual_stride + j]);
		y[i * y_stride + j] = narrow<T>(r);
		return v;
	}
};

template <class T>
struct GradientOut {  // dx
	T* dx;
	size_t stride;
	Kept<T> p;
	int act;
	ngp_checkpoint8 z8;  // unused (null)
	__device__ __forceinline__ float finish(size_t i, uint32_t j, float v) const {
		if (act != NGP_ACT_NONE) v *= act_slope(act, p.at(i, j));
		dx[i * stride + j] = narrow<T>(v);
		return v;
	}
};

template <class T>
struct WeightsOut {  // dW
	void* dw;
	size_t stride;
	int f32, accumulate;
	ngp_checkpoint8 z8;  // unused (null)
	__device__ __forceinline__ float finish(size_t i, uint32_t j, float v) const {
		if (f32) {
			float* d = static_cast<float*>(dw) + i * stride + j;
			*d = accumulate ? *d + v : v;
		} else {
			static_cast<T*>(dw)[i * stride + j] = narrow<T>(v);
		}
		return v;
	}
};

// A product's operand, element by element: kept activations, an activation of them, rounded to T.
template <class T>
struct Operand {
	Kept<T> v;
	int act = NGP_ACT_NONE;
	bool by_k = false;  // [k][row] in memory
	__device__ __forceinline__ float at(size_t row, size_t k) const {
		const float x = by_k ? v.at(k, (uint32_t)row) : v.at(row, (uint32_t)k);
		return act == NGP_ACT_NONE ? x : widen(narrow<T>(act_value(act, x)));
	}
};

constexpr int TILE = 64, TILE_K = 16;

// C[m][n] = sum over k of P[m][k] Q[n][k]: 64 x 64 per workgroup, 4 x 4 per thread, operands through LDS in fp32.
template <class T, class Out>
__global__ void __launch_bounds__(256) k_product(Operand<T> P, Operand<T> Q, size_t M, uint32_t N, size_t K, Out out) {
	__shared__ float sp[TILE_K][TILE + 1], sq[TILE_K][TILE + 1], sz[TILE][TILE + 1];
	const size_t m0 = (size_t)blockIdx.x * TILE;
	const uint32_t n0 = blockIdx.y * TILE;
	const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
	float c[4][4] = {};
	for (size_t k0 = 0; k0 < K; k0 += TILE_K) {
		for (int t = threadIdx.x; t < TILE * TILE_K; t += 256) {
			// neighbouring threads along whichever index is contiguous in memory
			const int pr = P.by_k ? t % TILE : t / TILE_K, pk = P.by_k ? t / TILE : t % TILE_K;
			const int qr = Q.by_k ? t % TILE : t / TILE_K, qk = Q.by_k ? t / TILE : t % TILE_K;
			sp[pk][pr] = m0 + pr < M && k0 + pk < K ? P.at(m0 + pr, k0 + pk) : 0.0f;
			sq[qk][qr] = n0 + qr < N && k0 + qk < K ? Q.at(n0 + qr, k0 + qk) : 0.0f;
		}
		__syncthreads();
		for (int k = 0; k < TILE_K; ++k)
			for (int a = 0; a < 4; ++a)
				for (int b = 0; b < 4; ++b) c[a][b] = __builtin_fmaf(sp[k][tm * 4 + a], sq[k][tn * 4 + b], c[a][b]);
		__syncthreads();
	}
	for (int a = 0; a < 4; ++a)
		for (int b = 0; b < 4; ++b) {
			const size_t i = m0 + tm * 4 + a;
			const uint32_t j = n0 + tn * 4 + b;
			sz[tm * 4 + a][tn * 4 + b] = i < M && j < N ? out.finish(i, j, c[a][b]) : 0.0f;
		}
	if (!out.z8.q) return;
	__syncthreads();
	if (threadIdx.x >= TILE * 2) return;
	const size_t i = m0 + threadIdx.x / 2;
	const uint32_t h = threadIdx.x % 2 * 32, j0 = n0 + h;
	if (i >= M || j0 >= N) return;
	const float* row = sz[threadIdx.x / 2] + h;
	uint32_t top = 0;
	for (int j = 0; j < 32; ++j) top = max(top, magnitude_bits(row[j]));
	const uint32_t scale = checkpoint_scale<T>(top);
	for (uint32_t j = 0; j < 32 && j0 + j < N; ++j) out.z8.q[i * out.z8.q_stride + j0 + j] = (int8_t)checkpoint_q(row[j], scale);
	out.z8.scale[i * out.z8.scale_stride + j0 / 32] = (uint8_t)scale;
}

// dz = dy act'(z) and its sums over a share of the rows: 64 columns x rows_each rows per workgroup.
template <class T>
__global__ void __launch_bounds__(256) k_linear_dz(const T* __restrict__ dy, size_t dy_stride, Kept<T> z, int act, uint32_t n,
                                                   uint32_t width, uint32_t rows_each, T* dz, float* part) {
	const uint32_t j = blockIdx.x * 64u + (threadIdx.x & 63u), w = threadIdx.x >> 6;
	const size_t begin = (size_t)blockIdx.y * rows_each, end = min(begin + rows_each, (size_t)n);
	float sum = 0.0f;
	if (j < width)
		for (size_t i = begin + w; i < end; i += 4) {
			float d = widen(dy[i * dy_stride + j]);
			if (act != NGP_ACT_NONE) d *= act_slope(act, z.at(i, j));
			if (dz) dz[i * width + j] = narrow<T>(d);
			sum += d;
		}
	__shared__ float s[256];
	s[threadIdx.x] = sum;
	__syncthreads();
	const uint32_t t = threadIdx.x;
	if (part && w == 0 && j < width) part[(size_t)blockIdx.y * width + j] = (s[t] + s[t + 64]) + (s[t + 128] + s[t + 192]);
}

__global__ void k_column_sum(const float* __restrict__ part, uint32_t shares, uint32_t width, float* out, int accumulate) {
	const uint32_t j = blockIdx.x * 256u + threadIdx.x;
	if (j >= width) return;
	float s = 0.0f;
	for (uint32_t k = 0; k < shares; ++k) s += part[(size_t)k * width + j];
	out[j] = accumulate ? out[j] + s : s;
}

size_t linear_workspace(const ngp_linear_args&) { return 0; }

static size_t up16(size_t b) { return (b + 15) & ~(size_t)15; }
static uint32_t row_shares(uint32_t n) { return std::max(1u, std::min(256u, n / 64u)); }

struct LinearBackwardPlan {
	size_t dz = 0, part = 0, bytes = 0;  // offsets in the workspace
};

static LinearBackwardPlan plan(const ngp_linear_backward_args& a) {
	LinearBackwardPlan p;
	if (a.activation != NGP_ACT_NONE) p.bytes += up16((size_t)a.n * a.n_out * 2);
	p.part = p.bytes;
	if (a.dbias) p.bytes += up16((size_t)row_shares(a.n) * a.n_out * 4);
	return p;
}

size_t linear_backward_workspace(const ngp_linear_backward_args& a) { return plan(a).bytes; }

template <class T>
static void linear_forward(const ngp_linear_args& a, hipStream_t s) {
	if (!a.n) return;
	const Operand<T> x{Kept<T>{static_cast<const T*>(a.x), a.x_stride}}, w{Kept<T>{static_cast<const T*>(a.weights), a.weights_stride}};
	const ForwardOut<T> out{a.bias, a.activation, static_cast<const T*>(a.residual), static_cast<T*>(a.y), static_cast<T*>(a.z),
	                        a.z8, a.residual_stride, a.y_stride, a.z_stride};
	k_product<T><<<dim3((a.n + TILE - 1) / TILE, (a.n_out + TILE - 1) / TILE), 256, 0, s>>>(x, w, a.n, a.n_out, a.n_in, out);
	NGP_HIP_CHECK(hipGetLastError());
}

template <class T>
static void linear_backward(const ngp_linear_backward_args& a, hipStream_t s) {
	const LinearBackwardPlan p = plan(a);
	char* ws = static_cast<char*>(a.workspace);
	const bool own = a.activation != NGP_ACT_NONE;
	T* dz_ws = reinterpret_cast<T*>(ws + p.dz);
	Operand<T> dz{own ? Kept<T>{dz_ws, a.n_out} : Kept<T>{static_cast<const T*>(a.dy), a.dy_stride}};
	if (own || a.dbias) {
		const uint32_t shares = row_shares(a.n), each = (a.n + shares - 1) / shares;
		float* part = a.dbias ? reinterpret_cast<float*>(ws + p.part) : nullptr;
		k_linear_dz<T><<<dim3((a.n_out + 63) / 64, shares), 256, 0, s>>>(
		    static_cast<const T*>(a.dy), a.dy_stride, kept<T>(a.z, a.z_stride, a.z8), a.activation, a.n, a.n_out, each,
		    own ? dz_ws : nullptr, part);
		NGP_HIP_CHECK(hipGetLastError());
		if (a.dbias) {
			k_column_sum<<<(a.n_out + 255) / 256, 256, 0, s>>>(part, shares, a.n_out, a.dbias, a.accumulate);
			NGP_HIP_CHECK(hipGetLastError());
		}
	}
	const Kept<T> x = kept<T>(a.x, a.x_stride, a.x8);
	if (a.dx && a.n) {
		Operand<T> w{Kept<T>{static_cast<const T*>(a.weights), a.weights_stride}};
		w.by_k = true;
		const GradientOut<T> out{static_cast<T*>(a.dx), a.dx_stride, x, a.x_activation, {}};
		k_product<T><<<dim3((a.n + TILE - 1) / TILE, (a.n_in + TILE - 1) / TILE), 256, 0, s>>>(dz, w, a.n, a.n_in, a.n_out, out);
		NGP_HIP_CHECK(hipGetLastError());
	}
	if (a.dweights) {
		dz.by_k = true;
		Operand<T> xs{x, a.x_activation, true};
		const WeightsOut<T> out{a.dweights, a.dweights_stride, a.dweights_type == NGP_TYPE_F32, a.accumulate, {}};
		k_product<T><<<dim3((a.n_out + TILE - 1) / TILE, (a.n_in + TILE - 1) / TILE), 256, 0, s>>>(dz, xs, a.n_out, a.n_in, a.n, out);
		NGP_HIP_CHECK(hipGetLastError());
	}
}

void run_linear_forward(const ngp_linear_args& a, hipStream_t s) {
	if (a.type == NGP_TYPE_F16) linear_forward<f16>(a, s);
	else linear_forward<bf16>(a, s);
}

void run_linear_backward(const ngp_linear_backward_args& a, hipStream_t s) {
	if (a.type == NGP_TYPE_F16) linear_backward<f16>(a, s);
	else linear_backward<bf16>(a, s);
}

}  // namespace ngp
