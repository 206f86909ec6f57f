// checkpoint8.hip — activations in 8 bits (ngp_checkpoint8): store and load.
#include "layer_math.h"
#include "ngp_internal.h"

namespace ngp {

template <class T>
__global__ void k_checkpoint_store(const T* __restrict__ v, size_t stride, uint32_t n, uint32_t width, ngp_checkpoint8 c) {
	const uint32_t blocks = (width + 31u) / 32u;
	const size_t t = (size_t)blockIdx.x * 256u + threadIdx.x;
	if (t >= (size_t)n * blocks) return;
	const size_t i = t / blocks;
	const uint32_t j0 = (uint32_t)(t % blocks) * 32u, j1 = min(j0 + 32u, width);
	uint32_t top = 0;
	for (uint32_t j = j0; j < j1; ++j) top = max(top, magnitude_bits(widen(v[i * stride + j])));
	const uint32_t scale = checkpoint_scale<T>(top);
	for (uint32_t j = j0; j < j1; ++j) c.q[i * c.q_stride + j] = (int8_t)checkpoint_q(widen(v[i * stride + j]), scale);
	c.scale[i * c.scale_stride + j0 / 32u] = (uint8_t)scale;
}

template <class T>
__global__ void k_checkpoint_load(ngp_checkpoint8 c, uint32_t n, uint32_t width, T* __restrict__ v, size_t stride) {
	const size_t t = (size_t)blockIdx.x * 256u + threadIdx.x;
	if (t >= (size_t)n * width) return;
	const size_t i = t / width;
	const uint32_t j = (uint32_t)(t % width);
	v[i * stride + j] = narrow<T>(checkpoint_value(c.q[i * c.q_stride + j], c.scale[i * c.scale_stride + j / 32u]));
}

template <class T>
static void store(const void* v, uint32_t stride, uint32_t n, uint32_t width, const ngp_checkpoint8& c, hipStream_t s) {
	const size_t items = (size_t)n * ((width + 31u) / 32u);
	k_checkpoint_store<T><<<(uint32_t)((items + 255) / 256), 256, 0, s>>>(static_cast<const T*>(v), stride, n, width, c);
	NGP_HIP_CHECK(hipGetLastError());
}

template <class T>
static void load(const ngp_checkpoint8& c, uint32_t n, uint32_t width, void* v, uint32_t stride, hipStream_t s) {
	const size_t items = (size_t)n * width;
	k_checkpoint_load<T><<<(uint32_t)((items + 255) / 256), 256, 0, s>>>(c, n, width, static_cast<T*>(v), stride);
	NGP_HIP_CHECK(hipGetLastError());
}

void run_checkpoint_store(const void* v, uint32_t stride, uint32_t n, uint32_t width, int type, const ngp_checkpoint8& c,
                          hipStream_t s) {
	if (type == NGP_TYPE_F32) store<float>(v, stride, n, width, c, s);
	else if (type == NGP_TYPE_F16) store<f16>(v, stride, n, width, c, s);
	else store<bf16>(v, stride, n, width, c, s);
}

void run_checkpoint_load(const ngp_checkpoint8& c, uint32_t n, uint32_t width, int type, void* v, uint32_t stride,
                         hipStream_t s) {
	if (type == NGP_TYPE_F32) load<float>(c, n, width, v, stride, s);
	else if (type == NGP_TYPE_F16) load<f16>(c, n, width, v, stride, s);
	else load<bf16>(c, n, width, v, stride, s);
}

}  // namespace ngp
