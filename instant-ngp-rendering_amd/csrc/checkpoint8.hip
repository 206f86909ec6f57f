// checkpoint8.hip — activations in 8 bits (ngp_checkpoint8): store and load.
//
// Nothing is computed to speak of: both move s + 33/32 bytes per value (s the type's size).  A thread takes eight
// neighbouring values, the four lanes of a quad a block, so that the block's largest magnitude stays in the quad and every
// access is wide: 16 bytes of 16-bit values, 8 bytes of q.
#include <algorithm>

#include "layer_math.h"
#include "ngp_internal.h"

namespace ngp {

// Four items per block of 32, of which the last ones of a row may have nothing to do; a quad leaves the loop together.
template <class T>
__global__ void __launch_bounds__(256) k_checkpoint_store(Kept<T> v, size_t n, uint32_t width, ngp_checkpoint8 c) {
	for (Walk w((width + 31u) / 32u * 4u); w.i < n; w.next()) {
		const uint32_t j = w.e * 8u, left = j < width ? width - j : 0u;
		float x[8] = {};
		if (left) v.at8(w.i, j, left, x);
		uint32_t top = 0;
#pragma unroll
		for (int k = 0; k < 8; ++k) top = max(top, magnitude_bits(x[k]));
		const uint32_t scale = checkpoint_scale<T>(quad_max(top));
		if (left) checkpoint_store8(c.q + w.i * c.q_stride + j, left, scale, x);
		if (j % 32u == 0) c.scale[w.i * c.scale_stride + j / 32u] = (uint8_t)scale;
	}
}

template <class T>
__global__ void __launch_bounds__(256) k_checkpoint_load(Kept<T> c, size_t n, uint32_t width, T* __restrict__ v, size_t v_stride) {
	for (Walk w((width + 7u) / 8u); w.i < n; w.next()) {
		const uint32_t j = w.e * 8u;
		float x[8];
		c.at8(w.i, j, width - j, x);
		store8(v + w.i * v_stride + j, width - j, x);
	}
}

// 16384 workgroups are eight rounds of the 256 CUs' eight workgroups; most sizes then leave a thread a few items
static uint32_t grid_of(size_t items) { return (uint32_t)std::min<size_t>((items + 255) / 256, 16384); }

template <class T>
static void store(const void* v, uint32_t stride, uint32_t n, uint32_t width, const ngp_checkpoint8& c, hipStream_t s) {
	const uint32_t grid = grid_of((size_t)n * ((width + 31u) / 32u * 4u));
	k_checkpoint_store<T><<<grid, 256, 0, s>>>(kept<T>(v, stride, {}), n, width, c);
	NGP_HIP_CHECK(hipGetLastError());
}

template <class T>
static void load(const ngp_checkpoint8& c, uint32_t n, uint32_t width, void* v, uint32_t stride, hipStream_t s) {
	const uint32_t grid = grid_of((size_t)n * ((width + 7u) / 8u));
	k_checkpoint_load<T><<<grid, 256, 0, s>>>(kept<T>(nullptr, 0, c), n, width, static_cast<T*>(v), stride);
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
