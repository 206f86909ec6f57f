// linear.hip — linear layers of any width: forward with bias, activation, residual and kept pre-activation; backward.
//
//   forward   z = x W^T + b, y = act(z) + r
//   backward  dz = dy act'(z), dx = (dz W) act_x'(p), dW = dz^T act_x(p), db = sum of dz
//
// Three products C[m][n] = sum over k of P[m][k] Q[n][k], one kernel (k_product):
//   y:  P = x  [row][k],  Q = W  [row][k]
//   dx: P = dz [row][k],  Q = W  [k][row]  (k runs over the outputs)
//   dW: P = dz [k][row],  Q = x  [k][row]  (k runs over the samples)
#include <algorithm>

#include "layer_math.h"
#include "ngp_internal.h"

namespace ngp {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr;

__device__ __forceinline__ f32x16 mfma(f16, s16x8 a, s16x8 b, f32x16 c) {
	return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8<f16>, a), __builtin_bit_cast(v8<f16>, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(bf16, s16x8 a, s16x8 b, f32x16 c) {
	return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8<bf16>, a), __builtin_bit_cast(v8<bf16>, b), c, 0, 0, 0);
}

// Half h of a 32 x 32 tile's columns: register r holds column r % 4 + 8 (r / 4) + 4 (lane / 32) of row lane % 32; groups of
// four columns change places between the half waves, which leaves a lane the eight at 16 h + 8 (lane / 32).
__device__ __forceinline__ void eight(const f32x16& c, int h, float (&v)[8]) {
#pragma unroll
	for (int k = 0; k < 4; ++k) {
		const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(c[8 * h + k]), __float_as_uint(c[8 * h + 4 + k]), false, false);
		v[k] = __uint_as_float(s[0]);
		v[k + 4] = __uint_as_float(s[1]);
	}
}

// ---- what a product does with its fp32 sums, eight neighbouring columns of a row at a time --------------------------
// Columns: what the rows share; Fetched: what is read for a row's eight, asked for before any of them is finished, by a
// `fetch` for each kind of source (by_kind), so that no branch stands among the loads and they wait for nothing.
template <int K>
using Kind = std::integral_constant<int, K>;
template <class T>
struct ForwardOut {
	const float* bias;
	const T* residual;
	T* y;
	T* z;
	ngp_checkpoint8 z8;
	size_t residual_stride, y_stride, z_stride;
	int act;
	struct Columns {
		float bias[8];
	};
	typedef v8<T> Fetched;
	__device__ __forceinline__ Columns columns(uint32_t j, uint32_t left) const {
		Columns c;
#pragma unroll
		for (int k = 0; k < 8; ++k) c.bias[k] = bias && (uint32_t)k < left ? bias[j + k] : 0.0f;
		return c;
	}
	template <class F>
	__device__ __forceinline__ void by_kind(F f) const { residual ? f(Kind<1>{}) : f(Kind<0>{}); }
	template <int K>
	__device__ __forceinline__ Fetched fetch(Kind<K>, size_t i, uint32_t j, uint32_t left) const {
		if constexpr (K == 1) return load8_raw(residual + i * residual_stride + j, left);
		else return {};
	}
	__device__ __forceinline__ void finish(size_t i, uint32_t j, uint32_t left, const Columns& c, const Fetched& f, float (&v)[8],
	                                       float (&kept)[8]) const {
#pragma unroll
		for (int k = 0; k < 8; ++k) kept[k] = v[k] += c.bias[k];
		if (z) store8(z + i * z_stride + j, left, v);
		act_values(act, v);
		if (residual) {
#pragma unroll
			for (int k = 0; k < 8; ++k) v[k] += widen(f[k]);
		}
		store8(y + i * y_stride + j, left, v);
	}
};

template <class T>
struct GradientOut {  // dx
	T* dx;
	size_t stride;
	Kept<T> p;
	int act;
	static constexpr ngp_checkpoint8 z8 = {};
	struct Columns {};
	typedef typename Kept<T>::Raw Fetched;
	__device__ __forceinline__ Columns columns(uint32_t, uint32_t) const { return {}; }
	template <class F>
	__device__ __forceinline__ void by_kind(F f) const { act == NGP_ACT_NONE ? f(Kind<0>{}) : p.v ? f(Kind<1>{}) : f(Kind<2>{}); }
	template <int K>
	__device__ __forceinline__ Fetched fetch(Kind<K>, size_t i, uint32_t j, uint32_t left) const {
		if constexpr (K == 1) return p.raw8_values(i, j, left);
		else if constexpr (K == 2) return p.raw8_checkpoint(i, j, left);
		else return {};
	}
	__device__ __forceinline__ void finish(size_t i, uint32_t j, uint32_t left, const Columns&, const Fetched& f, float (&v)[8],
	                                       float (&)[8]) const {
		if (act != NGP_ACT_NONE) {
			float s[8];
			p.widen8(f, s);
			act_slopes(act, s);
#pragma unroll
			for (int k = 0; k < 8; ++k) v[k] *= s[k];
		}
		store8(dx + i * stride + j, left, v);
	}
};

template <class T>
struct WeightsOut {  // dW
	void* dw;
	size_t stride;
	bool f32, accumulate;
	static constexpr ngp_checkpoint8 z8 = {};
	struct Columns {};
	struct Fetched {
		float before[8];
	};
	__device__ __forceinline__ Columns columns(uint32_t, uint32_t) const { return {}; }
	template <class F>
	__device__ __forceinline__ void by_kind(F f) const { accumulate ? f(Kind<1>{}) : f(Kind<0>{}); }
	template <int K>
	__device__ __forceinline__ Fetched fetch(Kind<K>, size_t i, uint32_t j, uint32_t left) const {
		Fetched f = {};
		if constexpr (K == 1) load8(static_cast<const float*>(dw) + i * stride + j, left, f.before);
		return f;
	}
	__device__ __forceinline__ void finish(size_t i, uint32_t j, uint32_t left, const Columns&, const Fetched& f, float (&v)[8],
	                                       float (&)[8]) const {
		if (f32) {
#pragma unroll
			for (int k = 0; k < 8; ++k) v[k] += f.before[k];
			store8(static_cast<float*>(dw) + i * stride + j, left, v);
		} else {
			store8(static_cast<T*>(dw) + i * stride + j, left, v);
		}
	}
};

// ---- the product ------------------------------------------------------------------------------------------------------
// An operand whose rows start on 16 bytes and are multiples of 8 elements long.
struct Matrix {
	const void* v;
	size_t stride;
};

struct ProductArgs {
	Matrix p, q;
	size_t M, K, k_each;  // k_each: how much of K a split takes, a multiple of PRODUCT_K
	uint32_t N, tiles_m, tiles_n, splits;
	float* partial;       // [splits][M][N up to 8] where splits > 1
};

constexpr int PRODUCT_K = 64;  // splits of K are multiples of it
constexpr int PRODUCT_THREADS = 256, WIDE_THREADS = 512;

// One stage of an operand in LDS: ROWS x DEEP (64 or 32) elements of 16 bits.  Each wave's load puts 64 chunks of 16 bytes
// one after another (buffer_load ... lds takes no other order), so rows are spread over the banks by what each lane fetches:
//  * [row][k] in memory: 2 DEEP bytes per row, chunk c of row r holds k chunk c ^ twist(r); ds_read_b128 of 32 rows' same
//    k chunk touches every bank equally.
//  * [k][row] in memory: 2 ROWS bytes per k, chunk c of line k holds rows' chunk c ^ twist(k); ds_read_b64_tr_b16 reads
//    four k lines x 64 bytes per half wave, which the twist puts on different banks.
template <class T, int ROWS, bool BY_K, int DEEP, int THREADS>
struct Stage {
	static constexpr int BYTES = ROWS * DEEP * 2;
	static constexpr int LOADS = BYTES / 16 / THREADS;
	static constexpr int LINE = BY_K ? ROWS * 2 : DEEP * 2;  // bytes
	static constexpr uint32_t OUTSIDE = 0xfffffff0u;         // past every buffer: the load gives zeros
	static_assert(BYTES % (16 * THREADS) == 0, "every thread loads the same number of chunks");
	__device__ static __forceinline__ uint32_t twist(uint32_t line) {
		if constexpr (!BY_K) return LINE >= 128 ? (line >> 1) & 7u : (line >> 2) & 3u;
		return LINE >= 256 ? ((line & 3u) << 2) | (line & 2u) : (((line >> 1) & 1u) << 2) | ((line & 1u) << 1);
	}

	const char* base;       // of the stage's first element (uniform)
	size_t step;            // bytes to the next stage
	uint32_t offset[LOADS]; // a thread's chunks
	__device__ static __forceinline__ uint32_t k_of(int l) {  // and their first k in the stage
		const uint32_t c = threadIdx.x + l * THREADS, line = c / (LINE / 16), at = c % (LINE / 16);
		return BY_K ? line : (at ^ twist(line)) * 8u;
	}

	size_t lines;           // [k][row]: lines of k that are left from `base` on
	uint32_t line_bytes;

	// rows [row0, rows) of the matrix, k from k0 to K
	__device__ __forceinline__ void begin(const Matrix& m, size_t row0, size_t rows, size_t k0, size_t K) {
		lines = K - k0;
		line_bytes = (uint32_t)m.stride * 2u;
		const uint32_t left = (uint32_t)min(rows - row0, (size_t)ROWS);
		base = static_cast<const char*>(m.v) + (BY_K ? k0 * m.stride + row0 : row0 * m.stride + k0) * 2;
		step = BY_K ? m.stride * (DEEP * 2) : DEEP * 2;
#pragma unroll
		for (int l = 0; l < LOADS; ++l) {
			const uint32_t c = threadIdx.x + l * THREADS, line = c / (LINE / 16), at = c % (LINE / 16);
			const uint32_t row = BY_K ? (at ^ twist(line)) * 8u : line;
			offset[l] = row < left ? (BY_K ? line * (uint32_t)m.stride + row : row * (uint32_t)m.stride + k_of(l)) * 2u : OUTSIDE;
		}
	}
	// The first stage, of which k below `k_in` is there (the rest is zeros), then the others, which are whole but for lines
	// past K.  Nothing is read without `more`.
	__device__ __forceinline__ void load_first(char* lds, uint32_t k_in) {
		uint32_t at[LOADS];
#pragma unroll
		for (int l = 0; l < LOADS; ++l) at[l] = k_of(l) < k_in ? offset[l] : OUTSIDE;
		issue(lds, at, true);
		base += (BY_K ? step / DEEP : 2) * k_in;
		lines -= min((size_t)k_in, lines);
	}
	__device__ __forceinline__ void load(char* lds, bool more) {
		issue(lds, offset, more);
		base += step;
		lines -= min((size_t)DEEP, lines);
	}
	__device__ __forceinline__ void issue(char* lds, const uint32_t (&at)[LOADS], bool more) {
		// the buffer's end, past which a load gives zeros: after the last line of k, or nowhere
		const uint32_t end = !more ? 0u : (BY_K ? (uint32_t)min((size_t)DEEP, lines) * line_bytes : 0x7fffffffu);
		const uintptr_t from = reinterpret_cast<uintptr_t>(base);
		const i32x4 rsrc = {(int)(uint32_t)from, (int)(uint32_t)(from >> 32), (int)end, 0x00027000};
		const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>((lds_ptr)lds) + (threadIdx.x & ~63u) * 16u);
		// not the builtin: the compiler then waits for every load into LDS before each transposed read from it, whichever
		// buffer they are for.  The waits are written out where the stages change; nothing is loaded into registers here.  The
		// block says what it writes, m0 (the LDS address) and memory, so that no access to LDS or memory moves over it.
#pragma unroll
		for (int l = 0; l < LOADS; ++l)
			asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
			             :
			             : "s"(to + l * THREADS * 16), "v"(at[l]), "s"(rsrc)
			             : "m0", "memory");
	}
};

// A wave's 32 x 16 fragments of a stage: lane l holds row l % 32 and k = 8 (l / 32) .. + 7 of each 16.
template <class Stage, int ROWS, bool BY_K, int DEEP, int TILES>
struct Fragments {
	uint32_t offset[BY_K ? TILES : DEEP / 16];
	__device__ __forceinline__ void begin(uint32_t row0) {
		const uint32_t lane = threadIdx.x & 63u;
		if constexpr (BY_K) {
			// 16 lanes read 4 k lines x 16 rows and get them transposed: lane j of them row j's four k
			const uint32_t g = lane >> 4, q = (lane & 15u) >> 2, p = lane & 3u;
#pragma unroll
			for (int t = 0; t < TILES; ++t) {
				const uint32_t chunk = (row0 + t * 32u + 16u * (g & 1u)) / 8u + (p >> 1);
				offset[t] = (8u * (g >> 1) + q) * (ROWS * 2) + ((chunk ^ Stage::twist(q)) << 4) + (p & 1u) * 8u;
			}
		} else {
#pragma unroll
			for (int s = 0; s < DEEP / 16; ++s)
				offset[s] = (row0 + (lane & 31u)) * (DEEP * 2) + (((s * 2u + (lane >> 5)) ^ Stage::twist(lane & 31u)) << 4);
		}
	}
	__device__ __forceinline__ s16x8 read(const char* lds, int s, int t) const {  // the s-th 16 of k, the t-th 32 rows
		if constexpr (BY_K) {
			typedef __attribute__((address_space(3))) s16x4* tr_ptr;
			const char* at = lds + offset[t] + s * 16 * (ROWS * 2);
			const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)at);
			const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 4 * (ROWS * 2)));
			return s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
		} else {
			return *reinterpret_cast<const s16x8*>(lds + offset[s] + t * 32 * (DEEP * 2));
		}
	}
};

// Eight neighbouring columns of C (j a multiple of 8, `left` of them and more up to the row's end; 0: none) to the caller's
// matrices.  The four lanes of a block of 32 call it together.
template <class T, class Out>
__device__ __forceinline__ void finish_block(const Out& out, size_t i, uint32_t j, uint32_t left, const typename Out::Columns& columns,
                                             const typename Out::Fetched& fetched, float (&v)[8]) {
	float z[8] = {};
	if (left) out.finish(i, j, left, columns, fetched, v, z);
	if (!out.z8.q) return;
	uint32_t top = 0;
#pragma unroll
	for (int k = 0; k < 8; ++k) top = max(top, magnitude_bits(z[k]));  // past the row's end: 0 (Q's rows are), or as the row
	top = quad_max(top);
	if (!left) return;
	const uint32_t scale = checkpoint_scale<T>(top);
	checkpoint_store8(out.z8.q + i * out.z8.q_stride + j, left, scale, z);
	if (j % 32u == 0) out.z8.scale[i * out.z8.scale_stride + j / 32u] = (uint8_t)scale;
}

// Where a workgroup works.  Workgroups go to the eight XCDs in turn: each XCD gets a run of neighbouring tiles, eight tile
// rows deep, so that its L2 holds what they share.
template <int TILE>
struct Place {
	uint32_t split, n0;
	size_t m0, k0, k1;
	__device__ __forceinline__ Place(const ProductArgs& a, uint32_t block, uint32_t blocks) {
		const uint32_t tiles = a.tiles_m * a.tiles_n, xcd = block % 8u;
		const uint32_t id = xcd * (blocks / 8u) + min(xcd, blocks % 8u) + block / 8u;
		split = id / tiles;
		const uint32_t tile = id % tiles, group = tile / (8u * a.tiles_n), first = group * 8u, deep = min(8u, a.tiles_m - first);
		const uint32_t in_group = tile - group * 8u * a.tiles_n;
		m0 = (size_t)(first + in_group % deep) * TILE;
		n0 = in_group / deep * TILE;
		// rows along k are filled up to 8 with zeros; lines past K are not there, which the loads know
		k0 = split * a.k_each;
		k1 = min(k0 + a.k_each, (a.K + 7u) & ~(size_t)7u);
	}
};

// A wave's TN x TM tiles of 32 x 32 sums, at row i0 and column j0 of C, to where they belong.  Register r of a tile holds
// column r % 4 + 8 (r / 4) + 4 (lane / 32) of row lane % 32.  The wave passes 32 rows at a time through its strip of LDS and
// takes them out again row by row, eight neighbouring columns per lane: whole lines of the caller's matrices per access, and
// one copy of the code that finishes a value.
template <int TN>
constexpr int STRIP = 32 * (TN * 32 + 4);  // floats; + 4: 32 rows' 16-byte pieces on different banks
// What the caller's matrices hold for a strip is asked for a strip ahead, for the first one before K is gone through.
template <class T, class Out, int TM, int TN>
struct WriteOut {
	static constexpr int PITCH = TN * 32 + 4, LANES = TN * 4, ROWS = 64 / LANES, TURNS = 32 / ROWS;
	const ProductArgs& a;
	const Out& out;
	size_t i0;      // the lane's first row,
	uint32_t j;     // its columns,
	uint32_t left;  // how many there are
	bool whole;     // the wave's tiles lie inside C: nothing is looked at again
	typename Out::Fetched ahead[TURNS];

	__device__ __forceinline__ WriteOut(const ProductArgs& a, const Out& out, size_t i, uint32_t j0) : a(a), out(out) {
		const uint32_t lane = threadIdx.x & 63u;
		i0 = i + lane / LANES;
		j = j0 + lane % LANES * 8u;
		left = j < a.N ? a.N - j : 0u;
		whole = i + TM * 32u <= a.M && j0 + TN * 32u <= a.N;
#pragma unroll
		for (int u = 0; u < TURNS; ++u) ahead[u] = {};
		if (a.splits == 1) whole ? fetch<true>(0) : fetch<false>(0);
	}
	template <bool WHOLE>
	__device__ __forceinline__ uint32_t here(int m, int u) const {
		return WHOLE ? 8u : i0 + m * 32u + u * ROWS < a.M ? left : 0u;
	}
	template <bool WHOLE>
	__device__ __forceinline__ void fetch(int m) {
		out.by_kind([&](auto kind) {
#pragma unroll
			for (int u = 0; u < TURNS; ++u)
				if (here<WHOLE>(m, u)) ahead[u] = out.fetch(kind, i0 + m * 32u + u * ROWS, j, here<WHOLE>(m, u));
		});
	}
	template <bool WHOLE, bool JOIN>
	__device__ __forceinline__ void write(uint32_t split, float* strip, const f32x16 (&c)[TN][TM]) {
		const uint32_t lane = threadIdx.x & 63u, n8 = (a.N + 7u) & ~7u;
		typename Out::Columns columns;
		if constexpr (!JOIN) columns = out.columns(j, WHOLE ? 8u : left);
#pragma unroll
		for (int m = 0; m < TM; ++m) {
			typename Out::Fetched fetched[TURNS];
#pragma unroll
			for (int u = 0; u < TURNS; ++u) fetched[u] = ahead[u];
			if constexpr (!JOIN)
				if (m + 1 < TM) fetch<WHOLE>(m + 1);
#pragma unroll
			for (int n = 0; n < TN; ++n)
#pragma unroll
				for (int g = 0; g < 4; ++g)
					*reinterpret_cast<f32x4*>(strip + (lane & 31u) * PITCH + n * 32 + g * 8 + (lane >> 5) * 4u) =
					    f32x4{c[n][m][4 * g], c[n][m][4 * g + 1], c[n][m][4 * g + 2], c[n][m][4 * g + 3]};
			__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
			for (int u = 0; u < TURNS; ++u) {
				const float* row = strip + (lane / LANES + u * ROWS) * PITCH + lane % LANES * 8u;
				const f32x4 lo = *reinterpret_cast<const f32x4*>(row), hi = *reinterpret_cast<const f32x4*>(row + 4);
				float v[8];
#pragma unroll
				for (int k = 0; k < 8; ++k) v[k] = k < 4 ? lo[k & 3] : hi[k & 3];
				const size_t i = i0 + m * 32u + u * ROWS;
				if constexpr (!JOIN) finish_block<T>(out, i, j, here<WHOLE>(m, u), columns, fetched[u], v);
				else if (here<WHOLE>(m, u)) store8(a.partial + ((size_t)split * a.M + i) * n8 + j, 8, v);
			}
			__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		}
	}
	__device__ __forceinline__ void operator()(uint32_t split, float* strip, const f32x16 (&c)[TN][TM]) {
		if (a.splits > 1) write<false, true>(split, strip, c);
		else if (whole) write<true, false>(split, strip, c);
		else write<false, false>(split, strip, c);
	}
};

// s_waitcnt's operand: vmcnt and lgkmcnt (15: any), expcnt any.
constexpr int waits(int vmcnt, int lgkmcnt) { return (vmcnt & 15) | 7 << 4 | lgkmcnt << 8 | (vmcnt >> 4) << 14; }
// Nothing moves over this point, in the compiler or among the waves.
__device__ __forceinline__ void meet() {
	asm volatile("" ::: "memory");
	__builtin_amdgcn_sched_barrier(0);
	__builtin_amdgcn_s_barrier();
	__builtin_amdgcn_sched_barrier(0);
	asm volatile("" ::: "memory");
}

// TILE x TILE of C per workgroup of four waves, two by two; K in stages of 64 through BUFFERS LDS buffers: while the matrix cores
// work on one stage, the others are on their way from memory into LDS without passing registers.  P's rows are the matrix
// instruction's columns and Q's its rows, so that a lane ends up with neighbouring columns of C.
template <class T, class Out, bool P_BY_K, bool Q_BY_K, int TILE, int BUFFERS>
__device__ __forceinline__ void product_tile(const ProductArgs& a, const Out& out, uint32_t block, uint32_t blocks, char* lds) {
	constexpr int DEEP = PRODUCT_K, TM = TILE / 64, TN = TILE / 64;  // 32 x 32 tiles per wave
	typedef Stage<T, TILE, P_BY_K, DEEP, PRODUCT_THREADS> PStage;
	typedef Stage<T, TILE, Q_BY_K, DEEP, PRODUCT_THREADS> QStage;
	constexpr int STAGE = PStage::BYTES + QStage::BYTES, LOADS = PStage::LOADS + QStage::LOADS;
	static_assert(4 * STRIP<TN> * 4 <= BUFFERS * STAGE, "the stages' LDS holds the strips");

	const Place<TILE> at(a, block, blocks);
	const uint32_t wave = threadIdx.x / 64u;
	const uint32_t wm = wave / 2u * (TILE / 2), wn = wave % 2u * (TILE / 2);
	const uint32_t stages = (uint32_t)((at.k1 - at.k0 + DEEP - 1) / DEEP);

	WriteOut<T, Out, TM, TN> write_out(a, out, at.m0 + wm, at.n0 + wn);
	f32x16 c[TN][TM] = {};
	if (stages) {
		PStage ps;
		QStage qs;
		Fragments<PStage, TILE, P_BY_K, DEEP, TM> pf;
		Fragments<QStage, TILE, Q_BY_K, DEEP, TN> qf;
		ps.begin(a.p, at.m0, a.M, at.k0, a.K);
		qs.begin(a.q, at.n0, a.N, at.k0, a.K);
		pf.begin(wm);
		qf.begin(wn);
		uint32_t to = 0, now = 0;
		auto next = [](uint32_t at) { return at == (BUFFERS - 1) * STAGE ? 0u : at + STAGE; };
		auto load = [&](bool more) {
			ps.load(lds + to, more);
			qs.load(lds + to + PStage::BYTES, more);
			to = next(to);
		};
		// the part of K that fills no stage comes first, so that the loop has whole stages only
		const uint32_t k_in = (uint32_t)((at.k1 - at.k0 - 1) % DEEP) + 1u;
		ps.load_first(lds, k_in);
		qs.load_first(lds + PStage::BYTES, k_in);
		to = next(to);
#pragma unroll
		for (uint32_t s = 1; s < BUFFERS - 1; ++s) load(s < stages);
		for (uint32_t s = 0; s < stages; ++s, now = next(now)) {
			// stage s has arrived, as far as this wave asked for it, and its reads of stage s - 1 are done; then everybody's
			__builtin_amdgcn_s_waitcnt(waits((BUFFERS - 2) * LOADS, 0));
			meet();
			load(s + BUFFERS - 1 < stages);
			s16x8 p[2][TM], q[2][TN];
			auto read = [&](int k) {
#pragma unroll
				for (int t = 0; t < TN; ++t) q[k & 1][t] = qf.read(lds + now + PStage::BYTES, k, t);
#pragma unroll
				for (int t = 0; t < TM; ++t) p[k & 1][t] = pf.read(lds + now, k, t);
			};
			read(0);
#pragma unroll
			for (int k = 0; k < DEEP / 16; ++k) {
				if (k < DEEP / 16 - 1) read(k + 1);
#pragma unroll
				for (int n = 0; n < TN; ++n)
#pragma unroll
					for (int m = 0; m < TM; ++m) c[n][m] = mfma(T{}, q[k & 1][n], p[k & 1][m], c[n][m]);
			}
		}
		__builtin_amdgcn_s_waitcnt(0);
	}
	__syncthreads();  // the last stage has been read
	write_out(at.split, reinterpret_cast<float*>(lds) + wave * STRIP<TN>, c);
}

template <class T, class Out, bool P_BY_K, bool Q_BY_K, int TILE, int BUFFERS>
__global__ void __launch_bounds__(PRODUCT_THREADS, 2) k_product(ProductArgs a, Out out) {
	extern __shared__ __attribute__((aligned(16))) char lds[];
	product_tile<T, Out, P_BY_K, Q_BY_K, TILE, BUFFERS>(a, out, blockIdx.x, gridDim.x, lds);
}

// A layer's dx and dW, and the join of db's shares, side by side in one launch: none of them fills the GPU in layers whose
// products take the smaller tiles, and none waits for another.
struct Sums {
	const float* part;
	uint32_t shares, columns;
	PutSums put;
};
template <class T, int TILE, int BUFFERS>
__global__ void __launch_bounds__(PRODUCT_THREADS, 2) k_backward_products(ProductArgs dx, GradientOut<T> dx_out, uint32_t dx_blocks, ProductArgs dw,
                                                                          WeightsOut<T> dw_out, uint32_t dw_blocks, Sums sums) {
	extern __shared__ __attribute__((aligned(16))) char lds[];
	if (blockIdx.x < dw_blocks)  // first, as K is the rows: the longest to take
		product_tile<T, WeightsOut<T>, true, true, TILE, BUFFERS>(dw, dw_out, blockIdx.x, dw_blocks, lds);
	else if (blockIdx.x - dw_blocks < dx_blocks)
		product_tile<T, GradientOut<T>, false, true, TILE, BUFFERS>(dx, dx_out, blockIdx.x - dw_blocks, dx_blocks, lds);
	else
		column_sums<PRODUCT_THREADS>(sums.part, sums.shares, sums.columns, sums.put, blockIdx.x - dx_blocks - dw_blocks);
}

// 256 x 256 of C per workgroup of eight waves, two by four, two waves to a SIMD: while the one of them multiplies, the other
// reads its next fragments and asks for a stage of K ahead, and then they change places.  A barrier after each half keeps
// the two sets of four waves in opposite phases.  K goes through 128 KiB of LDS in stages of DEEP, each multiplied in steps
// of 32: two buffers of 64 or four of 32.  Measured over 16384 rows of 2048 x 8192 (0.55 TFLOP, bf16; by card): dW
// 435..465 us (1.2 PFLOP/s, the matrix cores busy for 72 % of the CUs' busy cycles), y 575..615 and dx 570..625 us (busy for
// 51 %), of which about 0.14 ms are the epilogues, which have the CU to themselves: with a gelu and a checkpoint 28 instructions
// per value and 3 bytes written (with neither y is 55 us shorter).
template <class T, class Out, bool P_BY_K, bool Q_BY_K, int DEEP>
__global__ void __launch_bounds__(WIDE_THREADS, 2) k_product_wide(ProductArgs a, Out out) {
	constexpr int TILE = 256, TM = 4, TN = 2, BUFFERS = 128 / DEEP;
	typedef Stage<T, TILE, P_BY_K, DEEP, WIDE_THREADS> PStage;
	typedef Stage<T, TILE, Q_BY_K, DEEP, WIDE_THREADS> QStage;
	constexpr int STAGE = PStage::BYTES + QStage::BYTES, LOADS = PStage::LOADS + QStage::LOADS;
	static_assert(8 * STRIP<TN> * 4 <= BUFFERS * STAGE, "the stages' LDS holds the strips");
	extern __shared__ __attribute__((aligned(16))) char lds[];

	const Place<TILE> at(a, blockIdx.x, gridDim.x);
	const uint32_t wave = threadIdx.x / 64u;
	const uint32_t wm = wave / 4u * 128u, wn = wave % 4u * 64u;
	const uint32_t stages = (uint32_t)((at.k1 - at.k0 + DEEP - 1) / DEEP);

	WriteOut<T, Out, TM, TN> write_out(a, out, at.m0 + wm, at.n0 + wn);
	f32x16 c[TN][TM] = {};
	if (stages) {
		PStage ps;
		QStage qs;
		Fragments<PStage, TILE, P_BY_K, DEEP, TM> pf;
		Fragments<QStage, TILE, Q_BY_K, DEEP, TN> qf;
		ps.begin(a.p, at.m0, a.M, at.k0, a.K);
		qs.begin(a.q, at.n0, a.N, at.k0, a.K);
		pf.begin(wm);
		qf.begin(wn);
		auto load = [&](uint32_t s) {
			char* to = lds + s % BUFFERS * STAGE;
			ps.load(to, s < stages);
			qs.load(to + PStage::BYTES, s < stages);
		};
		// all but the latest BUFFERS - 2 stages a wave asked for are there, and its reads are done
		constexpr int ARRIVED = waits((BUFFERS - 2) * LOADS, 0), READ = waits(63, 0);
		const uint32_t k_in = (uint32_t)((at.k1 - at.k0 - 1) % DEEP) + 1u;
		ps.load_first(lds, k_in);
		qs.load_first(lds + PStage::BYTES, k_in);
#pragma unroll
		for (int s = 1; s < BUFFERS - 1; ++s) load(s);
		__builtin_amdgcn_s_waitcnt(ARRIVED);
		meet();
		if (wave >= 4u) meet();  // the second set runs half a step behind
		for (uint32_t s = 0; s < stages; ++s) {
			// the buffer of stage s - 1 is free: both sets have read it, the second before the barrier just passed
			load(s + BUFFERS - 1);
			const char* from = lds + s % BUFFERS * STAGE;
#pragma unroll
			for (int step = 0; step < DEEP / 32; ++step) {
				s16x8 p[2][TM], q[2][TN];
#pragma unroll
				for (int k = 0; k < 2; ++k) {
#pragma unroll
					for (int t = 0; t < TN; ++t) q[k][t] = qf.read(from + PStage::BYTES, 2 * step + k, t);
#pragma unroll
					for (int t = 0; t < TM; ++t) p[k][t] = pf.read(from, 2 * step + k, t);
				}
				// before the next stage is read: it has arrived as far as this wave asked for it; the barriers tell of the others
				if (step == DEEP / 32 - 1) __builtin_amdgcn_s_waitcnt(ARRIVED);
				else __builtin_amdgcn_s_waitcnt(READ);
				meet();
				__builtin_amdgcn_s_setprio(1);
#pragma unroll
				for (int k = 0; k < 2; ++k)
#pragma unroll
					for (int n = 0; n < TN; ++n)
#pragma unroll
						for (int m = 0; m < TM; ++m) c[n][m] = mfma(T{}, q[k][n], p[k][m], c[n][m]);
				__builtin_amdgcn_s_setprio(0);
				meet();
			}
		}
		if (wave < 4u) meet();
		__builtin_amdgcn_s_waitcnt(0);
	}
	__syncthreads();
	write_out(at.split, reinterpret_cast<float*>(lds) + wave * STRIP<TN>, c);
}

// The splits' sums to where the product would have put them.  `lines` threads (a power of two up to 32) share an eight's
// splits, each the ones in its turn; their sums meet in a fixed order.  Four neighbouring threads finish a block of 32.
template <class T, class Out>
__global__ void __launch_bounds__(256) k_product_join(const float* __restrict__ partial, uint32_t splits, size_t M, uint32_t N, uint32_t lines, Out out) {
	const uint32_t n8 = (N + 7u) & ~7u, chunks = (N + 31u) / 32u * 4u, items = 256u / lines;
	const uint32_t item = threadIdx.x % items, line = threadIdx.x / items;
	const size_t t = (size_t)blockIdx.x * items + item, i = t / chunks;
	const uint32_t j = (uint32_t)(t % chunks) * 8u;
	const bool in = i < M && j < N;
	float v[8] = {};
	if (in)
#pragma unroll 4
		for (uint32_t s = line; s < splits; s += lines) {
			float x[8];
			load8(partial + ((size_t)s * M + i) * n8 + j, 8, x);
#pragma unroll
			for (int k = 0; k < 8; ++k) v[k] += x[k];
		}
	if (lines > 1) {
		__shared__ float sums[8][256];
#pragma unroll
		for (int k = 0; k < 8; ++k) sums[k][threadIdx.x] = v[k];
		__syncthreads();
		if (line) return;
		for (uint32_t l = 1; l < lines; ++l)
#pragma unroll
			for (int k = 0; k < 8; ++k) v[k] += sums[k][l * items + item];
	}
	const uint32_t left = in ? N - j : 0u;
	typename Out::Fetched fetched = {};
	if (left) out.by_kind([&](auto kind) { fetched = out.fetch(kind, i, j, left); });
	finish_block<T>(out, i, j, left, out.columns(j, left), fetched, v);
}

// ---- a few rows ---------------------------------------------------------------------------------------------------------
// Forward for up to 16 rows, as a served network evaluates a query or a few: bound by the read of the weights, and for small
// ones by latency, so one launch and no workspace.  A workgroup of eight waves takes FEATURES outputs and all rows; the waves
// take 64 of k in turn, of which a lane reads 16 neighbouring ones (32 bytes of a weight's row and of a row of x, in whatever
// alignment) for two matrix instructions: their k is permuted the same way in both operands.  The waves' sums meet in LDS.
constexpr uint32_t FEW_ROWS = 16, FEW_THREADS = 512;
__device__ __forceinline__ f32x4 mfma16(f16, s16x8 a, s16x8 b, f32x4 c) {
	return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8<f16>, a), __builtin_bit_cast(v8<f16>, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bf16, s16x8 a, s16x8 b, f32x4 c) {
	return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8<bf16>, a), __builtin_bit_cast(v8<bf16>, b), c, 0, 0, 0);
}

template <class T, int FEATURES>
__global__ void __launch_bounds__(FEW_THREADS) k_few_rows(const T* __restrict__ x, size_t x_stride, const T* __restrict__ w, size_t w_stride,
                                                          uint32_t n, uint32_t n_in, uint32_t n_out, ForwardOut<T> out) {
	constexpr int TILES = FEATURES / 16, WAVES = FEW_THREADS / 64, AHEAD = 4;  // steps of 64 k whose reads go out together
	const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64u, row = lane & 15u, j0 = blockIdx.x * FEATURES;
	// rows that are not there: the last one's values, whose sums nobody takes
	const T* xr = x + min(row, n - 1u) * x_stride;
	const T* wr[TILES];
#pragma unroll
	for (int t = 0; t < TILES; ++t) wr[t] = w + min(j0 + t * 16u + row, n_out - 1u) * w_stride;
	f32x4 c[TILES] = {};
	const uint32_t whole = n_in / 64u;
	auto step = [&](uint32_t first, auto count) {  // `count` steps from step `first` on
		v8<T> xv[count][2], wv[count][TILES][2];
#pragma unroll
		for (int u = 0; u < count; ++u) {
			const uint32_t k = (first + u) * 64u + (lane >> 4) * 16u;
#pragma unroll
			for (int h = 0; h < 2; ++h) {
#pragma unroll
				for (int t = 0; t < TILES; ++t) wv[u][t][h] = *reinterpret_cast<const v8<T>*>(wr[t] + k + 8 * h);
				xv[u][h] = *reinterpret_cast<const v8<T>*>(xr + k + 8 * h);
			}
		}
#pragma unroll
		for (int u = 0; u < count; ++u)
#pragma unroll
			for (int h = 0; h < 2; ++h)
#pragma unroll
				for (int t = 0; t < TILES; ++t)
					c[t] = mfma16(T{}, __builtin_bit_cast(s16x8, wv[u][t][h]), __builtin_bit_cast(s16x8, xv[u][h]), c[t]);
	};
	// AHEAD neighbouring steps at a time, 512 bytes of a row, then what is left of them one by one
	uint32_t s = wave * AHEAD;
	for (; s + AHEAD <= whole; s += AHEAD * WAVES) step(s, Kind<AHEAD>{});
	for (uint32_t u = whole / AHEAD * AHEAD + wave; u < whole; u += WAVES) step(u, Kind<1>{});
	if (n_in % 64u && whole % WAVES == wave) {  // the rest of k, filled up with zeros
		const uint32_t k = whole * 64u + (lane >> 4) * 16u;
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			const uint32_t left = n_in > k + 8u * h ? n_in - k - 8u * h : 0u;
			const v8<T> xv = load8_raw(xr + k + 8 * h, left);
#pragma unroll
			for (int t = 0; t < TILES; ++t)
				c[t] = mfma16(T{}, __builtin_bit_cast(s16x8, load8_raw(wr[t] + k + 8 * h, left)), __builtin_bit_cast(s16x8, xv), c[t]);
		}
	}
	// register r of a tile: output 4 (lane / 16) + r of row lane % 16
	constexpr int PITCH = FEATURES + 4;
	__shared__ __attribute__((aligned(16))) float sums[WAVES][16][PITCH];
#pragma unroll
	for (int t = 0; t < TILES; ++t) *reinterpret_cast<f32x4*>(&sums[wave][row][t * 16 + (lane >> 4) * 4]) = c[t];
	__syncthreads();
	if (threadIdx.x >= 16 * FEATURES / 8) return;
	const uint32_t i = threadIdx.x / (FEATURES / 8), f = threadIdx.x % (FEATURES / 8) * 8u, j = j0 + f;
	float v[8] = {};
#pragma unroll
	for (int k = 0; k < WAVES; ++k)
#pragma unroll
		for (int e = 0; e < 8; ++e) v[e] += sums[k][i][f + e];
	const uint32_t left = i < n && j < n_out ? n_out - j : 0u;
#pragma unroll
	for (int e = 0; e < 8; ++e) v[e] = (uint32_t)e < left ? v[e] : 0.0f;
	typename ForwardOut<T>::Fetched fetched = {};
	if (left) out.by_kind([&](auto kind) { fetched = out.fetch(kind, i, j, left); });
	finish_block<T>(out, i, j, left, out.columns(j, left), fetched, v);
}

// ---- narrow layers ------------------------------------------------------------------------------------------------------
// Backward of layers of up to 128 x 128 over many rows: memory bound, so all of it in one pass over dy, z and x.  Persistent
// workgroups of four waves take ROWS rows at a time: dz and the layer's input go to LDS in 16 bits ([row][feature], from
// where dx reads dz along its rows and dW reads both transposed), the weights' fragments and the workgroup's share of dW stay
// in registers, the next rows are on their way from memory meanwhile.  dW and db leave as a share per workgroup.
// 64 -> 64 over 2^18 rows moves 134 MB instead of the 233 MB of separate passes: 30..33 us (4.1..4.5 TB/s), and 5 to join the
// shares.  The registers' bound is the grid's two workgroups per CU (one for 128 x 128): pressed into a third's, the odd
// widths' 195 registers spill (45 -> 61: 84 us and 60; the even ones' 168 fit either way, 30 us).  Of 64 / 128 the odd 64 -> 128
// still spills 47 (bf16) or 65 registers under the bound of two (45 -> 91: 111 us; 64 -> 128: 43), the even forms 2 and 10.
template <class T>
struct NarrowArgs {
	Kept<T> dy, z, x;
	int act, x_act;
	const T* w;
	size_t w_stride, n;
	uint32_t n_in, n_out;
	T* dx;
	size_t dx_stride;
	float* part;               // [workgroup][n_out][n_in up to 8], then n_out sums of dz
	bool want_dw;
};

template <class T, int NI, int NO, bool EVEN>
__global__ void __launch_bounds__(256, NI + NO > 192 ? 1 : 2) k_narrow_backward(NarrowArgs<T> a) {
	constexpr int ROWS = 64;
	constexpr int DZ_ITEMS = ROWS * NO / 8 / 256, X_ITEMS = ROWS * NI / 8 / 256;  // eights per thread
	constexpr int STRIPS = ROWS / 32, NT = NI / 32 / (4 / STRIPS);               // a wave's strip of dx: NT tiles of 32 columns
	constexpr int MW = NO / 32, WT = MW * (NI / 32) / 4;                           // dW: rows of tiles, tiles per wave
	__shared__ __attribute__((aligned(16))) char lds[ROWS * (NO + NI) * 2];
	char* const lds_dz = lds;
	char* const lds_x = lds + ROWS * NO * 2;
	const uint32_t tid = threadIdx.x, wave = tid / 64u, lane = tid & 63u;
	// 16-byte chunk c of a row lies at c ^ twist(row): 16 rows' same chunk (read along the rows) and 4 rows' 64 bytes (read
	// transposed) are each on all banks once
	auto twist = [](uint32_t r, int width) {
		return width == 64 ? (r & 2u) << 1 | (r & 4u) >> 1 | (r & 8u) >> 3 : (r & 3u) << 2 | ((r >> 2) & 3u);
	};
	auto place = [&](uint32_t r, uint32_t c, int width) { return r * (width * 2) + ((c ^ twist(r, width)) << 4); };
	// a transposed fragment's two halves: column tile t of rows 16 s ..
	auto transposed = [&](const char* from, int width, int s, uint32_t t) {
		typedef __attribute__((address_space(3))) s16x4* tr_ptr;
		const uint32_t g = lane >> 4, q = (lane & 15u) >> 2, p = lane & 3u, c = t * 4u + 2u * (g & 1u) + (p >> 1);
		const uint32_t r = 8u * (g >> 1) + q;  // (the twist repeats every 16 rows)
		from += s * 16 * (width * 2) + (p & 1u) * 8u;
		const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(from + place(r, c, width)));
		const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(from + place(r + 4u, c, width)));
		return s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
	};

	// the weights as dx's Q: row = input, k = output
	const uint32_t strip = wave % STRIPS, nt0 = wave / STRIPS * NT;
	s16x8 w[NT][NO / 16] = {};
	if (a.dx) {
#ifdef __HIP_DEVICE_COMPILE__
		// through a buffer, which gives zeros for what is not there: with a condition on the value the compiler puts a branch
		// and a wait around each of these loads (20 us in all)
		const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(a.w), (short)0, 0x7fffffff, 0x00027000);
#pragma unroll
		for (int t = 0; t < NT; ++t)
#pragma unroll
			for (int s = 0; s < NO / 16; ++s)
#pragma unroll
				for (int k = 0; k < 8; ++k) {
					const uint32_t row = (nt0 + t) * 32u + (lane & 31u), out = s * 16u + 8u * (lane >> 5) + k;
					const uint32_t at = row < a.n_in && out < a.n_out ? (out * (uint32_t)a.w_stride + row) * 2u : 0xfffffff0u;
					w[t][s][k] = (short)__builtin_amdgcn_raw_buffer_load_b16(rsrc, at, 0, 0);
				}
#endif
	}

	f32x16 dw[WT] = {};
	float db[8] = {};
	typename Kept<T>::Raw dy[DZ_ITEMS], z[DZ_ITEMS], x[X_ITEMS];
	auto items = [&](size_t row0, auto kind, const Kept<T>& m, uint32_t width, int padded, auto& raw, auto count) {
#pragma unroll
		for (int k = 0; k < count; ++k) {
			const uint32_t item = tid + k * 256u, c = item % (padded / 8u) * 8u;
			const size_t i = row0 + item / (padded / 8u);
			if constexpr (EVEN) {  // both widths are multiples of 8: rows and chunks that are not there are read as the last row's or the first chunk, and not used
				const size_t ic = min(i, a.n - 1);
				const uint32_t cc = c < width ? c : 0u;
				raw[k] = kind == 1 ? m.raw8_values(ic, cc, 8) : m.raw8_checkpoint(ic, cc, 8);
			} else {
				raw[k] = {};
				if (i < a.n && c < width) raw[k] = kind == 1 ? m.raw8_values(i, c, width - c) : m.raw8_checkpoint(i, c, width - c);
			}
		}
	};
	auto ask = [&](size_t row0) {
		items(row0, Kind<1>{}, a.dy, a.n_out, NO, dy, Kind<DZ_ITEMS>{});
		if (a.act != NGP_ACT_NONE) {
			if (a.z.v) items(row0, Kind<1>{}, a.z, a.n_out, NO, z, Kind<DZ_ITEMS>{});
			else items(row0, Kind<2>{}, a.z, a.n_out, NO, z, Kind<DZ_ITEMS>{});
		}
		if (a.want_dw) {
			if (a.x.v) items(row0, Kind<1>{}, a.x, a.n_in, NI, x, Kind<X_ITEMS>{});
			else items(row0, Kind<2>{}, a.x, a.n_in, NI, x, Kind<X_ITEMS>{});
		}
	};
	const size_t chunks = (a.n + ROWS - 1) / ROWS;
	if (blockIdx.x < chunks) ask((size_t)blockIdx.x * ROWS);
	for (size_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
		const size_t row0 = chunk * ROWS;
		__syncthreads();  // the last rows have been read
#pragma unroll
		for (int k = 0; k < DZ_ITEMS; ++k) {
			const uint32_t item = tid + k * 256u, r = item / (NO / 8u), c = item % (NO / 8u);
			float v[8], s[8];
			a.dy.widen8_values(dy[k], v);
			if (a.act != NGP_ACT_NONE) {
				a.z.widen8(z[k], s);
				act_slopes(a.act, s);
#pragma unroll
				for (int e = 0; e < 8; ++e) v[e] *= s[e];
			}
			v8<T> h;
			const bool in = row0 + r < a.n && c * 8u < a.n_out;
#pragma unroll
			for (int e = 0; e < 8; ++e) {
				v[e] = in && (EVEN || c * 8u + e < a.n_out) ? v[e] : 0.0f;
				db[e] += v[e];
				h[e] = narrow<T>(v[e]);
			}
			*reinterpret_cast<s16x8*>(lds_dz + place(r, c, NO)) = __builtin_bit_cast(s16x8, h);
		}
		if (a.want_dw)
#pragma unroll
			for (int k = 0; k < X_ITEMS; ++k) {
				const uint32_t item = tid + k * 256u, r = item / (NI / 8u), c = item % (NI / 8u);
				float v[8];
				a.x.widen8(x[k], v);
				act_values(a.x_act, v);
				v8<T> h;
				const bool in = row0 + r < a.n && c * 8u < a.n_in;
#pragma unroll
				for (int e = 0; e < 8; ++e) h[e] = narrow<T>(in && (EVEN || c * 8u + e < a.n_in) ? v[e] : 0.0f);
				*reinterpret_cast<s16x8*>(lds_x + place(r, c, NI)) = __builtin_bit_cast(s16x8, h);
			}
		__syncthreads();
		if (chunk + gridDim.x < chunks) ask(row0 + (size_t)gridDim.x * ROWS);

		if (a.dx) {
			f32x16 c[NT] = {};
#pragma unroll
			for (int s = 0; s < NO / 16; ++s) {
				const s16x8 p = *reinterpret_cast<const s16x8*>(lds_dz + place(strip * 32u + (lane & 31u), s * 2u + (lane >> 5), NO));
#pragma unroll
				for (int t = 0; t < NT; ++t) c[t] = mfma(T{}, w[t][s], p, c[t]);
			}
			const size_t i = row0 + strip * 32u + (lane & 31u);
#pragma unroll
			for (int t = 0; t < NT; ++t)
#pragma unroll
				for (int h = 0; h < 2; ++h) {
					const uint32_t j = (nt0 + t) * 32u + 16u * h + 8u * (lane >> 5);
					float v[8];
					eight(c[t], h, v);
					if (i >= a.n || j >= a.n_in) continue;
					const uint32_t left = EVEN ? 8u : a.n_in - j;
					if (a.x_act != NGP_ACT_NONE) {
						float s[8];
						a.x.at8(i, j, left, s);
						act_slopes(a.x_act, s);
#pragma unroll
						for (int k = 0; k < 8; ++k) v[k] *= s[k];
					}
					store8(a.dx + i * a.dx_stride + j, left, v);
				}
		}
		if (a.want_dw)
#pragma unroll
			for (int s = 0; s < ROWS / 16; ++s) {
				const s16x8 p = transposed(lds_dz, NO, s, wave % MW);
#pragma unroll
				for (int t = 0; t < WT; ++t) dw[t] = mfma(T{}, transposed(lds_x, NI, s, (wave + 4u * t) / MW), p, dw[t]);
			}
	}

	const uint32_t n8 = (a.n_in + 7u) & ~7u;
	float* part = a.part + (size_t)blockIdx.x * a.n_out * (n8 + 1u);
	if (a.want_dw)
#pragma unroll
		for (int t = 0; t < WT; ++t)
#pragma unroll
			for (int h = 0; h < 2; ++h) {
				const uint32_t i = wave % MW * 32u + (lane & 31u), j = (wave + 4u * t) / MW * 32u + 16u * h + 8u * (lane >> 5);
				float v[8];
				eight(dw[t], h, v);
				if (i < a.n_out && j < n8) store8(part + i * n8 + j, 8, v);
			}
	// the threads that share columns: every NO / 8-th
	float* sums = reinterpret_cast<float*>(lds);
	__syncthreads();
#pragma unroll
	for (int e = 0; e < 8; ++e) sums[tid * 9 + e] = db[e];
	__syncthreads();
	if (tid >= NO || tid >= a.n_out) return;
	float total = 0.0f;
	for (uint32_t o = tid / 8u; o < 256u; o += NO / 8u) total += sums[o * 9 + tid % 8u];
	part[a.n_out * n8 + tid] = total;
}

// A column of those shares to where it belongs.
template <class T>
struct PutNarrow {
	void* dw;
	size_t stride;
	bool f32, accumulate;
	uint32_t n_in, n_out;
	float* db;
	__device__ __forceinline__ void operator()(size_t c, float v) const {
		const uint32_t n8 = (n_in + 7u) & ~7u, i = (uint32_t)c / n8, j = (uint32_t)c % n8;
		if (i >= n_out) {
			float* d = db + (c - n_out * n8);
			if (db) *d = accumulate ? *d + v : v;
		} else if (dw && j < n_in) {
			float* d = static_cast<float*>(dw) + i * stride + j;
			if (f32) *d = accumulate ? *d + v : v;
			else static_cast<T*>(dw)[i * stride + j] = narrow<T>(v);
		}
	}
};

// ---- operands that do not lie as the product wants them ---------------------------------------------------------------
// act(v), rounded to T, in rows of `width` up to 8, filled up with zeros, by `blocks` workgroups.
template <class T>
struct LayOut {
	Kept<T> v;
	int act = NGP_ACT_NONE;
	size_t rows = 0;
	uint32_t width = 0, blocks = 0;
	T* to = nullptr;
	template <bool VALUES>
	__device__ __forceinline__ void run(uint32_t block) const {
		const uint32_t w8 = (width + 7u) & ~7u;
		for (Walk w(w8 / 8u, block, blocks); w.i < rows; w.next()) {
			const uint32_t j = w.e * 8u;
			float x[8];
			v.template at8_of<VALUES>(w.i, j, width - j, x);
			act_values(act, x);
			if (width - j < 8u)
#pragma unroll
				for (int k = 0; k < 8; ++k) x[k] = j + k < width ? x[k] : 0.0f;
			store8(to + w.i * w8 + j, 8, x);
		}
	}
};

// dz = dy act'(z), in rows of `width` up to 8 (to null: not kept), and its sums over a share of the rows (part null: not
// wanted).  A workgroup takes 8 * groups columns (groups a power of two up to 32) and 256 / groups rows at a time; `wide`
// workgroups lie side by side.
template <class T>
struct MakeDz {
	Kept<T> dy, z;
	int act = NGP_ACT_NONE;
	size_t n = 0, rows_each = 0;
	uint32_t width = 0, groups = 1, wide = 1, blocks = 0;
	T* to = nullptr;
	float* part = nullptr;
	__device__ __forceinline__ void run(uint32_t block) const {
		const uint32_t side = block % wide, share = block / wide;
		const uint32_t g = threadIdx.x % groups, lines = 256u / groups, j = (side * groups + g) * 8u;
		const size_t begin = share * rows_each, end = min(begin + rows_each, n);
		const uint32_t w8 = (width + 7u) & ~7u;
		float sum[8] = {};
		if (j < width)
			for (size_t i = begin + threadIdx.x / groups; i < end; i += lines) {
				float d[8];
				dy.template at8_of<true>(i, j, width - j, d);
				if (act != NGP_ACT_NONE) {
					float s[8];
					z.at8(i, j, width - j, s);
					act_slopes(act, s);
#pragma unroll
					for (int k = 0; k < 8; ++k) d[k] = j + k < width ? d[k] * s[k] : 0.0f;
				}
				if (to) store8(to + i * w8 + j, 8, d);
#pragma unroll
				for (int k = 0; k < 8; ++k) sum[k] += d[k];
			}
		if (!part) return;
		__shared__ float s[256][9];
#pragma unroll
		for (int k = 0; k < 8; ++k) s[threadIdx.x][k] = sum[k];
		__syncthreads();
		if (threadIdx.x >= groups * 8u) return;
		const uint32_t column = side * groups * 8u + threadIdx.x;
		if (column >= width) return;
		float total = 0.0f;
		for (uint32_t l = 0; l < lines; ++l) total += s[l * groups + threadIdx.x / 8u][threadIdx.x % 8u];
		part[(size_t)share * width + column] = total;
	}
};

// What the products need first, side by side in one launch.
template <class T>
__global__ void __launch_bounds__(256) k_prepare(MakeDz<T> dz, LayOut<T> a, LayOut<T> b) {
	if (blockIdx.x < dz.blocks) {
		dz.run(blockIdx.x);
		return;
	}
	const bool first = blockIdx.x - dz.blocks < a.blocks;
	const LayOut<T>& l = first ? a : b;
	const uint32_t block = blockIdx.x - dz.blocks - (first ? 0u : a.blocks);
	l.v.v ? l.template run<true>(block) : l.template run<false>(block);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
static size_t up16(size_t b) { return (b + 15) & ~(size_t)15; }
static uint32_t up8(uint32_t w) { return (w + 7u) & ~7u; }

// The workspace as a call deals it out, and how much of it is taken (the size to ask for, where nothing is launched).
struct Room {
	char* at;
	size_t bytes = 0;
	template <class U>
	U* take(size_t count) {
		U* p = reinterpret_cast<U*>(at + bytes);
		bytes += up16(count * sizeof(U));
		return p;
	}
};

struct ProductPlan {
	int tile = 64;
	uint32_t tiles_m = 0, tiles_n = 0, splits = 1;
	size_t k_each = 0;
	double us = 1e30;  // estimated
};

// The tile and how often K is split: whichever pair should take least, in microseconds as measured over products of 32 to
// 65536 rows (bf16, both operands along k; the estimate is within a quarter of the measured time).  With n workgroups per CU,
// rounded up, a stage of 64 k takes max(least, n each): a 64 tile's loads and barriers take as long as two of it multiply
// (1024^3: 8 us with 64 tiles, 12 with 128, 25 with 256), a 256 tile moves a quarter of the bytes per multiplication (4096 x
// 2048 x 4096: 105, 70 and 60 us).  Splits write their sums and read them again at about 4.2 TB/s, in a launch of their own
// (32 x 4096 x 4096: 19 us with 64 tiles, 12 with four splits; 2048 x 1024 x 1024: 10 us, 24 with two).  Each product is taken
// as if it had the GPU to itself: dx and dW side by side share it and take longer together than either estimate says (3001 rows
// 777 -> 1030: 15 us estimated for each, 31 measured for both).
static ProductPlan plan_product(size_t M, uint32_t N, size_t K, int only = 0) {
	struct Kind {
		int tile;
		double least, each;
	};
	ProductPlan best;
	const size_t stages = std::max<size_t>(1, (K + PRODUCT_K - 1) / PRODUCT_K);
	for (const Kind& kind : {Kind{64, 0.23, 0.185}, Kind{128, 0.5, 0.52}, Kind{256, 1.3, 1.68}}) {
		if (only && kind.tile != only) continue;
		const size_t tiles = ((M + kind.tile - 1) / kind.tile) * (((size_t)N + kind.tile - 1) / kind.tile);
		if (tiles >= 1u << 23) continue;  // (a launch has fewer than 2^32 threads; 256 tiles hold every matrix that memory does)
		for (size_t splits = 1; splits <= std::min<size_t>(64, stages); splits *= 2) {
			const size_t each = (stages + splits - 1) / splits, used = (stages + each - 1) / each;
			if (used > 1 && tiles * used > 65536) break;
			const double n = (double)((tiles * used + 255) / 256);
			const double join = used > 1 ? 3.0 + 8e-6 * (double)used * (double)M * N / 4.2 : 0.0;
			const double finish = 0.4 * (kind.tile / 64) * (kind.tile / 64);  // a tile's results at a CU's share of the memory's rate
			const double t = 4.0 + finish * n + each * std::max(kind.least, kind.each * n) + join;
			if (t >= best.us) continue;
			best.us = t;
			best.tile = kind.tile;
			best.splits = (uint32_t)used;
			best.k_each = each * PRODUCT_K;
		}
	}
	best.tiles_m = (uint32_t)((M + best.tile - 1) / best.tile);
	best.tiles_n = (uint32_t)((N + best.tile - 1) / best.tile);
	return best;
}

// A kernel's LDS past the default of 64 KiB (its own static LDS counted) has to be allowed, on each device that it runs on: at
// every launch, so that nothing is kept between calls.
template <class... Args>
static void launch_lds(void (*kernel)(Args...), uint32_t blocks, uint32_t threads, uint32_t lds, hipStream_t s, Args... args) {
	if (lds >= 65536)
		NGP_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
	kernel<<<blocks, threads, lds, s>>>(args...);
	NGP_HIP_CHECK(hipGetLastError());
}

// The more splits there are, and the fewer sums, the more threads share one's splits: about four each.
template <class T, class Out>
static void join(const float* partial, uint32_t splits, size_t M, uint32_t N, const Out& out, hipStream_t s) {
	const size_t items = M * ((N + 31u) / 32u * 4u);
	uint32_t lines = 1;
	while (lines < 32 && lines * 4 < splits && items * lines < 262144) lines *= 2;
	k_product_join<T, Out><<<(uint32_t)((items * lines + 255) / 256), 256, 0, s>>>(partial, splits, M, N, lines, out);
	NGP_HIP_CHECK(hipGetLastError());
}

// C[M][N] = P Q^T by a plan; the splits' sums take their place in the workspace.
static ProductArgs product_args(const ProductPlan& plan, const Matrix& p, const Matrix& q, size_t M, uint32_t N, size_t K, Room& room) {
	ProductArgs a{p, q, M, K, plan.k_each, N, plan.tiles_m, plan.tiles_n, plan.splits, nullptr};
	if (plan.splits > 1) a.partial = room.take<float>((size_t)plan.splits * M * up8(N));
	return a;
}
// (up to two stages of K take two buffers: more workgroups per CU hide what one stage cannot)
static bool is_short(const ProductPlan& plan) { return plan.k_each <= 2 * PRODUCT_K; }

template <class T, class Out, bool P_BY_K, bool Q_BY_K>
static void product(const ProductPlan& plan, const ProductArgs& a, const Out& out, hipStream_t s) {
	const uint32_t blocks = a.tiles_m * a.tiles_n * a.splits;
	// (rows along k come 128 bytes at a time from stages of 64: half the requests to L2, y of 16384 x 2048 x 8192 578 us, 603 with
	// stages of 32; with an operand by k, whose lines are long either way, stages of 32 ask further ahead: dx 260 M busy cycles,
	// 278 M with stages of 64 (574 us and 580); dW alone would have the stages of 64, 423 us and 436)
	if (plan.tile == 256) launch_lds(k_product_wide<T, Out, P_BY_K, Q_BY_K, P_BY_K || Q_BY_K ? 32 : 64>, blocks, WIDE_THREADS, 131072, s, a, out);
	else if (plan.tile == 128) launch_lds(k_product<T, Out, P_BY_K, Q_BY_K, 128, 2>, blocks, PRODUCT_THREADS, 2 * 32768, s, a, out);
	else if (is_short(plan)) launch_lds(k_product<T, Out, P_BY_K, Q_BY_K, 64, 2>, blocks, PRODUCT_THREADS, 2 * 16384, s, a, out);
	else launch_lds(k_product<T, Out, P_BY_K, Q_BY_K, 64, 3>, blocks, PRODUCT_THREADS, 3 * 16384, s, a, out);
	if (a.splits > 1) join<T>(a.partial, a.splits, a.M, a.N, out, s);
}

// Whether a product's loads, 16 bytes at a time, can take a matrix where it lies.
static bool in_place(const void* p, size_t stride, uint32_t width) {
	return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0 && width % 8 == 0;
}

// `v` where it lies if the product can read it there, else act(v) copied to the workspace by `lay`.
template <class T>
static Matrix operand(const Kept<T>& v, int act, size_t rows, uint32_t width, Room& room, LayOut<T>& lay) {
	if (v.v && act == NGP_ACT_NONE && in_place(v.v, v.stride, width)) return {v.v, v.stride};
	T* to = room.take<T>(rows * up8(width));
	const size_t blocks = (rows * (up8(width) / 8) + 255) / 256;
	lay = LayOut<T>{v, act, rows, width, (uint32_t)std::min<size_t>(blocks, 16384), to};
	return {to, up8(width)};
}

template <class T>
static void prepare(const MakeDz<T>& dz, const LayOut<T>& a, const LayOut<T>& b, hipStream_t s) {
	const uint32_t blocks = dz.blocks + a.blocks + b.blocks;
	if (!blocks) return;
	k_prepare<T><<<blocks, 256, 0, s>>>(dz, a, b);
	NGP_HIP_CHECK(hipGetLastError());
}

constexpr uint32_t NARROW_WIDTH = 128, NARROW_ROWS = 16384;

template <class T>
static size_t linear_forward(const ngp_linear_args& a, bool run, hipStream_t s) {
	Room room{static_cast<char*>(a.workspace)};
	if (!a.n) return 0;
	const ForwardOut<T> out{a.bias, static_cast<const T*>(a.residual), static_cast<T*>(a.y), static_cast<T*>(a.z), a.z8,
	                        a.residual_stride, a.y_stride, a.z_stride, a.activation};
	// 16 outputs per workgroup; 32 where a checkpoint's blocks are, or where that still gives every CU one.  A CU reads the
	// weights at 20 GB/s: with few outputs and a long K the product's splits use more of them (16 x 16384 x 1024: 30 us, 12).
	const bool pairs = a.z8.q || a.n_out > 256 * 16;
	const uint32_t groups = pairs ? (a.n_out + 31) / 32 : (a.n_out + 15) / 16;
	const double few_us = 2.5 + 2.0 * a.n_in * a.n_out / (std::min(groups, 256u) * 20e3);
	if (a.n <= FEW_ROWS && few_us <= plan_product(a.n, a.n_out, a.n_in).us) {
		if (!run) return 0;
		const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.weights);
		if (pairs)
			k_few_rows<T, 32><<<groups, FEW_THREADS, 0, s>>>(x, a.x_stride, w, a.weights_stride, a.n, a.n_in, a.n_out, out);
		else
			k_few_rows<T, 16><<<groups, FEW_THREADS, 0, s>>>(x, a.x_stride, w, a.weights_stride, a.n, a.n_in, a.n_out, out);
		NGP_HIP_CHECK(hipGetLastError());
		return 0;
	}
	LayOut<T> lay_x, lay_w;
	const Matrix x = operand<T>(kept<T>(a.x, a.x_stride, {}), NGP_ACT_NONE, a.n, a.n_in, room, lay_x);
	const Matrix w = operand<T>(kept<T>(a.weights, a.weights_stride, {}), NGP_ACT_NONE, a.n_out, a.n_in, room, lay_w);
	const ProductPlan plan = plan_product(a.n, a.n_out, a.n_in);
	const ProductArgs args = product_args(plan, x, w, a.n, a.n_out, a.n_in, room);
	if (!run) return room.bytes;
	prepare<T>({}, lay_x, lay_w, s);
	product<T, ForwardOut<T>, false, false>(plan, args, out, s);
	return room.bytes;
}

// Narrow layers' backward in one pass, where there are rows enough for every CU's first turn: two workgroups per CU, for
// 128 x 128 (with four times the sums to leave behind) one.
template <class T, int NI, int NO>
static void launch_narrow(const NarrowArgs<T>& a, uint32_t grid, hipStream_t s) {
	auto kernel = a.n_in % 8 == 0 && a.n_out % 8 == 0 ? k_narrow_backward<T, NI, NO, true> : k_narrow_backward<T, NI, NO, false>;
	kernel<<<grid, 256, 0, s>>>(a);
	NGP_HIP_CHECK(hipGetLastError());
}
template <class T>
static size_t narrow_backward(const ngp_linear_backward_args& a, bool run, hipStream_t s) {
	Room room{static_cast<char*>(a.workspace)};
	const bool ni = a.n_in > 64, no = a.n_out > 64;
	const uint32_t grid = ni && no ? 256 : 512;
	const size_t columns = (size_t)a.n_out * (up8(a.n_in) + 1);
	float* part = room.take<float>(grid * columns);
	if (!run) return room.bytes;
	const NarrowArgs<T> p{kept<T>(a.dy, a.dy_stride, {}), kept<T>(a.z, a.z_stride, a.z8), kept<T>(a.x, a.x_stride, a.x8), a.activation,
	                      a.x_activation, static_cast<const T*>(a.weights), a.weights_stride, a.n, a.n_in, a.n_out,
	                      static_cast<T*>(a.dx), a.dx_stride, part, a.dweights != nullptr};
	if (ni && no) launch_narrow<T, 128, 128>(p, grid, s);
	else if (ni) launch_narrow<T, 128, 64>(p, grid, s);
	else if (no) launch_narrow<T, 64, 128>(p, grid, s);
	else launch_narrow<T, 64, 64>(p, grid, s);
	if (a.dweights || a.dbias)
		launch_column_sums(part, grid, columns, PutNarrow<T>{a.dweights, a.dweights_stride, a.dweights_type == NGP_TYPE_F32,
		                                                     a.accumulate != 0, a.n_in, a.n_out, a.dbias}, s);
	return room.bytes;
}

template <class T>
static size_t linear_backward(const ngp_linear_backward_args& a, bool run, hipStream_t s) {
	if (a.n >= NARROW_ROWS && a.n_in <= NARROW_WIDTH && a.n_out <= NARROW_WIDTH && (a.dx || a.dweights)) return narrow_backward<T>(a, run, s);
	Room room{static_cast<char*>(a.workspace)};
	const bool want_dx = a.dx && a.n, want_dw = a.dweights;
	const Kept<T> x = kept<T>(a.x, a.x_stride, a.x8);
	// dz where it has to be made, or copied into rows that the products can read
	const bool make_dz = (want_dx || want_dw) && (a.activation != NGP_ACT_NONE || !in_place(a.dy, a.dy_stride, a.n_out));
	T* dz_to = make_dz ? room.take<T>((size_t)a.n * up8(a.n_out)) : nullptr;
	const Matrix dz = make_dz ? Matrix{dz_to, up8(a.n_out)} : Matrix{a.dy, a.dy_stride};
	MakeDz<T> job;
	Sums sums{nullptr, 0, 0, {a.dbias, nullptr, a.n_out, a.accumulate != 0}};
	if (make_dz || a.dbias) {
		uint32_t groups = 1;
		while (groups < 32 && groups * 8 < a.n_out) groups *= 2;
		const uint32_t wide = (a.n_out + groups * 8 - 1) / (groups * 8), lines = 256 / groups;
		// about four workgroups per CU
		const uint32_t shares = (uint32_t)std::max<size_t>(1, std::min<size_t>(((size_t)a.n + lines - 1) / lines, std::max(1u, 1024u / wide)));
		float* part = a.dbias ? room.take<float>((size_t)shares * a.n_out) : nullptr;
		job = MakeDz<T>{kept<T>(a.dy, a.dy_stride, {}), kept<T>(a.z, a.z_stride, a.z8), a.activation, a.n, ((size_t)a.n + shares - 1) / shares,
		                a.n_out, groups, wide, wide * shares, dz_to, part};
		if (a.dbias) sums.part = part, sums.shares = shares, sums.columns = a.n_out;
	}
	LayOut<T> lay_w, lay_x;
	ProductPlan dx_plan, dw_plan;
	ProductArgs dx_args{}, dw_args{};
	if (want_dx) dx_plan = plan_product(a.n, a.n_in, a.n_out);
	if (want_dw) dw_plan = plan_product(a.n_out, a.n_in, a.n);
	bool together = want_dx && want_dw && dx_plan.tile < 256 && dw_plan.tile < 256;
	if (together && dx_plan.tile != dw_plan.tile) {  // side by side they need the same tile
		const ProductPlan dx64 = plan_product(a.n, a.n_in, a.n_out, 64), dx128 = plan_product(a.n, a.n_in, a.n_out, 128);
		const ProductPlan dw64 = plan_product(a.n_out, a.n_in, a.n, 64), dw128 = plan_product(a.n_out, a.n_in, a.n, 128);
		const bool small = dx64.us + dw64.us < dx128.us + dw128.us;
		dx_plan = small ? dx64 : dx128;
		dw_plan = small ? dw64 : dw128;
	}
	if (want_dx) {
		const Matrix w = operand<T>(kept<T>(a.weights, a.weights_stride, {}), NGP_ACT_NONE, a.n_out, a.n_in, room, lay_w);
		dx_args = product_args(dx_plan, dz, w, a.n, a.n_in, a.n_out, room);
	}
	if (want_dw) {
		const Matrix xs = operand<T>(x, a.x_activation, a.n, a.n_in, room, lay_x);
		dw_args = product_args(dw_plan, dz, xs, a.n_out, a.n_in, a.n, room);
	}
	if (!run) return room.bytes;

	prepare<T>(job, lay_w, lay_x, s);
	const GradientOut<T> dx_out{static_cast<T*>(a.dx), a.dx_stride, x, a.x_activation};
	const WeightsOut<T> dw_out{a.dweights, a.dweights_stride, a.dweights_type == NGP_TYPE_F32, a.accumulate != 0};
	if (together) {
		const uint32_t dx_blocks = dx_args.tiles_m * dx_args.tiles_n * dx_args.splits, dw_blocks = dw_args.tiles_m * dw_args.tiles_n * dw_args.splits;
		const uint32_t blocks = dx_blocks + dw_blocks + (sums.columns + 15) / 16;
		if (dx_plan.tile == 128)
			launch_lds(k_backward_products<T, 128, 2>, blocks, PRODUCT_THREADS, 2 * 32768, s, dx_args, dx_out, dx_blocks, dw_args, dw_out, dw_blocks, sums);
		else if (is_short(dx_plan) && is_short(dw_plan))
			launch_lds(k_backward_products<T, 64, 2>, blocks, PRODUCT_THREADS, 2 * 16384, s, dx_args, dx_out, dx_blocks, dw_args, dw_out, dw_blocks, sums);
		else
			launch_lds(k_backward_products<T, 64, 3>, blocks, PRODUCT_THREADS, 3 * 16384, s, dx_args, dx_out, dx_blocks, dw_args, dw_out, dw_blocks, sums);
		if (dx_args.splits > 1) join<T>(dx_args.partial, dx_args.splits, a.n, a.n_in, dx_out, s);
		if (dw_args.splits > 1) join<T>(dw_args.partial, dw_args.splits, a.n_out, a.n_in, dw_out, s);
		return room.bytes;
	}
	if (sums.columns) launch_column_sums(sums.part, sums.shares, sums.columns, sums.put, s);
	if (want_dx) product<T, GradientOut<T>, false, true>(dx_plan, dx_args, dx_out, s);
	if (want_dw) product<T, WeightsOut<T>, true, true>(dw_plan, dw_args, dw_out, s);
	return room.bytes;
}

size_t linear_workspace(const ngp_linear_args& a) {
	return a.type == NGP_TYPE_F16 ? linear_forward<f16>(a, false, 0) : linear_forward<bf16>(a, false, 0);
}
size_t linear_backward_workspace(const ngp_linear_backward_args& a) {
	return a.type == NGP_TYPE_F16 ? linear_backward<f16>(a, false, 0) : linear_backward<bf16>(a, false, 0);
}

void run_linear_forward(const ngp_linear_args& a, hipStream_t s) {
	if (a.type == NGP_TYPE_F16) linear_forward<f16>(a, true, s);
	else linear_forward<bf16>(a, true, s);
}

void run_linear_backward(const ngp_linear_backward_args& a, hipStream_t s) {
	if (a.type == NGP_TYPE_F16) linear_backward<f16>(a, true, s);
	else linear_backward<bf16>(a, true, s);
}

}  // namespace ngp
