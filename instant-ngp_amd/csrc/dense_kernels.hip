// dense_kernels.hip -- dense layers of any width: Y = act(X W^T + b) + R (ngp_linear_*) and the gated projections
// H = act(X Wg^T + bg) * (X Wu^T + bu) (ngp_gated_*), forward and backward, on the matrix cores.
// Compiled once per element type (DENSE_BF16 undefined: half, defined: bfloat16).
//
// All three products of a layer are one kernel over tiles C[rows, cols] = sum_t A[rows, t] B[cols, t]; they differ in which
// dimension of an operand is contiguous:
//   forward   Y  = X  W^T   rows = samples, cols = outputs, t = inputs     both operands contiguous along t
//   input     dX = G  W     rows = samples, cols = inputs,  t = outputs    B contiguous along its columns
//   weights   dW = G^T X    rows = outputs, cols = inputs,  t = samples    both contiguous along rows / columns
// with G = dY * act'(Z).  Operands that are contiguous along t are read from LDS as 16-byte fragments, the others with the
// transposing LDS read (ds_read_b64_tr_b16: 16 lanes exchange a 4 x 16 block), so no operand is ever rearranged in memory.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <algorithm>
#include <cstring>
#include "ngp_kernels.hpp"

namespace ngp {
#ifdef DENSE_BF16
typedef __bf16 T;
#define DENSE_NAME(x) x##_bf16
#else
typedef _Float16 T;
#define DENSE_NAME(x) x##_half
#endif

namespace {
typedef T T8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

__device__ inline f4v mfma(T8 a, T8 b, f4v c) {
#ifdef DENSE_BF16
	return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
	return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#endif
}
// 8 consecutive elements at any 2-byte aligned address (one 16-byte access: global memory takes unaligned vectors); the first n of them where n < 8
__device__ inline T8 load8(const T* p) { T8 v; __builtin_memcpy(&v, p, 16); return v; }
__device__ inline T8 load8(const T* p, int n) {
	if (n >= 8) return load8(p);
	T8 v{};
#pragma unroll
	for (int i = 0; i < 8; ++i) if (i < n) v[i] = p[i];
	return v;
}
__device__ inline void store8(T* p, T8 v, int n) {
	if (n >= 8) { __builtin_memcpy(p, &v, 16); return; }
#pragma unroll
	for (int i = 0; i < 8; ++i) if (i < n) p[i] = v[i];
}

// ---- activations: values and derivatives in 32 bits.  1 / (1 + e^-z) through v_exp_f32 / v_rcp_f32 (1 ulp each): far below the 16-bit rounding of the result
__device__ inline float logistic(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
__device__ inline float act_value(int act, float z) {
	switch (act) {
		case NGP_ACT_RELU: return z < 0.f ? 0.f : z; // (NaN stays NaN)
		case NGP_ACT_LOGISTIC: return logistic(z);
		case NGP_ACT_EXPONENTIAL: return __expf(z);
		case NGP_ACT_SILU: return z * logistic(z);
		case NGP_ACT_GELU: return 0.5f * z * erfcf(-0.70710678f * z);
		default: return z;
	}
}
__device__ inline void act_value_slope(int act, float z, float& value, float& slope) {
	switch (act) {
		case NGP_ACT_RELU: value = z < 0.f ? 0.f : z; slope = z > 0.f ? 1.f : 0.f; break;
		case NGP_ACT_LOGISTIC: { const float p = logistic(z); value = p; slope = p * (1.f - p); break; }
		case NGP_ACT_EXPONENTIAL: value = slope = __expf(z); break;
		case NGP_ACT_SILU: { const float p = logistic(z); value = z * p; slope = p * (1.f + z * (1.f - p)); break; }
		case NGP_ACT_GELU: { const float c = 0.5f * erfcf(-0.70710678f * z); value = z * c; slope = c + z * 0.39894228f * __expf(-0.5f * z * z); break; }
		default: value = z; slope = 1.f;
	}
}

// ---- one operand's tile in LDS: EXTENT rows (A) or columns (B) x TK steps of the sum, in 16-byte slots.
// T_CONTIG: [EXTENT][TK] (a fragment = one 16-byte read), else [TK][EXTENT] (transposing reads).  The slots of a line are exchanged by an
// XOR with the line number so that the 16 lanes of a read hit different banks; a slot's source chunk is source(line, slot).
// B's columns are dealt to the fragments in groups of 4 (fragment j of a pair holds columns 8q + 4(j & 1) + 0..3): a lane then owns 8 consecutive columns of C.
constexpr int TK = 64;
template <int EXTENT, bool T_CONTIG, bool IS_B> struct Tile {
	static constexpr int SLOTS = T_CONTIG ? TK / 8 : EXTENT / 8, LINES = T_CONTIG ? EXTENT : TK, N_SLOTS = SLOTS * LINES, ELEMS = EXTENT * TK;
	__device__ static int source(int line, int slot) {
		if (T_CONTIG) return IS_B ? slot ^ ((line & 3) | ((line >> 1) & 4)) : slot ^ (line & 7);
		if (IS_B) return slot ^ ((line & (EXTENT >= 128 ? 3 : 1)) << 2);  // exchanged in 64-byte pieces (a pair of fragments' columns)
		return slot ^ ((line & (EXTENT >= 128 ? 7 : 3)) << 1);            // in 32-byte pieces (a fragment's rows)
	}
	// fragment of lane (g = lane / 16, i = lane % 16) for the 32 steps from ks * 32; `at` = first row of the fragment (A) or of the pair (B), odd = j & 1
	__device__ static T8 read(const T* lds, int at, int odd, int ks, int g, int i) {
		if constexpr (T_CONTIG) {
			const int line = IS_B ? at + ((i >> 2) << 3) + odd * 4 + (i & 3) : at + i;
			return *(const T8*)(lds + line * TK + source(line, ks * 4 + g) * 8); // (an XOR is its own inverse)
		} else {
			union { s4 h[2]; T8 v; } r;
#pragma unroll
			for (int h = 0; h < 2; ++h) {
				const int line = ks * 32 + g * 8 + h * 4 + (i >> 2);
				const int e = IS_B ? at + ((i & 3) << 3) + odd * 4 : at + ((i & 3) << 2);
				const T* p = lds + line * EXTENT + source(line, e >> 3) * 8 + (e & 7);
				r.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p);
			}
			return r.v;
		}
	}
};

enum { EPI_LINEAR, EPI_GATED, EPI_STORE, EPI_PARTIAL };
struct GemmArgs {
	const T* a; const T* b[2]; uint64_t lda, ldb;
	uint32_t rows, cols, steps;      // C is rows x cols; the sum runs over `segments` pieces of `steps`
	uint32_t segments; uint64_t a_segment; // dX of a gated layer: A's second piece is a_segment elements further along t, B's is b[1]
	uint64_t a_problem; uint32_t problems; // dW of a gated layer: two products with the same B (A a_problem elements further)
	uint32_t splits, chunks_per_split;     // the sum is split over blocks: partial sums to `partial`
	T* c[2]; uint64_t ldc;
	float* partial;                        // [split][problem][rows][cols8]
	int act; const T* bias[2]; const T* residual; uint64_t ld_residual; T* pre[2]; uint64_t ld_pre;
};
__host__ __device__ inline uint32_t up8(uint32_t v) { return (v + 7) & ~7u; }

// C tile BR x BC by WR x WC wavefronts; each owns (BR / WR) x (BC / WC) as 16 x 16 fragments (matrix instruction 16x16x32, C^T: a lane holds one row of C and 4 columns
// of each fragment).  EPI_GATED: the tile's columns are BC / 2 gate outputs and the same BC / 2 up outputs, every wavefront owns both of its columns.
template <int BR, int BC, int WR, int WC, bool A_T, bool B_T, int EPI>
__global__ __launch_bounds__(64 * WR * WC) void k_gemm(GemmArgs g) {
	typedef Tile<BR, A_T, false> TA; typedef Tile<BC, B_T, true> TB;
	constexpr int THREADS = 64 * WR * WC, FR = BR / WR / 16, FC = BC / WC / 16, NA = TA::N_SLOTS / THREADS, NB = TB::N_SLOTS / THREADS;
	constexpr int OUT = EPI == EPI_GATED ? BC / 2 : BC; // columns of C per tile
	static_assert(FC % (EPI == EPI_GATED ? 4 : 2) == 0, "pairs of fragments");
	__shared__ __attribute__((aligned(16))) T lds_a[TA::ELEMS];
	__shared__ __attribute__((aligned(16))) T lds_b[TB::ELEMS];
	const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wr = wave / WC, wc = wave % WC, gq = lane >> 4, li = lane & 15;
	const uint32_t col_tiles = (g.cols + OUT - 1) / OUT;
	const uint32_t r0 = blockIdx.x / col_tiles * BR, c0 = blockIdx.x % col_tiles * OUT;
	const uint32_t problem = blockIdx.y, split = blockIdx.z;
	const T* a = g.a + problem * g.a_problem;
	const uint32_t chunks_per_segment = (g.steps + TK - 1) / TK, n_chunks = chunks_per_segment * g.segments;
	const uint32_t t_begin = split * g.chunks_per_split, t_end = min(n_chunks, t_begin + g.chunks_per_split);
	auto pair_at = [&](int p) -> int { // first column (in the B tile) of fragment pair p of this wavefront
		if (EPI == EPI_GATED) return (p >= FC / 4 ? OUT : 0) + (int)wc * (OUT / WC) + (p % (FC / 4)) * 32;
		return (int)wc * (BC / WC) + p * 32;
	};
	f4v acc[FR][FC];
#pragma unroll
	for (int i = 0; i < FR; ++i)
#pragma unroll
		for (int j = 0; j < FC; ++j) acc[i][j] = f4v{0.f, 0.f, 0.f, 0.f};
	T8 ra[NA], rb[NB];
	auto load = [&](uint32_t t) {
		const uint32_t seg = t / chunks_per_segment, t0 = (t - seg * chunks_per_segment) * TK;
		const int left = (int)min((uint32_t)TK, g.steps - t0);
#pragma unroll
		for (int q = 0; q < NA; ++q) {
			const int slot = q * THREADS + tid, line = slot / TA::SLOTS, chunk = TA::source(line, slot % TA::SLOTS);
			const T* base = a + seg * g.a_segment;
			if (A_T) { const bool in = r0 + line < g.rows; ra[q] = load8(base + (uint64_t)(r0 + line) * g.lda + t0 + chunk * 8, in ? left - chunk * 8 : 0); }
			else { const uint32_t r = r0 + chunk * 8; ra[q] = load8(base + (uint64_t)(t0 + line) * g.lda + r, line < left ? (int)g.rows - (int)r : 0); }
		}
#pragma unroll
		for (int q = 0; q < NB; ++q) {
			const int slot = q * THREADS + tid, line = slot / TB::SLOTS, chunk = TB::source(line, slot % TB::SLOTS);
			if (B_T) {
				const uint32_t which = EPI == EPI_GATED && line >= OUT, col = c0 + line - which * OUT;
				rb[q] = load8(g.b[which] + (uint64_t)col * g.ldb + t0 + chunk * 8, col < g.cols ? left - chunk * 8 : 0);
			} else { const uint32_t c = c0 + chunk * 8; rb[q] = load8(g.b[seg] + (uint64_t)(t0 + line) * g.ldb + c, line < left ? (int)g.cols - (int)c : 0); }
		}
	};
	if (t_begin < t_end) load(t_begin);
	for (uint32_t t = t_begin; t < t_end; ++t) {
#pragma unroll
		for (int q = 0; q < NA; ++q) *(T8*)(lds_a + (q * THREADS + tid) * 8) = ra[q];
#pragma unroll
		for (int q = 0; q < NB; ++q) *(T8*)(lds_b + (q * THREADS + tid) * 8) = rb[q];
		__syncthreads();
		if (t + 1 < t_end) load(t + 1);
#pragma unroll
		for (int ks = 0; ks < TK / 32; ++ks) {
			T8 fa[FR], fb[FC];
#pragma unroll
			for (int i = 0; i < FR; ++i) fa[i] = TA::read(lds_a, wr * (BR / WR) + i * 16, 0, ks, gq, li);
#pragma unroll
			for (int j = 0; j < FC; ++j) fb[j] = TB::read(lds_b, pair_at(j / 2), j & 1, ks, gq, li);
#pragma unroll
			for (int i = 0; i < FR; ++i)
#pragma unroll
				for (int j = 0; j < FC; ++j) acc[i][j] = mfma(fb[j], fa[i], acc[i][j]);
		}
		__syncthreads();
	}
	// epilogue: lane owns row r and, per pair of fragments, the 8 columns from c
#pragma unroll
	for (int i = 0; i < FR; ++i) {
		const uint32_t r = r0 + wr * (BR / WR) + i * 16 + li;
		if (r >= g.rows) continue;
#pragma unroll
		for (int p = 0; p < (EPI == EPI_GATED ? FC / 4 : FC / 2); ++p) {
			const uint32_t c = c0 + pair_at(p) + gq * 8;
			if (c >= g.cols) continue;
			const int n = (int)min(8u, g.cols - c);
			float z[8];
#pragma unroll
			for (int e = 0; e < 8; ++e) z[e] = acc[i][2 * p + e / 4][e & 3];
			if constexpr (EPI == EPI_PARTIAL) {
				float* o = g.partial + (((uint64_t)split * g.problems + problem) * g.rows + r) * up8(g.cols) + c; // (lines are padded to 8: always whole)
				*(f4v*)o = f4v{z[0], z[1], z[2], z[3]}; *(f4v*)(o + 4) = f4v{z[4], z[5], z[6], z[7]};
			} else if constexpr (EPI == EPI_STORE) {
				T8 o;
#pragma unroll
				for (int e = 0; e < 8; ++e) o[e] = (T)z[e];
				store8(g.c[problem] + (uint64_t)r * g.ldc + c, o, n);
			} else {
				T8 o, s;
				if (g.bias[0]) { const T8 b = load8(g.bias[0] + c, n);
#pragma unroll
					for (int e = 0; e < 8; ++e) z[e] += (float)b[e]; }
				if (g.pre[0]) {
#pragma unroll
					for (int e = 0; e < 8; ++e) s[e] = (T)z[e];
					store8(g.pre[0] + (uint64_t)r * g.ld_pre + c, s, n);
				}
				if constexpr (EPI == EPI_LINEAR) {
					T8 res{};
					if (g.residual) res = load8(g.residual + (uint64_t)r * g.ld_residual + c, n);
#pragma unroll
					for (int e = 0; e < 8; ++e) { const float v = act_value(g.act, z[e]); o[e] = (T)(g.residual ? v + (float)res[e] : v); }
				} else {
					float u[8];
#pragma unroll
					for (int e = 0; e < 8; ++e) u[e] = acc[i][FC / 2 + 2 * p + e / 4][e & 3];
					if (g.bias[1]) { const T8 b = load8(g.bias[1] + c, n);
#pragma unroll
						for (int e = 0; e < 8; ++e) u[e] += (float)b[e]; }
					if (g.pre[1]) {
#pragma unroll
						for (int e = 0; e < 8; ++e) s[e] = (T)u[e];
						store8(g.pre[1] + (uint64_t)r * g.ld_pre + c, s, n);
					}
#pragma unroll
					for (int e = 0; e < 8; ++e) o[e] = (T)(act_value(g.act, z[e]) * u[e]);
				}
				store8(g.c[0] + (uint64_t)r * g.ldc + c, o, n);
			}
		}
	}
}

// G = dY * act'(Z) (gated: [dH * Zu * act'(Zg) | dH * act(Zg)]), lines padded with zeros to multiples of 8 columns, rounded once to the layer's type (the matrix
// instructions take 16-bit operands; the relative error of a rounding, 2^-12 / 2^-9 on average, is that of the result's own), and its column sums (in 32 bits,
// one line per block of rows, before the rounding).  Memory bound.  32 x 8 threads: 256 columns x 8 rows at a time.
struct GradArgs { uint32_t rows, cols; int act; const T* dy; uint64_t ld_dy; const T* pre[2]; uint64_t ld_pre; T* out; uint64_t ld_out; float* bias_partial; uint32_t rows_per_block; };
template <bool GATED> __global__ __launch_bounds__(256) void k_output_grad(GradArgs g) {
	const uint32_t cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 256 + cx * 8, pc = up8(g.cols);
	const uint32_t end = min(g.rows, (blockIdx.y + 1) * g.rows_per_block);
	float sum[GATED ? 2 : 1][8] = {};
	if (c < g.cols) {
		const int n = (int)min(8u, g.cols - c);
		for (uint32_t r = blockIdx.y * g.rows_per_block + ry; r < end; r += 8) {
			const T8 dy = load8(g.dy + (uint64_t)r * g.ld_dy + c, n);
			T8 z{}, u{}, o, o2;
			if (g.pre[0]) z = load8(g.pre[0] + (uint64_t)r * g.ld_pre + c, n);
			if (GATED) u = load8(g.pre[1] + (uint64_t)r * g.ld_pre + c, n);
#pragma unroll
			for (int e = 0; e < 8; ++e) {
				float value, slope;
				act_value_slope(g.act, (float)z[e], value, slope);
				const float v = e < n && slope != 0.f ? (GATED ? (float)dy[e] * (float)u[e] * slope : (float)dy[e] * slope) : 0.f; // (a closed unit passes nothing, whatever arrives)
				sum[0][e] += v; o[e] = (T)v;
				if (GATED) { const float w = e < n ? (float)dy[e] * value : 0.f; sum[GATED ? 1 : 0][e] += w; o2[e] = (T)w; }
			}
			if (g.out) {
				*(T8*)(g.out + (uint64_t)r * g.ld_out + c) = o;
				if (GATED) *(T8*)(g.out + (uint64_t)r * g.ld_out + pc + c) = o2;
			}
		}
	}
	if (!g.bias_partial) return;
	__shared__ float red[8][256 + 8];
#pragma unroll
	for (int k = 0; k < (GATED ? 2 : 1); ++k) {
		__syncthreads();
#pragma unroll
		for (int e = 0; e < 8; ++e) red[ry][cx * 8 + e] = sum[k][e];
		__syncthreads();
		float s = 0.f;
#pragma unroll
		for (int y = 0; y < 8; ++y) s += red[y][threadIdx.x];
		const uint32_t col = blockIdx.x * 256 + threadIdx.x;
		if (col < g.cols) g.bias_partial[((uint64_t)blockIdx.y * (GATED ? 2 : 1) + k) * g.cols + col] = s;
	}
}
// dbias = sum of the blocks' column sums, in their order
__global__ __launch_bounds__(256) void k_bias_grad(const float* partial, uint32_t blocks, uint32_t cols, uint32_t problems, T* out0, T* out1) {
	__shared__ float red[8][32];
	const uint32_t cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx, k = blockIdx.y;
	float s = 0.f;
	if (c < cols) {
#pragma unroll 4
		for (uint32_t b = ry; b < blocks; b += 8) s += partial[((uint64_t)b * problems + k) * cols + c];
	}
	red[ry][cx] = s;
	__syncthreads();
	if (ry == 0 && c < cols) {
		float t = 0.f;
#pragma unroll
		for (int y = 0; y < 8; ++y) t += red[y][cx];
		T* out = k ? out1 : out0;
		if (out) out[c] = (T)t;
	}
}
// C = sum over the splits, in their order, rounded once
__global__ __launch_bounds__(256) void k_join_splits(const float* partial, uint32_t splits, uint32_t problems, uint32_t rows, uint32_t cols, T* c0, T* c1, uint64_t ldc) {
	const uint32_t cc = up8(cols) / 8, problem = blockIdx.y;
	const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
	if (id >= (uint64_t)rows * cc) return;
	const uint32_t r = (uint32_t)(id / cc), c = (uint32_t)(id % cc) * 8;
	f4v s0{}, s1{};
#pragma unroll 4
	for (uint32_t k = 0; k < splits; ++k) {
		const float* p = partial + (((uint64_t)k * problems + problem) * rows + r) * (cc * 8) + c;
		s0 += *(const f4v*)p; s1 += *(const f4v*)(p + 4);
	}
	T8 o;
#pragma unroll
	for (int e = 0; e < 4; ++e) { o[e] = (T)s0[e]; o[e + 4] = (T)s1[e]; }
	store8((problem ? c1 : c0) + (uint64_t)r * ldc + c, o, (int)min(8u, cols - c));
}

uint32_t div_up(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }
template <bool A_T, bool B_T, int EPI> void launch_gemm(hipStream_t s, GemmArgs& g) {
	constexpr int BR = 128, BC = 128, OUT = EPI == EPI_GATED ? BC / 2 : BC;
	hipLaunchKernelGGL((k_gemm<BR, BC, 2, 2, A_T, B_T, EPI>), dim3(div_up(g.rows, BR) * div_up(g.cols, OUT), g.problems, g.splits), dim3(256), 0, s, g);
}
} // namespace

void DENSE_NAME(launch_dense_forward)(hipStream_t s, const DenseArgs& d) {
	if (!d.m || !d.n) return;
	GemmArgs g{};
	g.a = (const T*)d.x; g.lda = d.x_stride; g.ldb = d.w_stride;
	g.rows = d.m; g.cols = d.n; g.steps = d.k; g.segments = 1; g.problems = 1; g.splits = 1; g.chunks_per_split = div_up(d.k, TK);
	for (int i = 0; i < 2; ++i) { g.b[i] = (const T*)d.w[i]; g.bias[i] = (const T*)d.bias[i]; g.pre[i] = (T*)d.pre[i]; }
	g.c[0] = (T*)d.y; g.ldc = d.y_stride; g.act = d.act; g.residual = (const T*)d.residual; g.ld_residual = d.residual_stride; g.ld_pre = d.pre_stride;
	if (d.gated) launch_gemm<true, true, EPI_GATED>(s, g); else launch_gemm<true, true, EPI_LINEAR>(s, g);
}
void DENSE_NAME(launch_dense_backward)(hipStream_t s, const DenseArgs& d) {
	const DensePlan p = dense_plan(d.m, d.n, d.k, d.gated);
	const uint32_t problems = d.gated ? 2 : 1;
	char* ws = (char*)d.workspace;
	const bool bias = d.dbias[0] || d.dbias[1];
	const bool identity = !d.gated && d.act == NGP_ACT_NONE; // G is dY as it stands
	const bool products = d.dx || d.dw[0] || d.dw[1];
	const T* G = (const T*)d.dy; uint64_t ldg = d.dy_stride;
	if ((!identity && products) || bias) {
		GradArgs a{};
		a.rows = d.m; a.cols = d.n; a.act = d.act; a.dy = (const T*)d.dy; a.ld_dy = d.dy_stride; a.pre[0] = (const T*)d.pre[0]; a.pre[1] = (const T*)d.pre[1]; a.ld_pre = d.pre_stride;
		if (identity) a.pre[0] = nullptr;
		a.out = products && !identity ? (T*)(ws + p.grad) : nullptr; a.ld_out = (uint64_t)up8(d.n) * problems; a.bias_partial = bias ? (float*)(ws + p.bias) : nullptr; a.rows_per_block = p.rows_per_block;
		if (a.out) { G = a.out; ldg = a.ld_out; }
		const dim3 grid(div_up(d.n, 256), p.row_blocks);
		if (d.m && d.n) {
			if (d.gated) hipLaunchKernelGGL(k_output_grad<true>, grid, dim3(256), 0, s, a); else hipLaunchKernelGGL(k_output_grad<false>, grid, dim3(256), 0, s, a);
		}
		if (bias && d.n) hipLaunchKernelGGL(k_bias_grad, dim3(div_up(d.n, 32), problems), dim3(256), 0, s, (const float*)(ws + p.bias), p.row_blocks, d.n, problems, (T*)d.dbias[0], (T*)d.dbias[1]);
	}
	if (d.dx && d.m && d.k) {
		GemmArgs g{};
		g.a = G; g.lda = ldg; g.a_segment = up8(d.n); g.segments = problems; g.b[0] = (const T*)d.w[0]; g.b[1] = (const T*)d.w[1]; g.ldb = d.w_stride;
		g.rows = d.m; g.cols = d.k; g.steps = d.n; g.problems = 1; g.splits = 1; g.chunks_per_split = div_up(d.n, TK) * problems; g.c[0] = (T*)d.dx; g.ldc = d.dx_stride;
		launch_gemm<true, false, EPI_STORE>(s, g);
	}
	if ((d.dw[0] || d.dw[1]) && d.n && d.k) {
		GemmArgs g{};
		g.a = G; g.lda = ldg; g.a_problem = up8(d.n); g.problems = problems; g.b[0] = g.b[1] = (const T*)d.x; g.ldb = d.x_stride;
		g.rows = d.n; g.cols = d.k; g.steps = d.m; g.segments = 1; g.c[0] = (T*)d.dw[0]; g.c[1] = (T*)d.dw[1]; g.ldc = d.dw_stride;
		g.splits = p.splits; g.chunks_per_split = div_up(div_up(d.m, TK), p.splits);
		if (p.splits > 1) {
			g.partial = (float*)(ws + p.partial);
			launch_gemm<false, false, EPI_PARTIAL>(s, g);
			hipLaunchKernelGGL(k_join_splits, dim3(div_up((uint64_t)d.n * up8(d.k) / 8, 256), problems), dim3(256), 0, s, g.partial, p.splits, problems, d.n, d.k, g.c[0], g.c[1], g.ldc);
		} else launch_gemm<false, false, EPI_STORE>(s, g);
	}
}
} // namespace ngp
