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
#include <type_traits>
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
// the same with the sums held in place in accumulation registers (the compiler, left to itself, moves 256 of them about and spills).  Whoever reads the sums with
// other instructions waits first: settle().  The operands come from LDS reads alone (a vector instruction that wrote one would need two wait states in front).  The compiler does not see
// these instructions' hazards: tests/test_dense_instructions.py looks for them in the built library, and has to be run whenever this file or the compiler changes.
__device__ inline void mfma_in_place(T8 a, T8 b, f4v& c) {
#ifdef DENSE_BF16
	asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
#else
	asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
#endif
}
template <int N, int M> __device__ inline void settle(f4v (&c)[N][M]) { // more wait states than the longest matrix instruction needs, in front of every later use of c
	asm volatile("s_nop 15\n\ts_nop 15" ::);
#pragma unroll
	for (int i = 0; i < N; ++i)
#pragma unroll
		for (int j = 0; j < M; ++j) asm volatile("" : "+a"(c[i][j]));
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
// The same where p may lie between two dwords: memory answers 16 bytes from an odd element on two to three times slower (1 x 4097 inputs, 8192 outputs: 29.6 us against 13.1), so the dwords
// that hold them are read, five where p is odd.  (A dword with one element of the matrix in it can be read.)
__device__ inline T8 load8_odd(const T* p) {
	const uint32_t* q = (const uint32_t*)((uintptr_t)p & ~(uintptr_t)3);
	const bool odd = (uintptr_t)p & 2;
	uint32_t v[4];
	__builtin_memcpy(v, q, 16);
	const uint32_t t = q[odd ? 4 : 3];
	const uint32_t r[4] = {odd ? __builtin_amdgcn_alignbit(v[1], v[0], 16) : v[0], odd ? __builtin_amdgcn_alignbit(v[2], v[1], 16) : v[1],
		odd ? __builtin_amdgcn_alignbit(v[3], v[2], 16) : v[2], odd ? __builtin_amdgcn_alignbit(t, v[3], 16) : v[3]};
	T8 o;
	__builtin_memcpy(&o, r, 16);
	return o;
}
// elements c .. c + 7 of a line of `width` >= 8 out of the 16 bytes that were read at min(c, width - 8): moved down, zeros behind the line's end, without a branch
__device__ inline T8 shift8(T8 raw, int c, int width) {
	const int by = c - min(c, width - 8), d = by >> 1;
	uint32_t v[4], t[4];
	__builtin_memcpy(v, &raw, 16);
	t[0] = d & 2 ? v[2] : v[0]; t[1] = d & 2 ? v[3] : v[1]; t[2] = d & 2 ? 0 : v[2]; t[3] = d & 2 ? 0 : v[3];
	v[0] = d & 1 ? t[1] : t[0]; v[1] = d & 1 ? t[2] : t[1]; v[2] = d & 1 ? t[3] : t[2]; v[3] = d & 1 ? 0 : t[3];
	const bool odd = by & 1, none = by >= 8;
	t[0] = odd ? __builtin_amdgcn_alignbit(v[1], v[0], 16) : v[0]; t[1] = odd ? __builtin_amdgcn_alignbit(v[2], v[1], 16) : v[1];
	t[2] = odd ? __builtin_amdgcn_alignbit(v[3], v[2], 16) : v[2]; t[3] = odd ? v[3] >> 16 : v[3];
	T8 r;
#pragma unroll
	for (int i = 0; i < 4; ++i) t[i] = none ? 0 : t[i];
	__builtin_memcpy(&r, t, 16);
	return r;
}
// COUNT chunks of 8 elements of lines of one width, all on their way together: at(q, line) gives the line and returns the column.  Lines of 8 elements and more are read in whole chunks
// (at min(column, width - 8): shift8 puts them right later), shorter ones element by element.  (By the dword, as above, tiles of odd lines ran 15 % longer: they wait for other things.)
template <int COUNT, typename F> __device__ inline void load_chunks(T8* out, int width, F&& at) {
	if (width >= 8) {
#pragma unroll
		for (int q = 0; q < COUNT; ++q) { const T* line; const int c = at(q, line); out[q] = load8(line + min(c, width - 8)); }
	} else {
#pragma unroll
		for (int q = 0; q < COUNT; ++q) { const T* line; const int c = at(q, line); out[q] = load8(line + c, width - c); }
	}
}
// `streamed`: past the caches
__device__ inline void store8(T* p, T8 v, int n, bool streamed = false) {
	typedef float any4 __attribute__((ext_vector_type(4), aligned(2)));
	if (streamed && n >= 8) { __builtin_nontemporal_store(__builtin_bit_cast(f4v, v), (any4*)p); return; }
	if (n >= 8) { __builtin_memcpy(p, &v, 16); return; }
#pragma unroll
	for (int i = 0; i < 8; ++i) if (i < n) p[i] = v[i];
}

// a barrier that waits for LDS alone: loads and stores stay on their way
__device__ inline void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---- activations: values and derivatives in 32 bits.  1 / (1 + e^-z) through v_exp_f32 / v_rcp_f32 (1 ulp each): far below the 16-bit rounding of the result
__device__ inline float logistic(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
// the normal distribution function and e^(-z^2/2).  Lower tail at -|z|: t Q(t) e^(-z^2/2) with t = 1 / (1 + 0.35 |z|), Q = a least-squares fit (reweighted towards the largest relative
// error) of 0.5 erfcx(|z| / sqrt 2) / t over |z| < 14.5: 3.2e-8 relative, 2.8e-7 in 32 bits, in both tails; erfcf costs the epilogue three times as much
__device__ inline float normal_cdf(float z, float& e) {
	const float u = fabsf(z), t = __builtin_amdgcn_rcpf(fmaf(0.35f, u, 1.f));
	e = __builtin_amdgcn_exp2f(-0.72134752f * z * z);
	float q = -0.029158229008316994f;
	q = fmaf(q, t, 0.1440325528383255f); q = fmaf(q, t, -0.25584226846694946f); q = fmaf(q, t, 0.1593232899904251f); q = fmaf(q, t, -0.02321472205221653f);
	q = fmaf(q, t, 0.10555345565080643f); q = fmaf(q, t, 0.11982106417417526f); q = fmaf(q, t, 0.13986355066299438f); q = fmaf(q, t, 0.139621302485466f);
	q *= t * e;
	return z < 0.f ? q : 1.f - q;
}
__device__ inline void act_value8(int act, float z[8]) { // (one branch for 8 values)
#define EACH for (int e = 0; e < 8; ++e)
	switch (act) {
		case NGP_ACT_RELU: EACH z[e] = z[e] < 0.f ? 0.f : z[e]; break; // (NaN stays NaN)
		case NGP_ACT_LOGISTIC: EACH z[e] = logistic(z[e]); break;
		case NGP_ACT_EXPONENTIAL: EACH z[e] = __expf(z[e]); break;
		case NGP_ACT_SILU: EACH z[e] *= logistic(z[e]); break;
		case NGP_ACT_GELU: EACH { float x; z[e] *= normal_cdf(z[e], x); } break;
		default: break;
	}
}
// f(activation as a constant): one branch for a whole loop, whose code then stays small (an epilogue with the branch in every row ran 2.5 times longer, waiting for instructions)
template <typename F> __device__ inline void with_act(int act, F&& f) {
	switch (act) {
		case NGP_ACT_RELU: f(std::integral_constant<int, NGP_ACT_RELU>()); break;
		case NGP_ACT_LOGISTIC: f(std::integral_constant<int, NGP_ACT_LOGISTIC>()); break;
		case NGP_ACT_EXPONENTIAL: f(std::integral_constant<int, NGP_ACT_EXPONENTIAL>()); break;
		case NGP_ACT_SILU: f(std::integral_constant<int, NGP_ACT_SILU>()); break;
		case NGP_ACT_GELU: f(std::integral_constant<int, NGP_ACT_GELU>()); break;
		default: f(std::integral_constant<int, NGP_ACT_NONE>()); break;
	}
}
// G of 8 outputs: dY act'(Z); gated: dY Zu act'(Zg) and dY act(Zg).  Zeros give zeros.
template <bool GATED> __device__ inline void output_grad8(int act, const T8& dy, const T8& zt, const T8& ut, float g[8], float g2[8]) {
	float d[8], m[8], z[8];
	EACH { d[e] = (float)dy[e]; z[e] = (float)zt[e]; m[e] = GATED ? d[e] * (float)ut[e] : d[e]; }
	switch (act) {
		case NGP_ACT_RELU: EACH { g[e] = z[e] > 0.f ? m[e] : 0.f; if (GATED) g2[e] = z[e] > 0.f ? d[e] * z[e] : 0.f; } break; // (a closed unit passes nothing, whatever arrives)
		case NGP_ACT_LOGISTIC: EACH { const float x = __expf(-fabsf(z[e])), r = __builtin_amdgcn_rcpf(1.f + x); g[e] = m[e] * (x * r * r); if (GATED) g2[e] = d[e] * (z[e] < 0.f ? x * r : r); } break; // (p (1 - p) would lose its bits where p is near 1)
		case NGP_ACT_EXPONENTIAL: EACH { const float p = __expf(z[e]); g[e] = m[e] * p; if (GATED) g2[e] = d[e] * p; } break;
		case NGP_ACT_SILU: EACH { const float p = logistic(z[e]); g[e] = m[e] * (p * fmaf(z[e], 1.f - p, 1.f)); if (GATED) g2[e] = d[e] * (z[e] * p); } break;
		case NGP_ACT_GELU: EACH { float x; const float c = normal_cdf(z[e], x); g[e] = m[e] * fmaf(z[e] * 0.39894228f, x, c); if (GATED) g2[e] = d[e] * (z[e] * c); } break;
		default: EACH { g[e] = m[e]; if (GATED) g2[e] = d[e] * z[e]; } break;
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

enum { EPI_LINEAR, EPI_GATED, EPI_STORE /* as it is; partial sums where they are split */, EPI_PARTIAL, EPI_PARTIAL2 /* of both projections */ };
struct GemmArgs {
	const T* a; const T* b[2]; uint64_t lda, ldb;
	uint32_t rows, cols, steps;      // C is rows x cols; the sum runs over `segments` pieces of `steps`
	uint32_t segments; uint64_t a_segment; // A's next piece is a_segment elements further (dX of a gated layer, second terms of G), B's is the other one of b
	uint64_t a_problem; uint32_t problems; // dW of a gated layer: two products with the same B (A a_problem elements further)
	uint32_t splits, chunks_per_split;     // the sum is split over blocks: partial sums to `partial`
	T* c[2]; uint64_t ldc;
	float* partial;                        // [split][problem][rows][cols8]
	int act; const T* bias[2]; const T* residual; uint64_t ld_residual; T* pre[2]; uint64_t ld_pre;
	bool streamed; // a forward pass's outputs are more than the caches hold: written past them
};
__host__ __device__ inline uint32_t up8(uint32_t v) { return (v + 7) & ~7u; }

// 8 sums (gated: z of the gate, u of the up projection) to pre-activations and outputs
template <int EPI> __device__ inline void outputs8(float z[8], float u[8], const T8& bias0, const T8& bias1, const T8* residual, int act, T8& pre0, T8& pre1, T8& o) {
	EACH { z[e] += (float)bias0[e]; pre0[e] = (T)z[e]; }
	act_value8(act, z);
	if constexpr (EPI == EPI_LINEAR) {
		if (residual) { EACH z[e] += (float)(*residual)[e]; }
		EACH o[e] = (T)z[e];
	} else EACH { u[e] += (float)bias1[e]; pre1[e] = (T)u[e]; o[e] = (T)(z[e] * u[e]); }
}
// What becomes of 8 consecutive sums of row r from column c on (gated: z of the gate, u of the up projection), n <= 8 of them inside C.  Biases and the residual come as values: a caller
// with several rows loads them ahead.
template <int EPI> __device__ inline void epilogue8(const GemmArgs& g, uint32_t problem, uint32_t split, uint32_t r, uint32_t c, int n, float z[8], float u[8], const T8& bias0, const T8& bias1, const T8& residual, int act, bool streamed = false) {
	T8 o, s;
	if constexpr (EPI == EPI_PARTIAL || EPI == EPI_PARTIAL2) {
		const uint32_t parts = EPI == EPI_PARTIAL2 ? 2 : g.problems;
		float* q = g.partial + (((uint64_t)split * parts + problem) * g.rows + r) * up8(g.cols) + c; // (lines are padded to 8: always whole)
		*(f4v*)q = f4v{z[0], z[1], z[2], z[3]}; *(f4v*)(q + 4) = f4v{z[4], z[5], z[6], z[7]};
		if constexpr (EPI == EPI_PARTIAL2) { q += (uint64_t)g.rows * up8(g.cols); *(f4v*)q = f4v{u[0], u[1], u[2], u[3]}; *(f4v*)(q + 4) = f4v{u[4], u[5], u[6], u[7]}; }
		return;
	}
	if constexpr (EPI == EPI_STORE) {
		if (g.splits > 1) { epilogue8<EPI_PARTIAL>(g, problem, split, r, c, n, z, u, bias0, bias1, residual, act); return; }
		EACH o[e] = (T)z[e];
		store8(g.c[problem] + (uint64_t)r * g.ldc + c, o, n);
		return;
	}
	EACH z[e] += (float)bias0[e];
	if (g.pre[0]) { EACH s[e] = (T)z[e]; store8(g.pre[0] + (uint64_t)r * g.ld_pre + c, s, n, streamed); }
	act_value8(act, z);
	if constexpr (EPI == EPI_LINEAR) {
		if (g.residual) { EACH z[e] += (float)residual[e]; }
		EACH o[e] = (T)z[e];
	} else {
		EACH u[e] += (float)bias1[e];
		if (g.pre[1]) { EACH s[e] = (T)u[e]; store8(g.pre[1] + (uint64_t)r * g.ld_pre + c, s, n, streamed); }
		EACH o[e] = (T)(z[e] * u[e]);
	}
	store8(g.c[0] + (uint64_t)r * g.ldc + c, o, n, streamed);
}
template <int EPI> constexpr bool GATED_TILE = EPI == EPI_GATED || EPI == EPI_PARTIAL2; // the tile's columns are gate and up outputs
template <int EPI> __device__ inline T8 bias8(const GemmArgs& g, int k, uint32_t c, int n) { return (EPI == EPI_LINEAR || EPI == EPI_GATED) && g.bias[k] && n > 0 ? load8(g.bias[k] + c, n) : T8{}; }
template <int EPI> __device__ inline T8 residual8(const GemmArgs& g, uint32_t r, uint32_t c, int n) { return EPI == EPI_LINEAR && g.residual && n > 0 ? load8(g.residual + (uint64_t)r * g.ld_residual + c, n) : T8{}; }

// Consecutive blocks go to the 8 dies in turn, each with an L2 of its own: give every die one contiguous run of the work, ordered by piece of the sum, product, strips of 8 row
// tiles, so that its blocks share operands.  (Tiles of one piece on four dies: every operand line missed four L2s, dW of 2^18 samples 86 instead of 60 us.)
struct Work { uint32_t row, col, problem, split; };
__device__ inline Work work_of(const GemmArgs& g, uint32_t index, uint32_t n, uint32_t row_tiles, uint32_t col_tiles) { // block `index` of the n that share this product
	const uint32_t die = index & 7, per = n >> 3, rest = n & 7, t = die * per + min(die, rest) + (index >> 3), tiles = row_tiles * col_tiles;
	const uint32_t which = t / tiles, in = t - which * tiles, strip = 8 * col_tiles, s = in / strip, k = in - s * strip, rows = min(8u, row_tiles - s * 8);
	return {s * 8 + k % rows, k / rows, which % g.problems, which / g.problems};
}
// Staged through registers: operands at odd addresses, or with lines that are no whole 16-byte pieces, any size from 1.  The way to LDS bounds it (4096 x 4096 of 1000 inputs at an odd
// stride: 70 us, 480 TFLOP/s, half the rate of async_tile's), at 128 x 128 so that two blocks a compute unit cover each other's barriers.
// C tile BR x BC by WR x WC wavefronts; each owns (BR / WR) x (BC / WC) as 16 x 16 fragments (matrix instruction 16x16x32, C^T: a lane holds one row of C and 4 columns
// of each fragment).  EPI_GATED: the tile's columns are BC / 2 gate outputs and the same BC / 2 up outputs, every wavefront owns both of its columns.
template <int BR, int BC, int WR, int WC, bool A_T, bool B_T, int EPI> __device__ inline void any_tile(const GemmArgs& g, T* lds_a, T* lds_b, uint32_t index, uint32_t count) {
	typedef Tile<BR, A_T, false> TA; typedef Tile<BC, B_T, true> TB;
	constexpr int THREADS = 64 * WR * WC, FR = BR / WR / 16, FC = BC / WC / 16, NA = TA::N_SLOTS / THREADS, NB = TB::N_SLOTS / THREADS;
	constexpr int OUT = GATED_TILE<EPI> ? BC / 2 : BC; // columns of C per tile
	static_assert(FC % (GATED_TILE<EPI> ? 4 : 2) == 0, "pairs of fragments");
	const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wr = wave / WC, wc = wave % WC, gq = lane >> 4, li = lane & 15;
	const Work w = work_of(g, index, count, (g.rows + BR - 1) / BR, (g.cols + OUT - 1) / OUT);
	const uint32_t r0 = w.row * BR, c0 = w.col * OUT, problem = w.problem, split = w.split;
	const T* a = g.a + problem * g.a_problem;
	const uint32_t chunks_per_segment = (g.steps + TK - 1) / TK, n_chunks = chunks_per_segment * g.segments;
	const uint32_t t_begin = split * g.chunks_per_split, t_end = min(n_chunks, t_begin + g.chunks_per_split);
	auto pair_at = [&](int p) -> int { // first column (in the B tile) of fragment pair p of this wavefront
		if (GATED_TILE<EPI>) return (p >= FC / 4 ? OUT : 0) + (int)wc * (OUT / WC) + (p % (FC / 4)) * 32;
		return (int)wc * (BC / WC) + p * 32;
	};
	f4v acc[FR][FC];
#pragma unroll
	for (int i = 0; i < FR; ++i)
#pragma unroll
		for (int j = 0; j < FC; ++j) acc[i][j] = f4v{0.f, 0.f, 0.f, 0.f};
	T8 ra[NA], rb[NB];
	// An operand's share of a chunk: `extent` of the matrix from e0 on, `left` steps.  What lies outside the matrix only reaches sums that are dropped, so lines and columns are clamped
	// there; beyond the sum's last step both operands are zero (put right on the way to LDS, when the loads have arrived).
	auto load_operand = [&](auto tile_c, auto contig_c, T8* out, auto count_c, auto&& matrix, uint64_t ld, uint32_t e0, uint32_t extent, uint32_t t0, int left) {
		typedef decltype(tile_c) TX; constexpr bool CONTIG = decltype(contig_c)::value; constexpr int COUNT = decltype(count_c)::value;
		load_chunks<COUNT>(out, CONTIG ? (int)g.steps : (int)extent, [&](int q, const T*& p) -> int {
			const int slot = q * THREADS + tid, line = slot / TX::SLOTS, chunk = TX::source(line, slot % TX::SLOTS);
			uint32_t in_tile = line; // (CONTIG)
			const T* base = matrix(in_tile);
			p = CONTIG ? base + (uint64_t)min(e0 + in_tile, extent - 1) * ld : base + (uint64_t)(t0 + min(line, left - 1)) * ld;
			return (CONTIG ? (int)t0 : (int)e0) + chunk * 8;
		});
	};
	auto to_lds = [&](auto tile_c, auto contig_c, T8* in, auto count_c, T* lds, uint32_t e0, uint32_t extent, uint32_t t0, int left) {
		typedef decltype(tile_c) TX; constexpr bool CONTIG = decltype(contig_c)::value; constexpr int COUNT = decltype(count_c)::value;
		const int width = CONTIG ? (int)g.steps : (int)extent;
		if (width >= 8 && (CONTIG ? left < TK : e0 + TX::ELEMS / TK > extent)) {
#pragma unroll
			for (int q = 0; q < COUNT; ++q) {
				const int slot = q * THREADS + tid, chunk = TX::source(slot / TX::SLOTS, slot % TX::SLOTS);
				in[q] = shift8(in[q], (CONTIG ? (int)t0 : (int)e0) + chunk * 8, width);
			}
		}
		if (!CONTIG && left < TK) {
#pragma unroll
			for (int q = 0; q < COUNT; ++q) if ((q * THREADS + (int)tid) / TX::SLOTS >= left) in[q] = T8{};
		}
#pragma unroll
		for (int q = 0; q < COUNT; ++q) *(T8*)(lds + (q * THREADS + tid) * 8) = in[q];
	};
	uint32_t t0 = 0; int left = 0; // of the chunk in the registers
	auto load = [&](uint32_t t) {
		const uint32_t seg = t / chunks_per_segment;
		t0 = (t - seg * chunks_per_segment) * TK;
		left = (int)min((uint32_t)TK, g.steps - t0);
		load_operand(TA{}, std::integral_constant<bool, A_T>(), ra, std::integral_constant<int, NA>(), [&](uint32_t&) { return a + seg * g.a_segment; }, g.lda, r0, g.rows, t0, left);
		load_operand(TB{}, std::integral_constant<bool, B_T>(), rb, std::integral_constant<int, NB>(), [&](uint32_t& line) -> const T* {
			if (!B_T) return g.b[seg & 1];
			const uint32_t which = GATED_TILE<EPI> && line >= OUT; // (gated: the tile's second half is the up projection's)
			line -= which * OUT;
			return which ? g.b[1] : g.b[0];
		}, g.ldb, c0, g.cols, t0, left);
	};
	if (t_begin < t_end) load(t_begin);
	for (uint32_t t = t_begin; t < t_end; ++t) {
		to_lds(TA{}, std::integral_constant<bool, A_T>(), ra, std::integral_constant<int, NA>(), lds_a, r0, g.rows, t0, left);
		to_lds(TB{}, std::integral_constant<bool, B_T>(), rb, std::integral_constant<int, NB>(), lds_b, c0, g.cols, t0, left);
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
		for (int p = 0; p < (GATED_TILE<EPI> ? FC / 4 : FC / 2); ++p) {
			const uint32_t c = c0 + pair_at(p) + gq * 8;
			if (c >= g.cols) continue;
			const int n = (int)min(8u, g.cols - c);
			float z[8], u[8];
			EACH { z[e] = acc[i][2 * p + e / 4][e & 3]; u[e] = GATED_TILE<EPI> ? acc[i][(GATED_TILE<EPI> ? FC / 2 : 0) + 2 * p + e / 4][e & 3] : 0.f; }
			epilogue8<EPI>(g, problem, split, r, c, n, z, u, bias8<EPI>(g, 0, c, n), bias8<EPI>(g, 1, c, n), residual8<EPI>(g, r, c, n), g.act);
		}
	}
}

template <bool A_T, bool B_T, int EPI> __global__ __launch_bounds__(256) void k_gemm(GemmArgs g) {
	__shared__ __attribute__((aligned(16))) T lds[2][128 * TK];
	any_tile<128, 128, 2, 2, A_T, B_T, EPI>(g, lds[0], lds[1], blockIdx.x, gridDim.x);
}
// dX and dW, which do not wait for each other, side by side; the blocks with the longer sums begin
struct Share { bool x; uint32_t index, count; };
__device__ inline Share share_of(uint32_t blocks_x, uint32_t blocks_w, bool w_first) {
	const uint32_t b = blockIdx.x, first = w_first ? blocks_w : blocks_x;
	const bool x = (b < first) != w_first;
	return {x, b < first ? b : b - first, x ? blocks_x : blocks_w};
}
__global__ __launch_bounds__(256) void k_products(GemmArgs x, GemmArgs w, uint32_t blocks_x, uint32_t blocks_w, bool w_first) {
	__shared__ __attribute__((aligned(16))) T lds[2][128 * TK];
	const Share s = share_of(blocks_x, blocks_w, w_first);
	if (s.x) any_tile<128, 128, 2, 2, true, false, EPI_STORE>(x, lds[0], lds[1], s.index, s.count);
	else any_tile<128, 128, 2, 2, false, false, EPI_STORE>(w, lds[0], lds[1], s.index, s.count);
}

// ---- operands whose lines are whole 16-byte pieces: straight from memory to LDS (buffer loads with the LDS bit; what lies outside the matrix arrives as zero) in units of 64 steps
// of one operand (whole cache lines: 64-byte pieces ask the L2 twice as often, 65 instead of 70 % of the matrix rate).  UNITS of B and one more of A are in LDS: the one in use, and
// what is on its way.  At 256 x 256 that is 160 KB with UNITS = 2 (about 2000 clocks ahead); 128 x 128 tiles take a quarter of the time a unit and get UNITS = 4 where a compute
// unit has one block to itself (144 KB), 2 where it has two.  The matrix instructions run through a unit in two halves of 32 steps; A fragments
// come in three ahead of their use, the next half's B fragments into a second set of registers.  4 wavefronts with 128 x 128 of C each: 2 x 128 fragment rows per 128 x 128
// products is what LDS can deliver beside the incoming units (96 of the 128 bytes a clock; with 8 wavefronts of 128 x 64 it would be all of them).
// Bound by the matrix instructions: 8192 x 8192 x 8192 765 us, 1440 TFLOP/s, what a library product reaches here; a unit of a 256 x 256 tile takes 1.46 us, and a tile's outputs some 9 us
// more that nothing hides (8192 x 4096 of 4096 with gelu, residual and Z 231 to 245 us from card to card, 1120 to 1190 TFLOP/s; gated, 4096 x 4096 x 2 of 1024 with both Z 74 to 77 us, 890 to 930).
constexpr int AK = 64, A_RING = 4;
typedef int i4v __attribute__((ext_vector_type(4)));
template <int EXTENT, bool T_CONTIG, int WAVES> struct Async {
	static constexpr int SLOTS = T_CONTIG ? AK / 8 : EXTENT / 8, BYTES = EXTENT * AK * 2, LOADS = BYTES / 1024 / WAVES;
	static_assert(LOADS >= 2, "a wavefront has something to load");
	uint32_t at[LOADS], step; // byte offset from the tile's first element; first step of the chunk (T_CONTIG: the same for every load)
	__device__ static int source(int line, int slot) { // chunk that lies in a line's slot (its own inverse)
		if (T_CONTIG) return slot ^ (line & 7);                         // 8 lanes read 8 lines' 16-byte chunks
		return slot ^ (((line & 3) | ((line >> 1) & 4)) << 1);          // 32 lanes read 32 bytes of lines 0..3, 8..11 (4..7, 12..15)
	}
	__device__ void setup(uint32_t lane, uint32_t wave, uint64_t ld, uint32_t skip_lines /* wave-uniform: lines in front of this wavefront's that belong to another matrix */) {
#pragma unroll
		for (int q = 0; q < LOADS; ++q) {
			const int slot = (wave * LOADS + q) * 64 + lane, line = slot / SLOTS, chunk = source(line, slot % SLOTS);
			at[q] = (uint32_t)((line - (int)skip_lines) * ld * 2 + chunk * 16); step = chunk * 8;
		}
	}
	// one of this wavefront's loads: 1024 bytes to LDS from `lds` on; chunks behind the last of the `left` steps are out of range: zero.  (M0 lives inside this block alone: the
	// compiler sets it anew wherever it needs it; the same test finds no other use)
	__device__ void load(int q, i4v rsrc, uint32_t lds, int left) const {
		const uint32_t off = T_CONTIG && (int)step >= left ? 0x80000000u : at[q];
		asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc));
	}
};
// size in bytes of `elements` elements (none if negative) as a buffer resource holds it: loads beyond return zero
__device__ inline int records(int64_t elements) {
	const int64_t bytes = elements * 2;
	return __builtin_amdgcn_readfirstlane((int)(bytes <= 0 ? 0u : bytes > 0x7ffffff0ll ? 0x7ffffff0u : (uint32_t)bytes));
}
__device__ inline const T* uniform(const T* p) { // (a pointer that is the same in every lane, in scalar registers)
	const uint64_t a = (uint64_t)p;
	return (const T*)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)a));
}
__device__ inline i4v resource(const T* p, int records) { const uint64_t a = (uint64_t)p; return i4v{(int)(uint32_t)a, (int)((a >> 32) & 0xffff), records, 0x00020000}; }
// Where an operand's next unit comes from and goes to (all in scalar registers).  T_CONTIG: a line's elements beyond the sum are masked (Async::load), lines beyond the matrix lie
// behind `records` wherever the unit is; otherwise the lines beyond the sum do, in its last unit alone.
template <bool T_CONTIG, int UNITS, int BYTES> struct Cursor {
	const T* p; uint64_t inc, ld; uint32_t lds, lds0, seg, loaded, end, width; int left, full, rec;
	__device__ void limit() { // the size of what may be read of the unit at hand; nothing behind the last one
		rec = loaded < end ? full : 0;
		if (!T_CONTIG && loaded < end && left < AK) rec = records((int64_t)(left - 1) * (int64_t)ld + width);
	}
	template <typename F> __device__ void next(F&& segment_start, uint32_t steps) {
		++loaded; left -= AK; p += inc;
		lds = lds == lds0 + (UNITS - 1) * BYTES ? lds0 : lds + BYTES;
		if (loaded >= end || left < AK) { // seldom: the sum's or a segment's end
			if (loaded < end && left <= 0) { ++seg; left = steps; p = segment_start(seg); }
			limit();
		}
	}
};
constexpr int async_lds(int tile, int units) { return tile * AK * 2 * (2 * units + 1); }
template <int BR, int BC, int WR, int WC, bool A_T, bool B_T, int EPI, int UNITS> __device__ inline void async_tile(const GemmArgs& g, char* lds, uint32_t index, uint32_t count) {
	constexpr int WAVES = WR * WC, FR = BR / WR / 16, FC = BC / WC / 16, OUT = GATED_TILE<EPI> ? BC / 2 : BC;
	typedef Async<BR, A_T, WAVES> LA; typedef Async<BC, B_T, WAVES> LB;
	constexpr int UNITS_A = UNITS + 1, UNITS_B = UNITS, LDS = UNITS_A * LA::BYTES + UNITS_B * LB::BYTES;
	constexpr int STRIP = BC / WC + 4, PASS = FR > 4 ? 4 : FR; // epilogue: floats per row of a wavefront's strip of LDS, fragment rows in it
	static_assert(WAVES * PASS * 16 * STRIP * 4 <= LDS && FR % PASS == 0, "the epilogue's strips fit");
	static_assert(FC % (GATED_TILE<EPI> ? 4 : 2) == 0 && FR % A_RING == 0 && LA::LOADS % FR == 0 && LB::LOADS % FR == 0, "");
	static_assert(LDS == async_lds(BR, UNITS), "");
	const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
	const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave / WC, wc = wave % WC, gq = lane >> 4, li = lane & 15;
	const Work w = work_of(g, index, count, (g.rows + BR - 1) / BR, (g.cols + OUT - 1) / OUT);
	const uint32_t r0 = w.row * BR, c0 = w.col * OUT, problem = w.problem, split = w.split;
	const uint32_t units_per_segment = (g.steps + AK - 1) / AK, n_units = units_per_segment * g.segments;
	const uint32_t t_begin = min(n_units, split * g.chunks_per_split), t_end = min(n_units, t_begin + g.chunks_per_split);
	const uint32_t which = GATED_TILE<EPI> && wave * LB::LOADS * 8 >= OUT ? 1 : 0; // gated: this wavefront loads gate or up weights
	LA la; LB lb;
	la.setup(lane, wave, g.lda, 0); lb.setup(lane, wave, g.ldb, which * OUT);
	auto start_a = [&](uint32_t seg) -> const T* { return uniform(g.a + problem * g.a_problem + seg * g.a_segment + (A_T ? (uint64_t)r0 * g.lda : (uint64_t)r0)); };
	auto start_b = [&](uint32_t seg) -> const T* { return uniform(B_T ? g.b[which] + (uint64_t)c0 * g.ldb : g.b[seg & 1] + c0); };
	Cursor<A_T, UNITS_A, LA::BYTES> ca; Cursor<B_T, UNITS_B, LB::BYTES> cb;
	{
		const uint32_t seg = units_per_segment ? t_begin / units_per_segment : 0, t0 = (t_begin - seg * units_per_segment) * AK, steps8 = up8(g.steps);
		ca.ld = g.lda; cb.ld = g.ldb; ca.inc = A_T ? AK : AK * g.lda; cb.inc = B_T ? AK : AK * g.ldb;
		ca.lds = ca.lds0 = lds0; cb.lds = cb.lds0 = lds0 + UNITS_A * LA::BYTES;
		ca.width = up8(g.rows) - r0; cb.width = up8(g.cols) - c0;
		ca.full = A_T ? records((int64_t)(min((uint32_t)BR, g.rows - r0) - 1) * (int64_t)g.lda + steps8) : records((int64_t)(AK - 1) * (int64_t)g.lda + ca.width);
		cb.full = B_T ? records((int64_t)(min((uint32_t)OUT, g.cols - c0) - 1) * (int64_t)g.ldb + steps8) : records((int64_t)(AK - 1) * (int64_t)g.ldb + cb.width);
		ca.seg = cb.seg = seg; ca.loaded = cb.loaded = t_begin; ca.end = cb.end = t_end; ca.left = cb.left = (int)(g.steps - t0);
		ca.p = start_a(seg) + (A_T ? t0 : t0 * g.lda); cb.p = start_b(seg) + (B_T ? t0 : t0 * g.ldb);
		ca.limit(); cb.limit();
	}
	auto load_a = [&](int q) { la.load(q, resource(ca.p, ca.rec), ca.lds + (wave * LA::LOADS + q) * 1024, ca.left); };
	auto load_b = [&](int q) { lb.load(q, resource(cb.p, cb.rec), cb.lds + (wave * LB::LOADS + q) * 1024, cb.left); };
	// where the lane finds its fragments in a unit: an address for each half and constants for operands along t; for the others the XOR leaves one a fragment row (A) or pair (B)
	typedef __attribute__((address_space(3))) const T8 lds_T8;
	auto frag_at = [&](int j) -> int { return GATED_TILE<EPI> ? (j >= FC / 2 ? OUT : 0) + (j % (FC / 2)) * 16 : j * 16; }; // column (in the B tile) of fragment j behind the wavefront's first one
	const uint32_t col0 = wc * (GATED_TILE<EPI> ? OUT / WC : BC / WC), row0 = wr * (BR / WR), l4 = li >> 2, xr = l4 | ((gq & 1) << 2);
	constexpr int NA = A_T ? 2 : FR, NB = B_T ? 2 : FC;
	uint32_t fa_at[NA], fb_at[NB];
#pragma unroll
	for (int k = 0; k < NA; ++k) fa_at[k] = A_T ? (row0 + li) * AK * 2 + (((k * 4) + gq) ^ (li & 7)) * 16 : (gq * 8 + l4) * BR * 2 + ((row0 / 16 + k) ^ xr) * 32 + (li & 3) * 8;
#pragma unroll
	for (int k = 0; k < NB; ++k) fb_at[k] = B_T ? (col0 + li) * AK * 2 + (((k * 4) + gq) ^ (li & 7)) * 16 : (gq * 8 + l4) * BC * 2 + (((col0 + frag_at(k)) / 16) ^ xr) * 32 + (li & 3) * 8;
	auto tr4 = [](uint32_t at) -> s4 { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)at); };
	auto read_a = [&](int half, int i, uint32_t unit) -> T8 {
		if constexpr (A_T) return *(lds_T8*)(uintptr_t)(unit + fa_at[half] + i * 16 * AK * 2);
		else {
			const uint32_t at = unit + fa_at[i % NA] + half * 32 * BR * 2;
			const s4 lo = tr4(at), hi = tr4(at + 4 * BR * 2);
			return __builtin_bit_cast(T8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
		}
	};
	auto read_b = [&](int half, int j, uint32_t unit) -> T8 {
		if constexpr (B_T) return *(lds_T8*)(uintptr_t)(unit + fb_at[half] + frag_at(j) * AK * 2);
		else {
			const uint32_t at = unit + fb_at[j % NB] + half * 32 * BC * 2;
			const s4 lo = tr4(at), hi = tr4(at + 4 * BC * 2);
			return __builtin_bit_cast(T8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
		}
	};
	f4v acc[FR][FC];
#pragma unroll
	for (int i = 0; i < FR; ++i)
#pragma unroll
		for (int j = 0; j < FC; ++j) acc[i][j] = f4v{0.f, 0.f, 0.f, 0.f};
	constexpr int AHEAD = A_RING - 1;
	T8 fa[A_RING], fb[2][FC];
	uint32_t a_here = lds0, b_here = lds0 + UNITS_A * LA::BYTES;
	// The matrix instructions of one half of a unit.  One wavefront has the SIMD to itself, so whatever else is to be issued stands between two matrix instructions, a little at a
	// time.  Half 0: the barrier behind its first instructions says that every wavefront is through with the unit of A before this one, whose place the loads of the unit UNITS
	// ahead take.  Half 1: the barrier behind its first row of fragments says that every wavefront has this unit's B in registers and that the next units have arrived.
	auto half_step = [&](auto half_c, uint32_t a_next, uint32_t b_next) {
		constexpr int half = decltype(half_c)::value, Q = FC / 4;
#pragma unroll
		for (int i = 0; i < FR; ++i) {
#pragma unroll
			for (int j = 0; j < FC; ++j) {
				mfma_in_place(fb[half][j], fa[i % A_RING], acc[i][j]);
				if (j == (half == 1 && i == 0 ? FC - 1 : 0)) {
					if (half == 1 && i == 0) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((UNITS - 1) * LA::LOADS + (UNITS - 2) * LB::LOADS) : "memory");
					fa[(i + AHEAD) % A_RING] = i + AHEAD < FR ? read_a(half, i + AHEAD, a_here) : half == 0 ? read_a(1, i + AHEAD - FR, a_here) : read_a(0, i + AHEAD - FR, a_next);
				}
				if (half == 0 && i == 0 && j == Q) asm volatile("s_barrier" ::: "memory");
				if (j == 2 * Q && (half == 0 || i > 0)) { // (half 1: the loads begin with the second row)
#pragma unroll
					for (int q = 0; q < (half == 0 ? LA::LOADS / FR : LB::LOADS / FR); ++q) { if (half == 0) load_a(i * (LA::LOADS / FR) + q); else load_b((i - 1) * (LB::LOADS / FR) + q); }
				}
				if (half == 1 && i == FR - 1 && j == FC - 1) {
#pragma unroll
					for (int q = 0; q < LB::LOADS / FR; ++q) load_b((FR - 1) * (LB::LOADS / FR) + q);
				}
				if (j == 3 * Q) { // the next half's B fragments (half 1: they are the next unit's, from the second row on)
#pragma unroll
					for (int k = 0; k < FC; ++k) {
						constexpr int PER = FC / FR ? FC / FR : 1;
						if (half == 0 ? k / PER == i : i > 0 && (k / PER == i - 1 || (i == FR - 1 && k / PER >= FR - 1))) fb[half ^ 1][k] = half == 0 ? read_b(1, k, b_here) : read_b(0, k, b_next);
					}
				}
				__builtin_amdgcn_sched_barrier(0);
			}
		}
		if (half == 0) ca.next(start_a, g.steps); else cb.next(start_b, g.steps);
	};
	if (t_begin < t_end) {
		auto all_a = [&]() { for (int q = 0; q < LA::LOADS; ++q) load_a(q); ca.next(start_a, g.steps); };
		auto all_b = [&]() { for (int q = 0; q < LB::LOADS; ++q) load_b(q); cb.next(start_b, g.steps); };
#pragma unroll
		for (int k = 0; k < UNITS; ++k) { all_a(); all_b(); }
		asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((UNITS - 1) * (LA::LOADS + LB::LOADS)) : "memory");
#pragma unroll
		for (int i = 0; i < AHEAD; ++i) fa[i] = read_a(0, i, a_here);
#pragma unroll
		for (int j = 0; j < FC; ++j) fb[0][j] = read_b(0, j, b_here);
		for (uint32_t t = t_begin; t < t_end; ++t) {
			const uint32_t a_next = a_here == lds0 + (UNITS_A - 1) * LA::BYTES ? lds0 : a_here + LA::BYTES;
			const uint32_t b_next = b_here == lds0 + UNITS_A * LA::BYTES + (UNITS_B - 1) * LB::BYTES ? lds0 + UNITS_A * LA::BYTES : b_here + LB::BYTES;
			half_step(std::integral_constant<int, 0>(), a_next, b_next);
			half_step(std::integral_constant<int, 1>(), a_next, b_next);
			a_here = a_next; b_here = b_next;
		}
		settle(acc);
		asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); // nothing is under way to LDS any more
	}
	// epilogue through the wavefront's own strip of LDS: 8 consecutive columns a lane, whole lines a store, the residual of the next rows on its way
	float* strip = (float*)lds + wave * PASS * 16 * STRIP;
	constexpr int LANES = OUT / WC / 8, ROWS = 64 / LANES, AT_ONCE = 4; // lanes a row, rows at a time, such groups a turn
	static_assert(PASS * 16 % (ROWS * AT_ONCE) == 0, "");
	const uint32_t er = lane / LANES, ec = (lane % LANES) * 8, c = c0 + wc * (OUT / WC) + ec;
	const int n = (int)min(8u, g.cols > c ? g.cols - c : 0u);
	const T8 bias0 = bias8<EPI>(g, 0, c, n), bias1 = bias8<EPI>(g, 1, c, n);
#pragma unroll 1
	for (int pass = 0; pass < FR / PASS; ++pass) {
#pragma unroll
		for (int k = 0; k < FR / PASS; ++k)
			if (k == pass) {
#pragma unroll
				for (int i = 0; i < PASS; ++i)
#pragma unroll
					for (int j = 0; j < FC; ++j) *(f4v*)(strip + (i * 16 + li) * STRIP + j * 16 + gq * 4) = acc[k * PASS + i][j];
			}
		asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // (the strip is this wavefront's alone)
		const uint32_t r_pass = r0 + wr * (BR / WR) + pass * PASS * 16 + er;
		auto rows = [&](auto act_c, auto streamed_c) {
			T8 next[AT_ONCE];
			auto load_residual = [&](int k) {
#pragma unroll
				for (int q = 0; q < AT_ONCE; ++q) next[q] = residual8<EPI>(g, min(r_pass + k + q * ROWS, g.rows - 1), c, n);
			};
			load_residual(0);
#pragma unroll 1
			for (int k = 0; k < PASS * 16; k += ROWS * AT_ONCE) {
				T8 residual[AT_ONCE];
#pragma unroll
				for (int q = 0; q < AT_ONCE; ++q) residual[q] = next[q];
				if (k + ROWS * AT_ONCE < PASS * 16) load_residual(k + ROWS * AT_ONCE);
#pragma unroll
				for (int q = 0; q < AT_ONCE; ++q) {
					const uint32_t r = r_pass + k + q * ROWS;
					float z[8], u[8];
					const float* p = strip + (k + q * ROWS + er) * STRIP + ec;
					*(f4v*)z = *(const f4v*)p; *(f4v*)(z + 4) = *(const f4v*)(p + 4);
					if constexpr (GATED_TILE<EPI>) { *(f4v*)u = *(const f4v*)(p + OUT / WC); *(f4v*)(u + 4) = *(const f4v*)(p + OUT / WC + 4); }
					if (r < g.rows && n > 0) epilogue8<EPI>(g, problem, split, r, c, n, z, u, bias0, bias1, residual[q], decltype(act_c)::value, decltype(streamed_c)::value);
				}
			}
		};
		if constexpr (EPI == EPI_LINEAR || EPI == EPI_GATED) { if (g.streamed) with_act(g.act, [&](auto act_c) { rows(act_c, std::true_type()); }); else with_act(g.act, [&](auto act_c) { rows(act_c, std::false_type()); }); } else rows(std::integral_constant<int, NGP_ACT_NONE>(), std::false_type());
		asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
	}
}

template <int TILE, bool A_T, bool B_T, int EPI, int UNITS> __global__ __launch_bounds__(256, TILE >= 256 || UNITS > 2 ? 1 : 2) void k_gemm_async(GemmArgs g) {
	__shared__ __attribute__((aligned(1024))) char lds[async_lds(TILE, UNITS)];
	async_tile<TILE, TILE, 2, 2, A_T, B_T, EPI, UNITS>(g, lds, blockIdx.x, gridDim.x);
}
template <int UNITS> __global__ __launch_bounds__(256, UNITS > 2 ? 1 : 2) void k_products_async(GemmArgs x, GemmArgs w, uint32_t blocks_x, uint32_t blocks_w, bool w_first) { // (k_products)
	__shared__ __attribute__((aligned(1024))) char lds[async_lds(128, UNITS)];
	const Share s = share_of(blocks_x, blocks_w, w_first);
	if (s.x) async_tile<128, 128, 2, 2, true, false, EPI_STORE, UNITS>(x, lds, s.index, s.count);
	else async_tile<128, 128, 2, 2, false, false, EPI_STORE, UNITS>(w, lds, s.index, s.count);
}

// ---- few rows (a query at a time, a token at a time): bound by reading the weights once.  A wavefront takes 16 outputs (gated: of both projections) and a slice of the sum, weights
// straight from memory to registers as the matrix instruction's fragments, U loads on the way at a time; the samples (MT x 16 rows, the last one repeated where there are fewer)
// come out of the caches.  `slices` wavefronts share the sum and add up in LDS, in their order; where there are few outputs blocks share it too (EPI_PARTIAL*).
// 1 x 2048 -> 2 x 8192 (67 MB) 13.5 us, 5.0 TB/s; 1 x 2048 -> 2048 (8.4 MB) 5.9 us, of which a launch is most.
template <int MT, int EPI, bool ODD> __global__ __launch_bounds__(512) void k_few_rows(GemmArgs g, uint32_t slices, uint32_t steps_per_slice) {
	constexpr bool GATED = GATED_TILE<EPI>;
	constexpr int P = GATED ? 2 : 1, U = MT == 1 && !GATED ? 8 : 4;
	__shared__ float sums[8][P][MT * 16][20]; // [wavefront][projection][row][output]
	const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), gq = lane >> 4, li = lane & 15;
	const uint32_t slice = wave % slices, tile = blockIdx.x * (8 / slices) + wave / slices, c0 = tile * 16;
	const uint32_t t_begin = min(g.steps, (blockIdx.y * slices + slice) * steps_per_slice), t_end = min(g.steps, t_begin + steps_per_slice);
	const uint32_t col = min(c0 + li, g.cols - 1); // (outputs behind the last one repeat it and are dropped)
	const T* w[P]; const T* x[MT];
#pragma unroll
	for (int p = 0; p < P; ++p) w[p] = g.b[p] + (uint64_t)col * g.ldb + gq * 8;
#pragma unroll
	for (int m = 0; m < MT; ++m) x[m] = g.a + (uint64_t)min(m * 16 + li, g.rows - 1) * g.lda + gq * 8;
	f4v acc[P][MT];
#pragma unroll
	for (int p = 0; p < P; ++p)
#pragma unroll
		for (int m = 0; m < MT; ++m) acc[p][m] = f4v{0.f, 0.f, 0.f, 0.f};
	uint32_t t = t_begin;
	for (; t + U * 32 <= t_end; t += U * 32) {
		T8 fw[P][U], fx[MT][U];
#pragma unroll
		for (int u = 0; u < U; ++u)
#pragma unroll
			for (int p = 0; p < P; ++p) fw[p][u] = ODD ? load8_odd(w[p] + t + u * 32) : load8(w[p] + t + u * 32);
#pragma unroll
		for (int u = 0; u < U; ++u)
#pragma unroll
			for (int m = 0; m < MT; ++m) fx[m][u] = ODD ? load8_odd(x[m] + t + u * 32) : load8(x[m] + t + u * 32);
#pragma unroll
		for (int u = 0; u < U; ++u)
#pragma unroll
			for (int p = 0; p < P; ++p)
#pragma unroll
				for (int m = 0; m < MT; ++m) acc[p][m] = mfma(fw[p][u], fx[m][u], acc[p][m]);
	}
	for (; t < t_end; t += 32) { // what is left, the last chunk in part
		const int n = (int)(t_end - t) - (int)gq * 8;
		T8 fw[P], fx[MT];
#pragma unroll
		for (int p = 0; p < P; ++p) fw[p] = load8(w[p] + t, n);
#pragma unroll
		for (int m = 0; m < MT; ++m) fx[m] = load8(x[m] + t, n);
#pragma unroll
		for (int p = 0; p < P; ++p)
#pragma unroll
			for (int m = 0; m < MT; ++m) acc[p][m] = mfma(fw[p], fx[m], acc[p][m]);
	}
#pragma unroll
	for (int p = 0; p < P; ++p)
#pragma unroll
		for (int m = 0; m < MT; ++m) *(f4v*)&sums[wave][p][m * 16 + li][gq * 4] = acc[p][m];
	__syncthreads();
	// 8 outputs a thread: tile, row, half
	const uint32_t tiles = 8 / slices;
	for (uint32_t id = threadIdx.x; id < tiles * MT * 32; id += 512) {
		const uint32_t half = id & 1, r = (id >> 1) % (MT * 16), k = id / (MT * 32), c = (blockIdx.x * tiles + k) * 16 + half * 8;
		if (r >= g.rows || c >= g.cols) continue;
		const int n = (int)min(8u, g.cols - c);
		float z[8] = {}, u[8] = {};
		for (uint32_t q = 0; q < slices; ++q) {
			EACH z[e] += sums[k * slices + q][0][r][half * 8 + e];
			if (GATED) EACH u[e] += sums[k * slices + q][P - 1][r][half * 8 + e];
		}
		epilogue8<EPI>(g, 0, blockIdx.y, r, c, n, z, u, bias8<EPI>(g, 0, c, n), bias8<EPI>(g, 1, c, n), residual8<EPI>(g, r, c, n), g.act);
	}
}

// ---- narrow layers (up to 256 inputs and outputs) over many samples: bound by reading and writing the samples once.
// Forward: the weights lie in LDS as fragments (1 KB each, lane by lane), every wavefront takes 16 samples at a time straight from memory into its matrix operands, the next 16 on
// their way meanwhile, and has all of their outputs in registers.  No barrier after the first one.  Columns are dealt to fragments so that a lane owns 8 consecutive ones.
// 262144 x 256 of 256 (268 MB) 77 us, 3.5 TB/s; 65521 x 256 and Z of 63 (75 MB) 20.9 us a call, 21.2 to 22.5 us traced alone, 3.6 TB/s, of which staging the weights and filling the card take
// about 5.  Variants with 32 fragments of weights are held to 128 registers so that two blocks share a compute unit: 12 of these 22, gated ones or for EXCHANGE or odd lines,
// spill 1 to 38 registers.
// ODD: lines that begin between two dwords are read by the dword (65521 x 256 and Z of 63 21.8 -> 20.6 us, 262144 x 64 of 255 68 -> 55 us; a kernel of its own, since the others lose 3 to 10 %).
// NF: 16-column fragments of weights (gated: gate, then up), KS: steps of 32 inputs.
template <int NF, int KS, int EPI, bool EXCHANGE, bool ODD> __global__ __launch_bounds__(512, NF * KS <= 32 ? 4 : 2) void k_narrow_forward(GemmArgs g) {
	constexpr bool GATED = GATED_TILE<EPI>;
	constexpr int OF = GATED ? NF / 2 : NF; // fragments of outputs
	__shared__ __attribute__((aligned(16))) T w[NF * KS * 512];
	const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), gq = lane >> 4, li = lane & 15;
	const uint32_t slabs = (g.rows + 15) / 16, stride = gridDim.x * 8;
	uint32_t slab = blockIdx.x * 8 + wave;
	const int steps = (int)g.steps, whole_ks = steps / 32; // steps of 32 without a line's end
	T8 x[KS];
	uint32_t last[ODD ? KS : 1]; // fifth dwords
	auto load_x = [&](uint32_t s) {
		const T* line = g.a + (uint64_t)min(s * 16 + li, g.rows - 1) * g.lda; // (samples behind the last one repeat it and are dropped)
#pragma unroll
		for (int k = 0; k < KS; ++k) {
			const T* p = line + min(k * 32 + (int)gq * 8, steps - 8);
			if (ODD) { const uint32_t* q = (const uint32_t*)((uintptr_t)p & ~(uintptr_t)3); __builtin_memcpy(&x[k], q, 16); last[ODD ? k : 0] = q[(uintptr_t)p & 2 ? 4 : 3]; }
			else x[k] = load8(p);
		}
	};
	auto tail_x = [&](uint32_t s) { // the line's end
		if constexpr (ODD) { // elements out of the dwords (load8_odd in two steps: these loads were on their way)
			const bool odd_line = (uintptr_t)(g.a + (uint64_t)min(s * 16 + li, g.rows - 1) * g.lda) & 2;
#pragma unroll
			for (int k = 0; k < KS; ++k) {
				const bool odd = odd_line != (k * 32 + (int)gq * 8 > steps - 8 && (steps & 1));
				uint32_t v[4];
				__builtin_memcpy(v, &x[k], 16);
				const uint32_t r[4] = {odd ? __builtin_amdgcn_alignbit(v[1], v[0], 16) : v[0], odd ? __builtin_amdgcn_alignbit(v[2], v[1], 16) : v[1],
					odd ? __builtin_amdgcn_alignbit(v[3], v[2], 16) : v[2], odd ? __builtin_amdgcn_alignbit(last[ODD ? k : 0], v[3], 16) : v[3]};
				__builtin_memcpy(&x[k], r, 16);
			}
		}
		if (whole_ks == KS) return;
#pragma unroll
		for (int k = 0; k < KS; ++k) if (k >= whole_ks) x[k] = shift8(x[k], k * 32 + gq * 8, steps);
	};
	if (slab < slabs) load_x(slab);
	constexpr int EACH_THREAD = NF * KS / 8, BATCH = EACH_THREAD < 8 ? EACH_THREAD : 8;
	const bool odd = ((uintptr_t)g.b[0] | (uintptr_t)g.b[GATED ? 1 : 0] | g.ldb * 2) & 3;
#pragma unroll
	for (int q0 = 0; q0 < EACH_THREAD; q0 += BATCH) { // (all loads of a batch on their way together)
		T8 v[BATCH];
#pragma unroll
		for (int b = 0; b < BATCH; ++b) {
			const int q = (q0 + b) * 512 + threadIdx.x, l = q & 63, k = (q >> 6) % KS, f = (q >> 6) / KS, i = l & 15, col = (f / 2 % (OF / 2)) * 32 + (i >> 2) * 8 + (f & 1) * 4 + (i & 3);
			const T* p = g.b[GATED && f >= OF] + (uint64_t)min((uint32_t)col, g.cols - 1) * g.ldb + min(k * 32 + (l >> 4) * 8, steps - 8);
			v[b] = odd ? load8_odd(p) : load8(p);
		}
#pragma unroll
		for (int b = 0; b < BATCH; ++b) {
			const int q = (q0 + b) * 512 + threadIdx.x, c = ((q >> 6) % KS) * 32 + ((q & 63) >> 4) * 8;
			*(T8*)(w + q * 8) = steps == KS * 32 ? v[b] : shift8(v[b], c, steps);
		}
	}
	__syncthreads();
	for (; slab < slabs; slab += stride) {
		asm volatile("" ::: "memory"); // (the weights stay in LDS: kept in registers across samples they spill)
		f4v acc[NF];
#pragma unroll
		for (int f = 0; f < NF; ++f) acc[f] = f4v{0.f, 0.f, 0.f, 0.f};
		tail_x(slab);
#pragma unroll
		for (int k = 0; k < KS; ++k)
#pragma unroll
			for (int f = 0; f < NF; ++f) acc[f] = mfma(*(const T8*)(w + ((f * KS + k) * 64 + lane) * 8), x[k], acc[f]);
		if (slab + stride < slabs) load_x(slab + stride);
		const uint32_t r = slab * 16 + li;
		if constexpr (EXCHANGE) with_act(g.act, [&](auto act_c) {
			// EXCHANGE: two pieces of 32 columns at a time, neighbouring lanes (samples) swap one chunk each, so that a store writes 128 bytes of a line (262144 x 256 from 64 inputs 79 -> 58 us;
			// 65536 samples 14 -> 16 us, where a wavefront goes through this code once: not there)
			constexpr int PAIR = 2;
#pragma unroll
			for (int p = 0; p < OF / 2; p += PAIR) {
				T8 pre0[PAIR], pre1[PAIR], o[PAIR];
#pragma unroll
				for (int h = 0; h < PAIR; ++h) {
					const uint32_t c = (p + h) * 32 + gq * 8;
					const int n = (int)min(8u, g.cols > c ? g.cols - c : 0u), q = p + h;
					float z[8], u[8];
					EACH { z[e] = acc[2 * q + e / 4][e & 3]; u[e] = GATED ? acc[(GATED ? OF : 0) + 2 * q + e / 4][e & 3] : 0.f; }
					const T8 residual = r < g.rows ? residual8<EPI>(g, r, c, n) : T8{};
					outputs8<EPI>(z, u, bias8<EPI>(g, 0, c, n), bias8<EPI>(g, 1, c, n), g.residual ? &residual : nullptr, decltype(act_c)::value, pre0[h], pre1[h], o[h]);
				}
				auto store = [&](T* to, uint64_t ld, const T8 (&v)[PAIR]) {
					const bool second = li & 1;
					const uint32_t c = (p + second) * 32 + gq * 8, r0 = r & ~1u;
					const int n = (int)min(8u, g.cols > c ? g.cols - c : 0u);
					const T8 given = second ? v[0] : v[1], kept = second ? v[1] : v[0];
					uint32_t d[4];
					__builtin_memcpy(d, &given, 16);
#pragma unroll
					for (int i = 0; i < 4; ++i) d[i] = __builtin_amdgcn_mov_dpp(d[i], 0xb1 /* lanes 1, 0, 3, 2 of four */, 0xf, 0xf, true);
					T8 got;
					__builtin_memcpy(&got, d, 16);
					if (n > 0 && r0 < g.rows) store8(to + (uint64_t)r0 * ld + c, second ? got : kept, n, g.streamed);
					if (n > 0 && r0 + 1 < g.rows) store8(to + (uint64_t)(r0 + 1) * ld + c, second ? kept : got, n, g.streamed);
				};
				if (g.pre[0]) store(g.pre[0], g.ld_pre, pre0);
				if (GATED && g.pre[1]) store(g.pre[1], g.ld_pre, pre1);
				store(g.c[0], g.ldc, o);
			}
		}); else if (r < g.rows) with_act(g.act, [&](auto act_c) {
#pragma unroll
			for (int p = 0; p < OF / 2; ++p) {
				const uint32_t c = p * 32 + gq * 8;
				if (c >= g.cols) continue;
				const int n = (int)min(8u, g.cols - c);
				float z[8], u[8];
				EACH { z[e] = acc[2 * p + e / 4][e & 3]; u[e] = GATED ? acc[(GATED ? OF : 0) + 2 * p + e / 4][e & 3] : 0.f; }
				epilogue8<EPI>(g, 0, 0, r, c, n, z, u, bias8<EPI>(g, 0, c, n), bias8<EPI>(g, 1, c, n), residual8<EPI>(g, r, c, n), decltype(act_c)::value);
			}
		});
	}
}
// Backward in one pass: a block takes 32 samples at a time (the next 32 on their way), forms G = dY * act'(Z) and lays it and X into LDS; its 8 wavefronts multiply G with the weights
// (in LDS too) to dX, and G^T with X into their parts of dW, which stay in registers to the end: one partial sum a block, joined by a second launch.  Every sample's
// dY, Z, X is read once, dX written once.  262144 samples, 256 x 256 (537 MB): 142 us, 3.8 TB/s, bound by LDS (both products read G from it) as much as by memory.  NF: 16-column fragments of G (gated: gate, then up), KF: of X.
// No variant of a linear layer spills; two gated ones do (128 x 128: 18 registers, 256 x 256: 3).
struct NarrowArgs {
	uint32_t rows, n, k; int act; const T* x; uint64_t ld_x; const T* w[2]; uint64_t ld_w; const T* pre[2]; uint64_t ld_pre; const T* dy; uint64_t ld_dy; T* dx; uint64_t ld_dx;
	float* partial; float* bias_partial;
};
template <int NF, int KF, bool GATED> __global__ __launch_bounds__(512, NF <= 8 && KF <= 8 ? 4 : 2) void k_narrow_backward(NarrowArgs g) {
	constexpr int GC = NF * 16, XC = KF * 16, HALF = GC / 2, NS = NF / 2; // columns of G and X in LDS, first column of the up projection, steps of 32 outputs
	constexpr int CG = (GATED ? HALF : GC) / 8, CX = XC / 8, RG = 512 / CG, RX = 512 / CX, LG = RG >= 32 ? 1 : 32 / RG, LX = RX >= 32 ? 1 : 32 / RX; // chunks a line, lines at once, chunks a thread
	constexpr int UNITS = KF * 2 / 8, WN = NF / 4, WK = KF / 2; // 16 x 16 pieces of dX a wavefront has, fragments of dW (4 x 2 wavefronts)
	static_assert(NF >= 4 && KF >= 4, "");
	constexpr int RL = RG < 32 ? RG : 32, SLABS = 32 * (GC + XC) * 2, RED = RL * GC * 4; // (the bias's sums take the slabs' place at the end)
	__shared__ __attribute__((aligned(16))) char shared[GC * XC * 2 + (SLABS > RED ? SLABS : RED)];
	T* lw = (T*)shared; T* lg = lw + GC * XC; T* lx = lg + 32 * GC; // weights, G, X
	const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), gq = lane >> 4, li = lane & 15, l4 = li >> 2;
	const int gc = (tid % CG) * 8, gr = tid / CG, xc = (tid % CX) * 8, xr = tid / CX;
	const uint32_t slabs = (g.rows + 31) / 32;
	const bool ragged_n = g.n & 7 || g.n < (GATED ? HALF : GC), ragged_k = g.k & 7 || g.k < XC;
	// a line's 16-byte slots are exchanged by an XOR with bits of the line, so that 16 lines' chunks (dX) and 32 bytes of 8 lines (dW's transposing reads) lie in different banks
	auto slot = [](int line, int s, int slots) -> int { return s ^ ((((line & 3) << 1) | (line & 8) | ((line >> 2) & 1)) & (slots >= 16 ? 15 : slots - 1)); };
	T8 dy[LG], z[LG], u[GATED ? LG : 1], x[LX];
	auto load = [&](uint32_t s) {
		if (RG < 32 || gr < 32) {
#pragma unroll
			for (int q = 0; q < LG; ++q) {
				const uint64_t r = min(s * 32 + gr + q * RG, g.rows - 1);
				const int c = min(gc, (int)g.n - 8);
				dy[q] = load8(g.dy + r * g.ld_dy + c);
				z[q] = load8(g.pre[0] + r * g.ld_pre + c);
				if (GATED) u[GATED ? q : 0] = load8(g.pre[1] + r * g.ld_pre + c);
			}
		}
		if (RX < 32 || xr < 32) {
#pragma unroll
			for (int q = 0; q < LX; ++q) x[q] = load8(g.x + (uint64_t)min(s * 32 + xr + q * RX, g.rows - 1) * g.ld_x + min(xc, (int)g.k - 8));
		}
	};
	auto tails = [&]() { // the lines' ends
		if (ragged_n) {
#pragma unroll
			for (int q = 0; q < LG; ++q) { dy[q] = shift8(dy[q], gc, g.n); z[q] = shift8(z[q], gc, g.n); if (GATED) u[GATED ? q : 0] = shift8(u[GATED ? q : 0], gc, g.n); }
		}
		if (ragged_k) {
#pragma unroll
			for (int q = 0; q < LX; ++q) x[q] = shift8(x[q], xc, g.k);
		}
	};
	uint32_t s = blockIdx.x;
	if (s < slabs) load(s);
	auto tr8_at = [&](const T* base, int cols, int line0, int e) -> T8 { // 8 of the 32 lines from line0 on, of the column whose group of 4 the lane reads at e
		const int line = line0 + gq * 8 + l4;
		const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(base + line * cols + slot(line, e >> 3, cols / 8) * 8 + (e & 7)));
		const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(base + (line + 4) * cols + slot(line + 4, e >> 3, cols / 8) * 8 + (e & 7)));
		return __builtin_bit_cast(T8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
	};
	auto tr8 = [&](const T* base, int cols, int line0, int f) -> T8 { return tr8_at(base, cols, line0, f * 16 + (li & 3) * 4); }; // of column 16 f + li
	if (g.dx) { // the weights: lines behind the last output meet zeros of G, but must not be NaN
		constexpr int EACH_THREAD = GC * XC / 8 / 512, BATCH = EACH_THREAD < 8 ? EACH_THREAD : 8;
#pragma unroll
		for (int q0 = 0; q0 < EACH_THREAD; q0 += BATCH) {
			T8 v[BATCH];
#pragma unroll
			for (int b = 0; b < BATCH; ++b) {
				const int q = (q0 + b) * 512 + tid, l = q / CX, up = GATED && l >= HALF, n = l - up * HALF;
				v[b] = load8(g.w[up] + (uint64_t)min((uint32_t)n, g.n - 1) * g.ld_w + min((q % CX) * 8, (int)g.k - 8));
			}
#pragma unroll
			for (int b = 0; b < BATCH; ++b) {
				const int q = (q0 + b) * 512 + tid, line = q / CX, c = (q % CX) * 8, n = line - (GATED && line >= HALF) * HALF;
				const T8 w = ragged_k ? shift8(v[b], c, g.k) : v[b];
				*(T8*)(lw + line * XC + slot(line, c / 8, CX) * 8) = n < (int)g.n ? w : T8{};
			}
		}
	}
	float sum[GATED ? 2 : 1][8] = {};
	f4v acc[WN][WK];
#pragma unroll
	for (int i = 0; i < WN; ++i)
#pragma unroll
		for (int j = 0; j < WK; ++j) acc[i][j] = f4v{0.f, 0.f, 0.f, 0.f};
	for (; s < slabs; s += gridDim.x) {
		// G and X into LDS; samples behind the last one are zero
		const bool last = s * 32 + 32 > g.rows;
		tails();
#pragma unroll
		for (int q = 0; q < LG; ++q) if (RG < 32 || gr < 32) {
			const int line = gr + q * RG;
			if (last && s * 32 + line >= g.rows) { dy[q] = z[q] = T8{}; u[GATED ? q : 0] = T8{}; }
			float v[8], v2[8];
			T8 o, o2;
			output_grad8<GATED>(g.act, dy[q], z[q], u[GATED ? q : 0], v, v2);
			EACH { sum[0][e] += v[e]; o[e] = (T)v[e]; if (GATED) { sum[GATED ? 1 : 0][e] += v2[e]; o2[e] = (T)v2[e]; } }
			*(T8*)(lg + line * GC + slot(line, gc / 8, GC / 8) * 8) = o;
			if (GATED) *(T8*)(lg + line * GC + slot(line, (HALF + gc) / 8, GC / 8) * 8) = o2;
		}
#pragma unroll
		for (int q = 0; q < LX; ++q) if (RX < 32 || xr < 32) {
			const int line = xr + q * RX;
			*(T8*)(lx + line * XC + slot(line, xc / 8, XC / 8) * 8) = last && s * 32 + line >= g.rows ? T8{} : x[q];
		}
		const uint32_t here = s;
		if (s + gridDim.x < slabs) load(s + gridDim.x);
		lds_barrier();
		if (g.dx) {
			// pieces of 16 samples x 16 inputs, two at a time: with 256 inputs a wavefront has 32 of them, dealt to two fragments so that a lane owns 8 consecutive ones; with 128 it has 16, of both
			// halves of the samples; with 64 one piece
			constexpr bool WIDE = UNITS == 4;
			constexpr int PAIR = UNITS == 1 ? 1 : 2;
#pragma unroll 1
			for (int q = 0; q < UNITS / PAIR; ++q) {
				const int kf = UNITS == 1 ? wave >> 1 : WIDE ? wave * 2 : wave;
				f4v d[PAIR];
#pragma unroll
				for (int h = 0; h < PAIR; ++h) d[h] = f4v{0.f, 0.f, 0.f, 0.f};
				auto rows_at = [&](int h) -> int { return UNITS == 1 ? (int)(wave & 1) * 16 : WIDE ? q * 16 : h * 16; };
#pragma unroll 4
				for (int ns = 0; ns < NS; ++ns) {
					T8 a, b;
#pragma unroll
					for (int h = 0; h < PAIR; ++h) {
						if (!WIDE || h == 0) { const int line = rows_at(h) + li; a = *(const T8*)(lg + line * GC + slot(line, ns * 4 + gq, GC / 8) * 8); }
						if (WIDE) b = tr8_at(lw, XC, ns * 32, kf * 16 + (li & 3) * 8 + h * 4); else if (h == 0) b = tr8(lw, XC, ns * 32, kf);
						d[h] = mfma(b, a, d[h]);
					}
				}
				if constexpr (WIDE) {
					const uint32_t r = here * 32 + rows_at(0) + li, c = kf * 16 + gq * 8;
					T8 o;
					EACH o[e] = (T)d[e / 4][e & 3];
					if (r < g.rows && c < g.k) store8(g.dx + (uint64_t)r * g.ld_dx + c, o, (int)min(8u, g.k - c));
				} else {
#pragma unroll
					for (int h = 0; h < PAIR; ++h) {
						const uint32_t r = here * 32 + rows_at(h) + li, c = kf * 16 + gq * 4;
						if (r < g.rows && c < g.k) {
							T* o = g.dx + (uint64_t)r * g.ld_dx + c;
							T v[4] = {(T)d[h][0], (T)d[h][1], (T)d[h][2], (T)d[h][3]};
							if (c + 4 <= g.k) __builtin_memcpy(o, v, 8);
							else {
#pragma unroll
								for (int e = 0; e < 3; ++e) if (c + e < g.k) o[e] = v[e];
							}
						}
					}
				}
			}
		}
		if (g.partial) {
			T8 a[WN];
#pragma unroll
			for (int i = 0; i < WN; ++i) a[i] = tr8(lg, GC, 0, (wave >> 1) * WN + i);
#pragma unroll
			for (int j = 0; j < WK; ++j) {
				const T8 b = tr8(lx, XC, 0, (wave & 1) * WK + j);
#pragma unroll
				for (int i = 0; i < WN; ++i) acc[i][j] = mfma(b, a[i], acc[i][j]);
			}
		}
		lds_barrier();
	}
	if (g.partial) {
		const uint32_t k8 = up8(g.k);
#pragma unroll
		for (int i = 0; i < WN; ++i)
#pragma unroll
			for (int j = 0; j < WK; ++j) {
				const uint32_t c = ((wave >> 1) * WN + i) * 16 + li, problem = GATED && c >= HALF, n = c - problem * HALF, k = ((wave & 1) * WK + j) * 16 + gq * 4;
				if (n < g.n && k < k8) *(f4v*)(g.partial + (((uint64_t)blockIdx.x * (GATED ? 2 : 1) + problem) * g.n + n) * k8 + k) = acc[i][j];
			}
	}
	if (g.bias_partial) {
		float* red = (float*)lg; // [RL][GC]
#pragma unroll
		for (int p = 0; p < (GATED ? 2 : 1); ++p)
			if (gr < RL) { EACH red[gr * GC + p * HALF + gc + e] = sum[p][e]; }
		__syncthreads();
		for (uint32_t c = tid; c < (uint32_t)GC; c += 512) {
			float t = 0.f;
			for (int y = 0; y < RL; ++y) t += red[y * GC + c];
			const uint32_t problem = GATED && c >= (uint32_t)HALF, n = c - problem * HALF;
			if (n < g.n) g.bias_partial[((uint64_t)blockIdx.x * (GATED ? 2 : 1) + problem) * g.n + n] = t;
		}
	}
}

// G = dY * act'(Z) (gated: [dH * Zu * act'(Zg) | dH * act(Zg)]), lines padded with zeros to multiples of 8 columns, rounded once to the layer's type (the matrix
// instructions take 16-bit operands; the relative error of a rounding, 2^-12 / 2^-9 on average, is that of the result's own; small sets in two terms), and its column sums (in 32 bits,
// one line per block of rows, before the rounding; the gradient itself where there is one block).  Memory bound (gated,
// 8192 x 8192, 671 MB: 117 us, 5.7 TB/s; 90765 x 1928, 1.75 GB: 370 us, 4.7 TB/s).  256 threads: COLS / 8 along a line, the rest on further lines.
struct GradArgs { uint32_t rows, cols; int act; const T* dy; uint64_t ld_dy; const T* pre[2]; uint64_t ld_pre; T* out; uint64_t ld_out; float* bias_partial; T* dbias[2]; uint32_t rows_per_block; bool two_terms; };
template <bool GATED, uint32_t COLS> __global__ __launch_bounds__(256) void k_output_grad(GradArgs g) {
	constexpr uint32_t CX = COLS / 8, RY = 256 / CX;
	const uint32_t cx = threadIdx.x % CX, ry = threadIdx.x / CX, c = blockIdx.x * COLS + cx * 8, pc = up8(g.cols);
	const uint32_t end = min(g.rows, (blockIdx.y + 1) * g.rows_per_block);
	const bool odd = ((uintptr_t)g.dy | (uintptr_t)g.pre[0] | (uintptr_t)g.pre[1] | g.ld_dy * 2 | g.ld_pre * 2) & 3;
	float sum[GATED ? 2 : 1][8] = {};
	if (c < g.cols) {
		// lines of 8 elements and more: the last chunk is read from 8 in front of the end and moved down
		const bool ragged = g.cols & 7 && g.cols >= 8;
		const int n = ragged ? 8 : (int)min(8u, g.cols - c), at = ragged ? min((int)c, (int)g.cols - 8) : (int)c;
		for (uint32_t r = blockIdx.y * g.rows_per_block + ry; r < end; r += RY) {
			auto load = [&](const T* p) -> T8 {
				if (n < 8) return load8(p, n);
				const T8 v = odd ? load8_odd(p) : load8(p);
				return ragged ? shift8(v, c, g.cols) : v;
			};
			const T8 dy = load(g.dy + (uint64_t)r * g.ld_dy + at);
			T8 z{}, u{}, o, o2;
			if (g.pre[0]) z = load(g.pre[0] + (uint64_t)r * g.ld_pre + at);
			if (GATED) u = load(g.pre[1] + (uint64_t)r * g.ld_pre + at);
			float v[8], v2[8];
			output_grad8<GATED>(g.act, dy, z, u, v, v2);
			EACH { sum[0][e] += v[e]; o[e] = (T)v[e]; if (GATED) { sum[GATED ? 1 : 0][e] += v2[e]; o2[e] = (T)v2[e]; } }
			if (g.out) {
				*(T8*)(g.out + (uint64_t)r * g.ld_out + c) = o;
				if (GATED) *(T8*)(g.out + (uint64_t)r * g.ld_out + pc + c) = o2;
				if (g.two_terms) { // what the rounding lost, behind all rounded ones
					auto lost = [](float exact, T rounded) -> T { const float d = exact - (float)rounded; return (T)(fabsf(d) < __builtin_inff() ? d : 0.f); }; // (nothing of what is not finite)
					EACH { o[e] = lost(v[e], o[e]); if (GATED) o2[e] = lost(v2[e], o2[e]); }
					*(T8*)(g.out + (uint64_t)r * g.ld_out + (GATED ? 2 : 1) * pc + c) = o;
					if (GATED) *(T8*)(g.out + (uint64_t)r * g.ld_out + 3 * pc + c) = o2;
				}
			}
		}
	}
	if (!g.bias_partial && !g.dbias[0] && !g.dbias[1]) return;
	__shared__ float red[RY][COLS + 8];
#pragma unroll
	for (int k = 0; k < (GATED ? 2 : 1); ++k) {
		__syncthreads();
#pragma unroll
		for (int e = 0; e < 8; ++e) red[ry][cx * 8 + e] = sum[k][e];
		__syncthreads();
		for (uint32_t i = threadIdx.x; i < COLS; i += 256) {
			float s = 0.f;
#pragma unroll
			for (uint32_t y = 0; y < RY; ++y) s += red[y][i];
			const uint32_t col = blockIdx.x * COLS + i;
			if (col >= g.cols) break;
			if (g.bias_partial) g.bias_partial[((uint64_t)blockIdx.y * (GATED ? 2 : 1) + k) * g.cols + col] = s;
			else if (g.dbias[k]) g.dbias[k][col] = (T)s; // (one block of rows: the sum is whole)
		}
	}
}
// dbias = sum of the blocks' column sums: a block takes 16 columns, 16 threads each, then adds the shares up in their order
struct BiasArgs { const float* partial; uint32_t blocks, cols, problems; T* out[2]; };
__device__ inline void bias_grad(const BiasArgs& a, uint32_t index, float* shared) {
	const uint32_t cx = threadIdx.x & 15, ry = threadIdx.x >> 4, per = (a.cols + 15) / 16, k = index / per, c = (index % per) * 16 + cx;
	float s = 0.f;
	if (c < a.cols) {
#pragma unroll 8
		for (uint32_t b = ry; b < a.blocks; b += 16) s += a.partial[((uint64_t)b * a.problems + k) * a.cols + c];
	}
	shared[ry * 17 + cx] = s;
	__syncthreads();
	if (ry || c >= a.cols || !a.out[k]) return;
	s = 0.f;
#pragma unroll
	for (int y = 0; y < 16; ++y) s += shared[y * 17 + cx];
	a.out[k][c] = (T)s;
}
// the splits' sums, GROUPS threads sharing them out (in a fixed order), then the product's own epilogue (EPI_GATED: partial sums of both projections)
template <int EPI, int GROUPS> __device__ inline void join_splits(const GemmArgs& g, uint32_t index, float* shared) {
	constexpr int P = EPI == EPI_GATED ? 2 : 1, ITEMS = 256 / GROUPS;
	const uint32_t cc = up8(g.cols) / 8, per = (uint32_t)(((uint64_t)g.rows * cc + ITEMS - 1) / ITEMS), problem = index / per, parts = P == 2 ? 2 : g.problems, item = threadIdx.x % ITEMS, group = threadIdx.x / ITEMS;
	const uint64_t id = (uint64_t)(index % per) * ITEMS + item;
	const bool in = id < (uint64_t)g.rows * cc;
	if (GROUPS == 1 && !in) return;
	const uint32_t r = in ? (uint32_t)(id / cc) : 0, c = in ? (uint32_t)(id % cc) * 8 : 0;
	const uint64_t part = (uint64_t)g.rows * cc * 8;
	const int n = (int)min(8u, g.cols - c);
	T8 bias0{}, bias1{}, residual{};
	if (group == 0) { bias0 = bias8<EPI>(g, 0, c, n); bias1 = bias8<EPI>(g, 1, c, n); residual = residual8<EPI>(g, r, c, in ? n : 0); }
	float z[8] = {}, u[8] = {};
	const float* p = g.partial + problem * part + (uint64_t)r * cc * 8 + c + (uint64_t)group * parts * part;
#pragma unroll 4
	for (uint32_t k = group; k < g.splits; k += GROUPS, p += (uint64_t)GROUPS * parts * part) {
		const f4v a = *(const f4v*)p, b = *(const f4v*)(p + 4);
#pragma unroll
		for (int e = 0; e < 4; ++e) { z[e] += a[e]; z[e + 4] += b[e]; }
		if constexpr (P == 2) {
			const f4v d = *(const f4v*)(p + part), f = *(const f4v*)(p + part + 4);
#pragma unroll
			for (int e = 0; e < 4; ++e) { u[e] += d[e]; u[e + 4] += f[e]; }
		}
	}
	if constexpr (GROUPS > 1) {
		float* red = shared + ((group * P) * ITEMS + item) * 9;
		EACH { red[e] = z[e]; if (P == 2) red[ITEMS * 9 + e] = u[e]; }
		__syncthreads();
		if (group || !in) return;
#pragma unroll
		for (int q = 1; q < GROUPS; ++q) EACH { z[e] += red[q * P * ITEMS * 9 + e]; if (P == 2) u[e] += red[(q * P + 1) * ITEMS * 9 + e]; }
	}
	if constexpr (EPI == EPI_STORE) { // (the sums are whole now)
		T8 o;
		EACH o[e] = (T)z[e];
		store8(g.c[problem] + (uint64_t)r * g.ldc + c, o, n);
	} else epilogue8<EPI>(g, problem, 0, r, c, n, z, u, bias0, bias1, residual, g.act);
}
template <int EPI> __device__ inline void join_any(const GemmArgs& g, int groups, uint32_t index, float* shared) {
	if (groups > 8) join_splits<EPI, 32>(g, index, shared); else if (groups > 1) join_splits<EPI, 8>(g, index, shared); else join_splits<EPI, 1>(g, index, shared);
}
template <int EPI> __global__ __launch_bounds__(256) void k_join_splits(GemmArgs g, int groups) {
	__shared__ float shared[(EPI == EPI_GATED ? 2 : 1) * 256 * 9];
	join_any<EPI>(g, groups, blockIdx.x, shared);
}
// what is left of a backward pass in one launch: dX's and dW's split sums, the bias's (256 x 256 of 256 pieces, 67 MB: 12 us, 5.6 TB/s, out of the last cache)
__global__ __launch_bounds__(256) void k_finish(GemmArgs x, int groups_x, uint32_t blocks_x, GemmArgs w, int groups_w, uint32_t blocks_w, BiasArgs bias) {
	__shared__ float shared[256 * 9];
	uint32_t b = blockIdx.x;
	if (b < blocks_x) { join_any<EPI_STORE>(x, groups_x, b, shared); return; }
	b -= blocks_x;
	if (b < blocks_w) { join_any<EPI_STORE>(w, groups_w, b, shared); return; }
	bias_grad(bias, b - blocks_w, shared);
}

uint32_t div_up(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }
bool whole(const void* p, uint64_t ld, uint64_t width) { return ((uintptr_t)p & 3) == 0 && (ld & 1) == 0 && (width & 7) == 0 && ld <= DENSE_LINE; } // 16-byte pieces, each from a dword on; a tile's offsets fit 31 bits
// X and the weights with their lines padded with zeros to whole 16-byte pieces, for the tiles that take nothing else; memory bound (200000 x 500: 64 us, 6.3 TB/s)
struct PackArgs { const T* from[3]; T* to[3]; uint64_t ld[3]; uint32_t lines[3]; uint32_t width; };
constexpr uint32_t PACK_BLOCKS = 1u << 16; // at most; each then goes on to further chunks (X may have more chunks than a launch has threads)
__global__ __launch_bounds__(256) void k_pack(PackArgs g) {
	const uint32_t cc = up8(g.width) / 8;
	const uint64_t total = ((uint64_t)g.lines[0] + g.lines[1] + g.lines[2]) * cc;
	for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (uint64_t)gridDim.x * 256) {
		uint64_t id = at;
#pragma unroll
		for (int k = 0; k < 3; ++k) {
			const uint64_t n = (uint64_t)g.lines[k] * cc;
			if (id < n) {
				const uint32_t line = (uint32_t)(id / cc), c = (uint32_t)(id % cc) * 8;
				const T* p = g.from[k] + (uint64_t)line * g.ld[k];
				const int start = min((int)c, (int)g.width - 8);
				*(T8*)(g.to[k] + ((uint64_t)line * cc * 8 + c)) = shift8(load8_odd(p + start), c, g.width);
				break;
			}
			id -= n;
		}
	}
}
// what the products read: the caller's matrices, or (with `room` for them) packed ones; X and the weights as far as they are wanted
struct Operands { const T* x; const T* w[2]; uint64_t ld_x, ld_w; bool whole_x, whole_w; };
Operands operands(hipStream_t s, const DenseArgs& d, void* packed, bool room, bool want_x, bool want_w) {
	Operands o{(const T*)d.x, {(const T*)d.w[0], (const T*)d.w[1]}, d.x_stride, d.w_stride, whole(d.x, d.x_stride, d.k), whole(d.w[0], d.w_stride, d.k) && whole(d.w[1], d.w_stride, d.k)};
	const bool pack_x = room && want_x && !o.whole_x, pack_w = room && want_w && !o.whole_w;
	if (!pack_x && !pack_w) return o;
	PackArgs a{};
	const uint64_t k8 = up8(d.k);
	T* to = (T*)packed;
	uint64_t chunks = 0;
	auto pack = [&](int i, const T*& p, uint64_t lines, uint64_t ld) {
		if (!p) return;
		a.from[i] = p; a.ld[i] = ld; a.lines[i] = (uint32_t)lines; p = a.to[i] = to;
		to += lines * k8; chunks += lines * (k8 / 8);
	};
	a.width = d.k;
	if (pack_x) { pack(0, o.x, d.m, d.x_stride); o.ld_x = k8; }
	if (pack_w) { pack(1, o.w[0], d.n, d.w_stride); pack(2, o.w[1], d.n, d.w_stride); o.ld_w = k8; }
	if (chunks) hipLaunchKernelGGL(k_pack, dim3((uint32_t)std::min<uint64_t>((chunks + 255) / 256, PACK_BLOCKS)), dim3(256), 0, s, a);
	if (pack_x) o.whole_x = whole(o.x, o.ld_x, k8);
	if (pack_w) o.whole_w = whole(o.w[0], o.ld_w, k8) && whole(o.w[1], o.ld_w, k8);
	return o;
}
// threads that share the pieces of 8 sums: more for many pieces of few sums (56 x 56 of 512 pieces, with the bias: 6.4 us, 9.6 with 8; 256 x 256 of 256 the other way: 14.3 and 11.9)
int join_groups(const GemmArgs& g) { return g.splits >= 128 && (uint64_t)g.rows * up8(g.cols) * g.problems <= 1u << 14 ? 32 : g.splits >= 16 ? 8 : 1; }
uint32_t join_blocks(const GemmArgs& g) { return div_up((uint64_t)g.rows * (up8(g.cols) / 8), 256 / join_groups(g)) * g.problems; }
template <int EPI> void launch_join(hipStream_t s, GemmArgs g) { g.problems = 1; hipLaunchKernelGGL((k_join_splits<EPI>), dim3(join_blocks(g)), dim3(256), 0, s, g, join_groups(g)); }
template <int EPI> uint32_t tiles(const GemmArgs& g, uint32_t tile) { return div_up(g.rows, tile) * div_up(g.cols, tile / (GATED_TILE<EPI> ? 2 : 1)) * g.problems * g.splits; }
static_assert(TK == 64 && AK == 64, "splits are counted in chunks of 64 steps");
// `wholes`: both operands come in whole 16-byte pieces
template <bool A_T, bool B_T, int EPI> void launch_tiles(hipStream_t s, const GemmArgs& g, bool wholes, bool large) {
	const uint32_t n = tiles<EPI>(g, large ? 256 : 128);
	if (!wholes) hipLaunchKernelGGL((k_gemm<A_T, B_T, EPI>), dim3(n), dim3(256), 0, s, g);
	else if (large) {
		if constexpr (EPI != EPI_PARTIAL && EPI != EPI_PARTIAL2) hipLaunchKernelGGL((k_gemm_async<256, A_T, B_T, EPI, 2>), dim3(n), dim3(256), 0, s, g); // (large tiles are many: their sums are not split)
	} else if (n <= 256) hipLaunchKernelGGL((k_gemm_async<128, A_T, B_T, EPI, 4>), dim3(n), dim3(256), 0, s, g);
	else hipLaunchKernelGGL((k_gemm_async<128, A_T, B_T, EPI, 2>), dim3(n), dim3(256), 0, s, g);
}
// splits of a product; true: large tiles
bool set_split(GemmArgs& g, const DenseSplit& d, float* partial) {
	g.splits = d.splits; g.partial = partial;
	g.chunks_per_split = div_up(div_up(g.steps, 64) * g.segments, g.splits);
	return d.large;
}
template <int EPI> void launch_forward(hipStream_t s, GemmArgs& g, bool wholes, float* partial) {
	const bool large = set_split(g, dense_split(g.rows, g.cols, g.steps, 1, EPI == EPI_GATED ? 2 : 1), partial) && wholes;
	if (g.splits > 1) {
		launch_tiles<true, true, EPI == EPI_GATED ? EPI_PARTIAL2 : EPI_PARTIAL>(s, g, wholes, false);
		launch_join<EPI>(s, g);
	} else launch_tiles<true, true, EPI>(s, g, wholes, large);
}
void launch_finish(hipStream_t s, const GemmArgs* x, const GemmArgs* w, const BiasArgs& bias) {
	static const GemmArgs none{};
	if (!x) x = &none;
	if (!w) w = &none;
	const uint32_t bx = x->splits > 1 ? join_blocks(*x) : 0, bw = w->splits > 1 ? join_blocks(*w) : 0, bb = bias.partial ? div_up(bias.cols, 16) * bias.problems : 0;
	if (bx + bw + bb) hipLaunchKernelGGL(k_finish, dim3(bx + bw + bb), dim3(256), 0, s, *x, join_groups(*x), bx, *w, join_groups(*w), bw, bias);
}
bool odd_lines(const void* p, uint64_t ld) { return ((uintptr_t)p | ld * 2) & 3; }
template <int MT, int EPI> void launch_few_rows(hipStream_t s, GemmArgs& g, float* partial) {
	const DenseFewRows f = dense_few_rows(g.cols, g.steps);
	const dim3 grid(div_up(div_up(g.cols, 16), 8 / f.slices), f.splits);
	const uint32_t per = (div_up(g.steps, f.slices * f.splits) + 31) & ~31u;
	const bool odd = odd_lines(g.a, g.lda) || odd_lines(g.b[0], g.ldb) || odd_lines(g.b[1], g.ldb);
	g.splits = f.splits; g.partial = partial;
	constexpr int PART = EPI == EPI_GATED ? EPI_PARTIAL2 : EPI_PARTIAL;
	if (f.splits > 1) {
		if (odd) hipLaunchKernelGGL((k_few_rows<MT, PART, true>), grid, dim3(512), 0, s, g, f.slices, per); else hipLaunchKernelGGL((k_few_rows<MT, PART, false>), grid, dim3(512), 0, s, g, f.slices, per);
		launch_join<EPI>(s, g);
	} else if (odd) hipLaunchKernelGGL((k_few_rows<MT, EPI, true>), grid, dim3(512), 0, s, g, f.slices, per);
	else hipLaunchKernelGGL((k_few_rows<MT, EPI, false>), grid, dim3(512), 0, s, g, f.slices, per);
}
template <int NF, int KS, int EPI, bool EXCHANGE> void launch_narrow_forward_nk(hipStream_t s, const GemmArgs& g, uint32_t blocks) {
	if (odd_lines(g.a, g.lda)) hipLaunchKernelGGL((k_narrow_forward<NF, KS, EPI, EXCHANGE, true>), dim3(blocks), dim3(512), 0, s, g);
	else hipLaunchKernelGGL((k_narrow_forward<NF, KS, EPI, EXCHANGE, false>), dim3(blocks), dim3(512), 0, s, g);
}
template <int NF, int EPI, bool EXCHANGE> void launch_narrow_forward_n(hipStream_t s, const GemmArgs& g, uint32_t blocks) {
	if (g.steps <= 64) launch_narrow_forward_nk<NF, 2, EPI, EXCHANGE>(s, g, blocks);
	else if (g.steps <= 128) launch_narrow_forward_nk<NF, 4, EPI, EXCHANGE>(s, g, blocks);
	else if (NF > 4 || g.steps <= 256) launch_narrow_forward_nk<NF, 8, EPI, EXCHANGE>(s, g, blocks);
	else if constexpr (NF == 4) launch_narrow_forward_nk<NF, 16, EPI, EXCHANGE>(s, g, blocks);
}
template <int EPI, bool EXCHANGE> void launch_narrow_forward(hipStream_t s, const GemmArgs& g) {
	const uint32_t cols = g.cols * (EPI == EPI_GATED ? 2 : 1), blocks = std::min(div_up(g.rows, 128), 512u);
	if (cols <= 64) { if constexpr (!(EXCHANGE && EPI == EPI_GATED)) launch_narrow_forward_n<4, EPI, EXCHANGE>(s, g, blocks); } // (up to 32 gated outputs: one piece, nothing to exchange)
	else if (cols <= 128) launch_narrow_forward_n<8, EPI, EXCHANGE>(s, g, blocks); else launch_narrow_forward_n<16, EPI, EXCHANGE>(s, g, std::min(blocks, g.steps > 128 ? 256u : 512u));
}
template <int NF, int KF, bool GATED> void launch_narrow_backward_nk(hipStream_t s, const NarrowArgs& a, uint32_t blocks) {
	hipLaunchKernelGGL((k_narrow_backward<NF, KF, GATED>), dim3(blocks), dim3(512), 0, s, a);
}
template <int NF, bool GATED> void launch_narrow_backward_n(hipStream_t s, const NarrowArgs& a, uint32_t blocks) {
	if (a.k <= 64) launch_narrow_backward_nk<NF, 4, GATED>(s, a, blocks); else if (a.k <= 128) launch_narrow_backward_nk<NF, 8, GATED>(s, a, blocks); else launch_narrow_backward_nk<NF, 16, GATED>(s, a, blocks);
}
template <bool GATED> void launch_narrow_backward(hipStream_t s, const NarrowArgs& a, uint32_t blocks) {
	const uint32_t cols = a.n * (GATED ? 2 : 1);
	if (cols <= 64) launch_narrow_backward_n<4, GATED>(s, a, blocks); else if (cols <= 128) launch_narrow_backward_n<8, GATED>(s, a, blocks); else launch_narrow_backward_n<16, GATED>(s, a, blocks);
}
} // namespace

void DENSE_NAME(launch_dense_forward)(hipStream_t s, const DenseArgs& d) {
	if (!d.m || !d.n) return;
	GemmArgs g{};
	g.a = (const T*)d.x; g.lda = d.x_stride; g.ldb = d.w_stride;
	g.rows = d.m; g.cols = d.n; g.steps = d.k; g.segments = 1; g.problems = 1;
	for (int i = 0; i < 2; ++i) { g.b[i] = (const T*)d.w[i]; g.bias[i] = (const T*)d.bias[i]; g.pre[i] = (T*)d.pre[i]; }
	g.c[0] = (T*)d.y; g.ldc = d.y_stride; g.act = d.act; g.residual = (const T*)d.residual; g.ld_residual = d.residual_stride; g.ld_pre = d.pre_stride;
	// Outputs that the 256 MB of the last cache would not hold beside the inputs go past the caches (262144 x 256 from 64 inputs: 95 -> 78 us; 8192 x 4096 x 2 from 4096: 237 -> 230 us; 72112 x 1894
	// from 1224: 405 -> 365 us); smaller ones stay there for their readers (65521 x 256 x 2 from 63: 23 us then, past the caches 25 us).  Narrow layers' only in whole cache lines,
	// which the caches need not join (262144 x 256 x 2 at a stride of 264: 165 us, 246 us past the caches).
	const bool large = g.streamed = (uint64_t)d.m * d.n * 2 * (1 + (d.pre[0] != nullptr) + (d.pre[1] != nullptr)) >= 128ull << 20;
	float* partial = (float*)d.workspace;
	if (d.m <= FEW_ROWS && d.k) {
		if (d.m <= 16) { if (d.gated) launch_few_rows<1, EPI_GATED>(s, g, partial); else launch_few_rows<1, EPI_LINEAR>(s, g, partial); }
		else { if (d.gated) launch_few_rows<2, EPI_GATED>(s, g, partial); else launch_few_rows<2, EPI_LINEAR>(s, g, partial); }
		return;
	}
	if (dense_narrow_forward(d.m, d.n, d.k, d.gated)) {
		g.streamed &= (((uintptr_t)d.y | (uintptr_t)d.pre[0] | (uintptr_t)d.pre[1] | d.y_stride * 2 | (d.pre[0] || d.pre[1] ? d.pre_stride * 2 : 0)) & 127) == 0;
		if (large && d.n > 32) { if (d.gated) launch_narrow_forward<EPI_GATED, true>(s, g); else launch_narrow_forward<EPI_LINEAR, true>(s, g); }
		else { if (d.gated) launch_narrow_forward<EPI_GATED, false>(s, g); else launch_narrow_forward<EPI_LINEAR, false>(s, g); }
		return;
	}
	const uint64_t room = dense_pack_bytes(d.m, d.n, d.k, d.gated, false);
	const Operands o = operands(s, d, (char*)d.workspace + dense_forward_bytes(d.m, d.n, d.k, d.gated) - room, room != 0, true, true);
	const bool wholes = o.whole_x && o.whole_w;
	g.a = o.x; g.lda = o.ld_x; g.b[0] = o.w[0]; g.b[1] = o.w[1]; g.ldb = o.ld_w;
	if (d.gated) launch_forward<EPI_GATED>(s, g, wholes, partial); else launch_forward<EPI_LINEAR>(s, g, wholes, partial);
}
void DENSE_NAME(launch_dense_backward)(hipStream_t s, const DenseArgs& d) {
	const DensePlan p = dense_plan(d.m, d.n, d.k, d.gated);
	const uint32_t problems = d.gated ? 2 : 1;
	char* ws = (char*)d.workspace;
	const bool bias = d.dbias[0] || d.dbias[1];
	const bool none = !d.gated && d.act == NGP_ACT_NONE;
	// G is dY as it stands, unless the products are worth a padded copy (14724 x 7414 from 2072 inputs: 1525 us without, 1198 us; 2000 x 1001 from 1000: 39.7, 29.8 us)
	const bool identity = none && (whole(d.dy, d.dy_stride, d.n) || (double)d.m * d.n * d.k < 1e8);
	const bool products = d.dx || d.dw[0] || d.dw[1];
	if ((products || bias) && dense_narrow_backward(d.m, d.n, d.k, d.gated)) {
		NarrowArgs a{};
		a.rows = d.m; a.n = d.n; a.k = d.k; a.act = d.act; a.x = (const T*)d.x; a.ld_x = d.x_stride; a.ld_w = d.w_stride; a.ld_pre = d.pre_stride; a.dy = (const T*)d.dy; a.ld_dy = d.dy_stride;
		for (int i = 0; i < 2; ++i) { a.w[i] = (const T*)d.w[i]; a.pre[i] = (const T*)d.pre[i]; }
		if (none) { a.pre[0] = a.dy; a.ld_pre = a.ld_dy; } // (read, not used)
		if (!d.dw[0]) { a.x = a.dy; a.ld_x = 0; }              // (dW is not wanted: something to read in the place of X, where nothing looks)
		a.dx = (T*)d.dx; a.ld_dx = d.dx_stride; a.partial = d.dw[0] ? (float*)(ws + p.partial) : nullptr; a.bias_partial = bias ? (float*)(ws + p.bias) : nullptr;
		if (d.gated) launch_narrow_backward<true>(s, a, p.row_blocks); else launch_narrow_backward<false>(s, a, p.row_blocks);
		GemmArgs w{};
		w.rows = d.n; w.cols = d.k; w.problems = problems; w.splits = p.row_blocks; w.partial = a.partial; w.c[0] = (T*)d.dw[0]; w.c[1] = (T*)d.dw[1]; w.ldc = d.dw_stride;
		BiasArgs b{a.bias_partial, p.row_blocks, d.n, problems, {(T*)d.dbias[0], (T*)d.dbias[1]}};
		launch_finish(s, nullptr, a.partial ? &w : nullptr, b);
		return;
	}
	const uint32_t terms = !none && dense_two_terms(d.m, d.n, d.k) ? 2 : 1;
	const T* G = (const T*)d.dy; uint64_t ldg = d.dy_stride;
	BiasArgs b{nullptr, p.row_blocks, d.n, problems, {(T*)d.dbias[0], (T*)d.dbias[1]}};
	if ((!identity && products) || bias) {
		GradArgs a{};
		a.rows = d.m; a.cols = d.n; a.act = d.act; a.dy = (const T*)d.dy; a.ld_dy = d.dy_stride; a.pre[0] = (const T*)d.pre[0]; a.pre[1] = (const T*)d.pre[1]; a.ld_pre = d.pre_stride;
		if (none) a.pre[0] = nullptr;
		a.out = products && !identity ? (T*)(ws + p.grad) : nullptr; a.ld_out = (uint64_t)up8(d.n) * problems * terms; a.two_terms = terms == 2; a.rows_per_block = p.rows_per_block;
		if (p.row_blocks > 1) a.bias_partial = bias ? (float*)(ws + p.bias) : nullptr; else for (int k = 0; k < 2; ++k) a.dbias[k] = (T*)d.dbias[k];
		if (a.out) { G = a.out; ldg = a.ld_out; }
		const uint32_t cols = dense_grad_cols(d.m, d.n);
		const dim3 grid(div_up(d.n, cols), std::max(1u, p.row_blocks)); // (no samples: the bias's gradient is zero)
		if (d.n) {
			if (cols > 256) { if (d.gated) hipLaunchKernelGGL((k_output_grad<true, 1024>), grid, dim3(256), 0, s, a); else hipLaunchKernelGGL((k_output_grad<false, 1024>), grid, dim3(256), 0, s, a); }
			else { if (d.gated) hipLaunchKernelGGL((k_output_grad<true, 256>), grid, dim3(256), 0, s, a); else hipLaunchKernelGGL((k_output_grad<false, 256>), grid, dim3(256), 0, s, a); }
		}
		b.partial = a.bias_partial;
	}
	const bool g_whole = whole(G, ldg, G == d.dy ? d.n : 8); // (the workspace's lines are padded with zeros)
	GemmArgs x{}, w{};
	bool large_x = false, large_w = false;
	const bool want_x = d.dx && d.m && d.k, want_w = d.dw[0] && d.n && d.k;
	const Operands o = want_x || want_w ? operands(s, d, ws + p.pack, p.bytes > p.pack, want_w, want_x) : Operands{}; // (dW reads X, dX the weights)
	const bool whole_x = g_whole && o.whole_w, whole_w = g_whole && o.whole_x;
	if (want_x) {
		x.a = G; x.lda = ldg; x.a_segment = up8(d.n); x.segments = problems * terms; x.b[0] = o.w[0]; x.b[1] = d.gated ? o.w[1] : o.w[0]; x.ldb = o.ld_w;
		x.rows = d.m; x.cols = d.k; x.steps = d.n; x.problems = 1; x.c[0] = (T*)d.dx; x.ldc = d.dx_stride;
		large_x = set_split(x, dense_split(d.m, d.k, d.n, problems * terms, 1), (float*)(ws + p.partial_x)) && whole_x;
	}
	if (want_w) {
		w.a = G; w.lda = ldg; w.a_problem = up8(d.n); w.problems = problems; w.b[0] = w.b[1] = o.x; w.ldb = o.ld_x;
		w.rows = d.n; w.cols = d.k; w.steps = d.m; w.segments = terms; w.a_segment = (uint64_t)up8(d.n) * problems; w.c[0] = (T*)d.dw[0]; w.c[1] = (T*)d.dw[1]; w.ldc = d.dw_stride;
		large_w = set_split(w, dense_split_dw(d.m, d.n, d.k, problems, terms), (float*)(ws + p.partial)) && whole_w;
	}
	if (want_x && want_w && !large_x && !large_w && whole_x == whole_w) {
		const uint32_t bx = tiles<EPI_STORE>(x, 128), bw = tiles<EPI_STORE>(w, 128);
		const bool w_first = w.chunks_per_split > x.chunks_per_split;
		if (!whole_x) hipLaunchKernelGGL(k_products, dim3(bx + bw), dim3(256), 0, s, x, w, bx, bw, w_first);
		else if (bx + bw <= 256) hipLaunchKernelGGL(k_products_async<4>, dim3(bx + bw), dim3(256), 0, s, x, w, bx, bw, w_first);
		else hipLaunchKernelGGL(k_products_async<2>, dim3(bx + bw), dim3(256), 0, s, x, w, bx, bw, w_first);
	} else {
		if (want_x) launch_tiles<true, false, EPI_STORE>(s, x, whole_x, large_x);
		if (want_w) launch_tiles<false, false, EPI_STORE>(s, w, whole_w, large_w);
	}
	launch_finish(s, &x, &w, b);
}
} // namespace ngp
