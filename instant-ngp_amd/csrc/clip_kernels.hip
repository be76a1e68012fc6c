// clip_kernels.hip -- the norm of a gradient that lies in many tensors, and its clipping (ngp_gradient_norm, ngp_clip_gradients).
//   norm = sqrt(sum of g^2 over all tensors) / loss_scale;   c = max_norm / norm where norm > max_norm, else 1;   clipped = c g
// Memory bound: one pass reads every gradient for the sum, one reads and writes it (nothing is written in place where c = 1): 400 M bfloat16 in 300 tensors 515 us, 4.7 TB/s over the
// three; 12.2 M half in 9 tensors 18 us; 7168 elements 8.5 us, a launch.  The tensors' table travels in the
// kernel arguments (no upload that a captured graph would have to keep alive), TABLE tensors a launch.  Every block owns a contiguous range of the tensors' chunks;
// the second pass takes launches and ranges backwards, so that it begins with what the first one left in the caches.  Up to SMALL elements in
// FEW tensors one block does it all, in one launch: 4096 elements in 2 tensors 4.2 us against 9.7, in 8 tensors, one after the other, 8.0 against 7.4, in 100 48 against 11.  Sums are double, in a fixed order: the result
// does not depend on timing, and squares of any bfloat16 / float fit.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <algorithm>
#include <vector>
#include "ngp_kernels.hpp"

namespace ngp {
namespace {
constexpr uint32_t TABLE = 112, CHUNK = 8192, THREADS = 256, SMALL = 65536, FEW = 8;
struct ClipTable { const void* grad[TABLE]; void* clipped[TABLE]; uint64_t size[TABLE]; uint32_t first[TABLE + 1]; uint8_t type[TABLE]; uint32_t n; };
struct Range { uint32_t begin, end; };
__device__ inline Range block_range(uint32_t chunks) {
	return {(uint32_t)((uint64_t)chunks * blockIdx.x / gridDim.x), (uint32_t)((uint64_t)chunks * (blockIdx.x + 1) / gridDim.x)};
}
__device__ inline uint32_t tensor_of(const ClipTable& t, uint32_t chunk) { // last tensor whose first chunk is at or before `chunk` (empty tensors have none)
	uint32_t lo = 0, hi = t.n;
	while (hi - lo > 1) { const uint32_t mid = (lo + hi) / 2; if (t.first[mid] <= chunk) lo = mid; else hi = mid; }
	return lo;
}
template <typename T, int N> struct Vec { T v[N]; };
// elements in front of the first 16-byte boundary of p, n at most (a tensor begins wherever its elements allow)
template <typename T> __device__ inline uint32_t head_of(const T* p, uint32_t n) { return min(n, (uint32_t)(-(uintptr_t)p & 15) / (uint32_t)sizeof(T)); }
template <uint32_t THREADS, typename T> __device__ inline double sum_squares(const T* p, uint32_t n) {
	constexpr int N = 16 / sizeof(T);
	const uint32_t head = head_of(p, n);
	double s = 0;
	if (threadIdx.x < head) { const double d = (double)(float)p[threadIdx.x]; s = d * d; }
	p += head; n -= head;
	const uint32_t tail = n % N;
	if (threadIdx.x >= THREADS - tail) { const double d = (double)(float)p[n - (THREADS - threadIdx.x)]; s = fma(d, d, s); } // (one element a thread: a loop waits for every load)
#pragma unroll 4
	for (uint32_t i = threadIdx.x * N; i + N <= n; i += THREADS * N) {
		Vec<T, N> v;
		__builtin_memcpy(&v, __builtin_assume_aligned(p + i, 16), 16);
#pragma unroll
		for (int e = 0; e < N; ++e) { const double d = (double)(float)v.v[e]; s = fma(d, d, s); }
	}
	return s;
}
// C: float, or double for factors below what a float holds in full (1e-3 / 1e37: g c is an ordinary number, c is not)
template <uint32_t THREADS, typename C, typename T> __device__ inline void scale(const T* p, T* q, uint32_t n, C c) {
	constexpr int N = 16 / sizeof(T);
	const uint32_t head = head_of(q, n); // (whole lines are written; p has the same alignment or is read across it)
	if (threadIdx.x < head) q[threadIdx.x] = (T)(float)((C)(float)p[threadIdx.x] * c);
	p += head; q += head; n -= head;
	const uint32_t tail = n % N;
	if (threadIdx.x >= THREADS - tail) { const uint32_t i = n - (THREADS - threadIdx.x); q[i] = (T)(float)((C)(float)p[i] * c); }
#pragma unroll 4
	for (uint32_t i = threadIdx.x * N; i + N <= n; i += THREADS * N) {
		Vec<T, N> v;
		__builtin_memcpy(&v, p + i, 16);
#pragma unroll
		for (int e = 0; e < N; ++e) v.v[e] = (T)(float)((C)(float)v.v[e] * c); // rounded once, to the gradient's own type
		typedef float f4 __attribute__((ext_vector_type(4)));
		__builtin_nontemporal_store(__builtin_bit_cast(f4, v), (f4*)(q + i)); // (not wanted again: the caches keep gradients that are still to be read)
	}
}
template <uint32_t THREADS> __device__ inline double sum_tensor(int type, const void* p, uint64_t at, uint32_t n) {
	switch (type) {
		case NGP_TYPE_HALF: return sum_squares<THREADS>((const _Float16*)p + at, n);
		case NGP_TYPE_BFLOAT16: return sum_squares<THREADS>((const __bf16*)p + at, n);
		default: return sum_squares<THREADS>((const float*)p + at, n);
	}
}
template <uint32_t THREADS, typename C> __device__ inline void scale_typed(int type, const void* p, void* q, uint64_t at, uint32_t n, C c) {
	switch (type) {
		case NGP_TYPE_HALF: scale<THREADS>((const _Float16*)p + at, (_Float16*)q + at, n, c); break;
		case NGP_TYPE_BFLOAT16: scale<THREADS>((const __bf16*)p + at, (__bf16*)q + at, n, c); break;
		default: scale<THREADS>((const float*)p + at, (float*)q + at, n, c); break;
	}
}
template <uint32_t THREADS> __device__ inline void scale_tensor(int type, const void* p, void* q, uint64_t at, uint32_t n, double c) {
	if (c >= 1.17549435e-38) scale_typed<THREADS>(type, p, q, at, n, (float)c); else scale_typed<THREADS>(type, p, q, at, n, c);
}
template <uint32_t THREADS = 256> __device__ inline double block_sum(double s) { // the sum over the block, in every thread
	__shared__ double red[THREADS / 64];
#pragma unroll
	for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
	__syncthreads();
	if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
	__syncthreads();
	s = 0;
#pragma unroll
	for (uint32_t i = 0; i < THREADS / 64; ++i) s += red[i];
	return s;
}
// max_norm / norm where the norm is beyond it and finite as the caller sees it, in 32 bits; itself a 32-bit number unless it is too small for one
__device__ inline double clip_factor(double norm, float max_norm) {
	if (!((float)norm <= 3.402823466e38f && norm > (double)max_norm)) return 1.0;
	const double c = (double)max_norm / norm;
	return c >= 1.17549435e-38 ? (double)(float)c : c;
}
__global__ __launch_bounds__(THREADS) void k_norm_partial(ClipTable t, double* slots, uint32_t written) {
	const Range r = block_range(t.first[t.n]);
	double s = 0;
	uint32_t i = r.begin < r.end ? tensor_of(t, r.begin) : 0;
	for (uint32_t k = r.begin; k < r.end; ++k) {
		while (t.first[i + 1] <= k) ++i;
		const uint64_t at = (uint64_t)(k - t.first[i]) * CHUNK, left = t.size[i] - at;
		const uint32_t n = left < CHUNK ? (uint32_t)left : CHUNK;
		s += sum_tensor<THREADS>(t.type[i], t.grad[i], at, n);
	}
	s = block_sum(s);
	if (threadIdx.x == 0) slots[blockIdx.x] = (blockIdx.x < written ? slots[blockIdx.x] : 0.0) + s;
}
__device__ inline double norm_of(const double* slots, uint32_t n_slots, float loss_scale) {
	double s = 0;
	for (uint32_t i = threadIdx.x; i < n_slots; i += THREADS) s += slots[i];
	return sqrt(block_sum(s)) / (double)loss_scale;
}
__global__ __launch_bounds__(THREADS) void k_norm_finish(const double* slots, uint32_t n_slots, float loss_scale, float* norm) {
	const double v = norm_of(slots, n_slots, loss_scale);
	if (threadIdx.x == 0) *norm = (float)v;
}
__global__ __launch_bounds__(THREADS) void k_clip(ClipTable t, const double* slots, uint32_t n_slots, float loss_scale, float max_norm, float* norm) {
	const double v = norm_of(slots, n_slots, loss_scale);
	if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
	const double c = clip_factor(v, max_norm);
	const Range r = block_range(t.first[t.n]);
	if (r.begin >= r.end) return;
	uint32_t i = tensor_of(t, r.end - 1);
	for (uint32_t k = r.end; k-- > r.begin;) {
		while (t.first[i] > k) --i;
		if (!t.clipped[i] || (c == 1.0 && t.clipped[i] == t.grad[i])) continue;
		const uint64_t at = (uint64_t)(k - t.first[i]) * CHUNK, left = t.size[i] - at;
		const uint32_t n = left < CHUNK ? (uint32_t)left : CHUNK;
		scale_tensor<THREADS>(t.type[i], t.grad[i], t.clipped[i], at, n, c);
	}
}
// all of it by one block
__global__ __launch_bounds__(1024) void k_clip_small(ClipTable t, float loss_scale, float max_norm, float* norm) {
	double s = 0;
	for (uint32_t i = 0; i < t.n; ++i) s += sum_tensor<1024>(t.type[i], t.grad[i], 0, (uint32_t)t.size[i]);
	const double v = sqrt(block_sum<1024>(s)) / (double)loss_scale;
	if (threadIdx.x == 0) *norm = (float)v;
	const double c = clip_factor(v, max_norm);
	for (uint32_t i = 0; i < t.n; ++i)
		if (t.clipped[i] && !(c == 1.0 && t.clipped[i] == t.grad[i])) scale_tensor<1024>(t.type[i], t.grad[i], t.clipped[i], 0, (uint32_t)t.size[i], c);
}
} // namespace

void launch_gradient_norm(hipStream_t s, uint32_t n, const ngp_gradient* tensors, float loss_scale, bool clip, float max_norm, float* norm, double* slots) {
	// the tensors in tables of at most TABLE (a table's chunks fit 31 bits; one tensor alone does: checked at the entry point)
	auto table = [&](uint32_t& i, ClipTable& t) { // from tensor i on; i: the first one that is left
		t.n = 0; t.first[0] = 0;
		for (; i < n && t.n < TABLE; ++i) {
			if (!tensors[i].size) continue;
			const uint64_t chunks = (tensors[i].size + CHUNK - 1) / CHUNK;
			if (t.n && t.first[t.n] + chunks > 0x7fffffffull) break;
			t.grad[t.n] = tensors[i].grad; t.clipped[t.n] = clip ? tensors[i].clipped : nullptr; t.size[t.n] = tensors[i].size; t.type[t.n] = (uint8_t)tensors[i].type;
			t.first[t.n + 1] = t.first[t.n] + (uint32_t)chunks; ++t.n;
		}
	};
	ClipTable t;
	uint64_t total = 0;
	for (uint32_t i = 0; i < n && total <= SMALL; ++i) total += tensors[i].size;
	uint32_t i = 0;
	if (total <= SMALL) {
		table(i, t);
		if (i >= n && t.n <= FEW) { hipLaunchKernelGGL(k_clip_small, dim3(1), dim3(1024), 0, s, t, loss_scale, max_norm, norm); return; }
		i = 0;
	}
	std::vector<uint32_t> starts; // first tensor of each table
	uint32_t written = 0;         // slots
	while (i < n) {
		const uint32_t from = i;
		table(i, t);
		if (!t.n) { table(i = starts.back(), t); break; } // (only empty ones were left)
		starts.push_back(from);
		const uint32_t blocks = std::min(t.first[t.n], CLIP_SLOTS);
		hipLaunchKernelGGL(k_norm_partial, dim3(blocks), dim3(THREADS), 0, s, t, slots, written);
		written = std::max(written, blocks);
	}
	if (!clip) { hipLaunchKernelGGL(k_norm_finish, dim3(1), dim3(THREADS), 0, s, slots, written, loss_scale, norm); return; }
	for (size_t k = starts.size(); k-- > 0;) { // the last table first (it is still there)
		i = starts[k];
		if (k + 1 < starts.size()) table(i, t);
		hipLaunchKernelGGL(k_clip, dim3(std::min(t.first[t.n], CLIP_SLOTS)), dim3(THREADS), 0, s, t, slots, written, loss_scale, max_norm, k + 1 == starts.size() ? norm : nullptr);
	}
}
} // namespace ngp
