// Products in double for the vocabulary head's way through Gram matrices (vocab.hip): C = A^H diag(weight) A, and C = conj(A) G with
// such a G.  The operands A are fp32 planes, G and all sums are double.
//
// Why double: what the head takes from a Gram matrix (a row's sum |z|^2, the gradients) is small where the rows of A lie in
// directions that the other operand hardly has, while the terms it is summed from are not.  Products of two fp32 numbers are exact
// in double, and 29 bits to spare cover every such difference that the logits themselves would still show (whose fp32 sums lose
// all digits long before).
//
// One workgroup of eight wavefronts forms 64 x 64 of C, each 32 x 16 of it with v_mfma_f64_16x16x4_f64, K in chunks of 16 through two
// buffers of LDS.  Three real products per complex one (with a' = conj(a): Re = ar br - ai' bi, Im = (ar + ai')(br + bi) - ar br - ai' bi;
// the differences cost a few of the bits to spare).
// Bound by the matrix pipe: 64 cycles an instruction, 128 flop a cycle and compute unit, half of what fp32 has.  A loop of nothing else
// reaches 75.7 TFLOP/s; 1024 columns over 32768 rows take 1.74 ms and 32768 rows times 1024 x 1024 3.23 ms, 63 and 64 TFLOP/s (of three products).
// With 64 cycles an instruction everything else has time (32 bytes of LDS a cycle and compute unit, accesses of 4 and 8 bytes whatever
// the operands' alignment); what is lost is lost at the barriers, hence eight wavefronts of 32 x 16, four to a SIMD with a second workgroup
// beside (four of 32 x 32: 3.39 ms).
#include "common.hpp"
#include "gram.hpp"
#include "rows.hpp"

#include <algorithm>
#include <cmath>

namespace {

using namespace cnet::rows;
using cnet::Gram64;
using cnet::GramOut;

constexpr int TPB = 512, EACH = cnet::GRAM_TILE * cnet::GRAM_CHUNK / TPB;  // EACH: elements of a chunk's plane per thread
constexpr int JOIN_TPB = 1024;
constexpr int BT = cnet::GRAM_TILE, KC = cnet::GRAM_CHUNK;
// (66: with a row-major operand 16 lanes write 16 different k of one row, 132 words apart: all 64 banks; the reads go two ways)
constexpr int LD = BT + 2;

typedef double double4_t __attribute__((ext_vector_type(4)));

struct Stage {
	double v[2][2][KC][LD];  // [A, B][re, im][k][row of A / column of B]
};

// rows m0 .. of the block's part of A (or columns, KMAJOR), columns n0 .. of B, and the end of what is summed over
template <class TB>
struct Tile {
	const float *a_re, *a_im;
	const TB *b_re, *b_im;
	const double *weight;  // of the rows of A and B
	long lda, ldb;
	int M, N, m0, n0, k_end;
};

struct Sums {
	double4_t p1[2], p2[2], p3[2];  // ar br, ai' bi, (ar + ai')(br + bi)
};

// p[offset], offset counted in elements; uniform p and 32-bit offsets make one address register of it
template <class T, class Off>
__device__ __forceinline__ T at_offset(const T *p, Off offset) {
	return *reinterpret_cast<const T *>(reinterpret_cast<const char *>(p) + offset * (Off) sizeof(T));
}

// The sum over k from k0 (a multiple of KC) to t.k_end.  What lies behind k_end is zero in both operands; rows and columns beyond M and N repeat
// the last ones, and nobody stores what comes of them.  KMAJOR: A is given as [k][m] like B.  Off: what holds a block's offsets into its operands.
// Addresses are uniform bases with constant offsets and only the last chunk looks at the bounds (looked at in every one: 6 % slower).
template <bool KMAJOR, bool WEIGHT, class TB, class Off>
__device__ __forceinline__ void tile_product(const Tile<TB> &t, int k0, Stage (&st)[2], Sums &s) {
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 2, wn = wave & 3, r = lane & 15, q = lane >> 4;
#pragma unroll
	for (int i = 0; i < 2; ++i) s.p1[i] = s.p2[i] = s.p3[i] = double4_t{0.0, 0.0, 0.0, 0.0};
	// element i of a thread: k-major operands: column tid % 64, k = tid / 64 + 4 i; row-major: k = tid % 16, row tid / 16 + 16 i
	const int m = min(tid % BT, t.M - 1 - t.m0), n = min(tid % BT, t.N - 1 - t.n0);
	Off a_off[EACH], b_off[EACH];
	// (the k of element i, counted from the chunk's first; behind k_end the last one again)
	auto offsets = [&](int left) {
#pragma unroll
		for (int i = 0; i < EACH; ++i) {
			const int kb = min(tid / BT + TPB / BT * i, left - 1), ka = min(tid % KC, left - 1);
			a_off[i] = KMAJOR ? (Off) kb * (Off) t.lda + (Off) m : (Off) min(tid / KC + TPB / KC * i, t.M - 1 - t.m0) * (Off) t.lda + (Off) ka;
			b_off[i] = (Off) kb * (Off) t.ldb + (Off) n;
		}
	};
	struct Operands {
		float a_r[EACH], a_i[EACH];
		TB b_r[EACH], b_i[EACH];
		double g[EACH];
	} chunk[2];
	auto fetch = [&](Operands &o, int k) {
		if (t.k_end - k < KC) offsets(t.k_end - k);
		const long a = KMAJOR ? (long) k * t.lda + t.m0 : (long) t.m0 * t.lda + k, b = (long) k * t.ldb + t.n0;
#pragma unroll
		for (int i = 0; i < EACH; ++i) {
			o.a_r[i] = at_offset(t.a_re + a, a_off[i]);
			o.a_i[i] = at_offset(t.a_im + a, a_off[i]);
			o.b_r[i] = at_offset(t.b_re + b, b_off[i]);
			o.b_i[i] = at_offset(t.b_im + b, b_off[i]);
			if (WEIGHT) o.g[i] = t.weight[min(k + tid / BT + TPB / BT * i, t.k_end - 1)];
		}
	};
	auto put_stage = [&](Stage &to, Operands &o, int k) {
		if (t.k_end - k < KC) {
#pragma unroll
			for (int i = 0; i < EACH; ++i) {
				const bool in_b = k + tid / BT + TPB / BT * i < t.k_end, in_a = KMAJOR ? in_b : k + tid % KC < t.k_end;
				if (!in_a) o.a_r[i] = o.a_i[i] = 0.f;
				if (!in_b) o.b_r[i] = o.b_i[i] = (TB) 0;
			}
		}
#pragma unroll
		for (int i = 0; i < EACH; ++i) {
			const int kb = tid / BT + TPB / BT * i, ka = KMAJOR ? kb : tid % KC, row = KMAJOR ? tid % BT : tid / KC + TPB / KC * i;
			if (WEIGHT && o.g[i] == 0.0) o.a_r[i] = o.a_i[i] = o.b_r[i] = o.b_i[i] = (TB) 0;  // left out whatever the row holds
			const double x = (double) o.a_r[i], y = -(double) o.a_i[i];
			to.v[0][0][ka][row] = WEIGHT ? x * o.g[i] : x;
			to.v[0][1][ka][row] = WEIGHT ? y * o.g[i] : y;
			to.v[1][0][kb][tid % BT] = (double) o.b_r[i];
			to.v[1][1][kb][tid % BT] = (double) o.b_i[i];
		}
	};
	auto multiply = [&](const Stage &from, int step) {
		const double br = from.v[1][0][4 * step + q][16 * wn + r], bi = from.v[1][1][4 * step + q][16 * wn + r], bs = br + bi;
		double ar[2], ai[2];
#pragma unroll
		for (int i = 0; i < 2; ++i) {
			ar[i] = from.v[0][0][4 * step + q][32 * wm + 16 * i + r];
			ai[i] = from.v[0][1][4 * step + q][32 * wm + 16 * i + r];
		}
#pragma unroll
		for (int i = 0; i < 2; ++i) {
			s.p1[i] = __builtin_amdgcn_mfma_f64_16x16x4f64(ar[i], br, s.p1[i], 0, 0, 0);
			s.p2[i] = __builtin_amdgcn_mfma_f64_16x16x4f64(ai[i], bi, s.p2[i], 0, 0, 0);
			s.p3[i] = __builtin_amdgcn_mfma_f64_16x16x4f64(ar[i] + ai[i], bs, s.p3[i], 0, 0, 0);
		}
	};
	// Chunk k is multiplied from one buffer of LDS; chunk k + 1 lies in registers and goes to the other buffer (last read before this chunk's
	// barrier) while the last matrix instructions are under way; chunk k + 2 is requested.
	auto round = [&](int k, const Stage &from, Stage &to, Operands &next, Operands &after) {
		__syncthreads();
		if (k + 2 * KC < t.k_end) fetch(after, k + 2 * KC);
		__builtin_amdgcn_sched_barrier(0);  // (the loads go out before the products, not after them)
#pragma unroll
		for (int step = 0; step < KC / 4 - 1; ++step) multiply(from, step);
		__builtin_amdgcn_sched_barrier(0);
		if (k + KC < t.k_end) put_stage(to, next, k + KC);
		multiply(from, KC / 4 - 1);
	};
	offsets(KC);
	fetch(chunk[0], k0);
	if (k0 + KC < t.k_end) fetch(chunk[1], k0 + KC);
	put_stage(st[0], chunk[0], k0);
	for (int k = k0; k < t.k_end; k += 2 * KC) {
		round(k, st[0], st[1], chunk[1], chunk[0]);
		if (k + KC < t.k_end) round(k + KC, st[1], st[0], chunk[0], chunk[1]);
	}
}

// calls f(row, column, i, e, re, im) for a lane's 8 elements of the block: element e of tile i is row 4 e + lane / 16, column lane % 16
template <class F>
__device__ __forceinline__ void each_element(const Sums &s, int m0, int n0, F f) {
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
	for (int i = 0; i < 2; ++i)
#pragma unroll
		for (int e = 0; e < 4; ++e)
			f(m0 + 32 * (wave >> 2) + 16 * i + 4 * e + (lane >> 4), n0 + 16 * (wave & 3) + (lane & 15), i, e, s.p1[i][e] - s.p2[i][e],
					s.p3[i][e] - s.p1[i][e] - s.p2[i][e]);
}

// C = A^H diag(weight) A [K][K] over the rows [split * per, ..) of A, blocks on and above the diagonal: blockIdx.x counts them column by
// column, blockIdx.y the shares of the rows, each with planes of its own in `part`.
template <bool WEIGHT, class Off>
__global__ __launch_bounds__(TPB, 4) void gram_kernel(const float *a_re, const float *a_im, long lda, const double *weight, int K, int L, int per,
		double *__restrict__ part, long plane, long ldc) {
	__shared__ Stage st[2];
	const int pid = blockIdx.x;
	int j = (int) ((sqrtf(8.0f * (float) pid + 1.0f) - 1.0f) * 0.5f);  // block column j starts at number j (j + 1) / 2
	while (j * (j + 1) / 2 > pid) --j;
	while ((j + 1) * (j + 2) / 2 <= pid) ++j;
	const int m0 = (pid - j * (j + 1) / 2) * BT, n0 = j * BT;
	const int k0 = blockIdx.y * per, k1 = min(L, k0 + per);
	const Tile<float> t = {a_re, a_im, a_re, a_im, weight, lda, lda, K, K, m0, n0, k1};
	Sums s;
	tile_product<true, WEIGHT, float, Off>(t, k0, st, s);
	double *re = part + (long) blockIdx.y * 2 * plane, *im = re + plane;
	each_element(s, m0, n0, [&](int row, int col, int, int, double x, double y) {
		if (row < K && col < K) {
			re[row * ldc + col] = x;
			im[row * ldc + col] = y;
		}
	});
}

// The shares added in order, and what lies below the diagonal filled in from above: C[j][i] = conj(C[i][j]).  A workgroup takes 32 x 32
// elements, turned over in LDS.  With one share `part` is C itself.
__global__ __launch_bounds__(JOIN_TPB) void gram_join_kernel(const double *part, int splits, double *c_re, double *c_im, long plane, long ldc, int K) {
	__shared__ double tile[2][32][33];
	const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
	if (c0 < r0) return;
	const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
	if (r0 + ty < K && c0 + tx < K) {
		const long at = (long) (r0 + ty) * ldc + c0 + tx;
		double re = part[at], im = part[at + plane];
#pragma unroll 8
		for (int s = 1; s < splits; ++s) {
			re += part[at + 2 * s * plane];
			im += part[at + (2 * s + 1) * plane];
		}
		if (r0 + ty == c0 + tx) im = 0.0;
		tile[0][ty][tx] = re;
		tile[1][ty][tx] = im;
		if (r0 + ty <= c0 + tx) {
			c_re[at] = re;
			c_im[at] = im;
		}
	}
	__syncthreads();
	if (c0 + ty < K && r0 + tx < K && c0 + ty > r0 + tx) {
		const long at = (long) (c0 + ty) * ldc + r0 + tx;
		c_re[at] = tile[0][tx][ty];
		c_im[at] = -tile[1][tx][ty];
	}
}

// C = conj(A) G for M rows of A: as an fp32 gradient with its conjugate, added or not, and (part != NULL) with Re sum_j C_ij A_ij over the
// block's columns to part[row][block column], in double from the sums themselves.
// The blocks of an XCD (consecutive numbers go to the XCDs in turn) are a contiguous strip, walked in groups of four block rows, column
// by column, so that what its L2 holds of A (2 MB for K = 1024) meets one block column of G after the other.
template <bool PART, class Off>
__global__ __launch_bounds__(TPB, 4) void times_gram_kernel(const float *a_re, const float *a_im, long lda, const double *g_re, const double *g_im, long ldg,
		int M, int K, const GramOut out) {
	__shared__ Stage st[2];
	const int tiles_m = (M + BT - 1) / BT, tiles_n = (K + BT - 1) / BT, total = gridDim.x;
	constexpr int XCDS = 8, GROUP = 4;
	const int xcd = blockIdx.x % XCDS, pid = xcd * (total / XCDS) + min(xcd, total % XCDS) + blockIdx.x / XCDS;
	const int group = pid / (GROUP * tiles_n), rows = min(GROUP, tiles_m - group * GROUP), in = pid - group * GROUP * tiles_n;
	const int m0 = (group * GROUP + in % rows) * BT, n0 = in / rows * BT;
	const Tile<double> t = {a_re, a_im, g_re, g_im, nullptr, lda, ldg, M, K, m0, n0, K};
	Sums s;
	tile_product<false, false, double, Off>(t, 0, st, s);
	double sum[2][4];
#pragma unroll
	for (int i = 0; i < 2; ++i)
#pragma unroll
		for (int e = 0; e < 4; ++e) sum[i][e] = 0.0;
	if (PART) {  // (what A has there, all of it requested before the first is used)
		float x_r[2][4], x_i[2][4];
		each_element(s, m0, n0, [&](int row, int col, int i, int e, double, double) {
			const long at = min(row, M - 1) * lda + min(col, K - 1);
			x_r[i][e] = a_re[at];
			x_i[i][e] = a_im[at];
		});
		each_element(s, m0, n0, [&](int, int col, int i, int e, double x, double y) {
			sum[i][e] = col < K ? x * (double) x_r[i][e] - y * (double) x_i[i][e] : 0.0;
		});
	}
	auto give = [&](float *p, long at, double v) { p[at] = out.accumulate ? (float) ((double) p[at] + v) : (float) v; };
	if (out.re)
		each_element(s, m0, n0, [&](int row, int col, int, int, double x, double y) {
			if (row >= M || col >= K) return;
			const long at = row * out.ld + col;
			give(out.re, at, x);
			give(out.im, at, y);
			if (out.sre) {
				give(out.sre, at, x);
				give(out.sim, at, -y);
			}
		});
	if (!PART) return;
	double(*met)[BT] = reinterpret_cast<double(*)[BT]>(&st[0]);  // [wave column][row]
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	__syncthreads();  // (the stages' last readers)
#pragma unroll
	for (int i = 0; i < 2; ++i)
#pragma unroll
		for (int e = 0; e < 4; ++e) {
			double v = sum[i][e];
			v += exchange<double, 0>(v);
			v += exchange<double, 1>(v);
			v += exchange<double, 2>(v);
			v += exchange<double, 3>(v);
			if ((lane & 15) == 0) met[wave & 3][32 * (wave >> 2) + 16 * i + 4 * e + (lane >> 4)] = v;
		}
	__syncthreads();
	const int row = m0 + (int) threadIdx.x;
	if (threadIdx.x < BT && row < M) out.part[(long) row * tiles_n + n0 / BT] = met[0][threadIdx.x] + met[1][threadIdx.x] + met[2][threadIdx.x] + met[3][threadIdx.x];
}

// leading dimensions below this keep the byte offsets inside a block (64 rows of floats, 16 of doubles) within 32 bits
constexpr long NEAR = 1L << 23;

// microseconds of one chunk of one block on a compute unit of its own: 48 matrix instructions of 64 cycles on each of the four pipes
double chunk_us() {
	const int khz = cnet::rt().prop.clockRate;
	return 48 * 64 / (khz > 0 ? khz * 1e-3 : 2.4e3);
}

// shares of the rows of A: as many as spread the blocks evenly over the compute units, as long as adding them up costs less
int gram_splits(int K, int L) {
	const double tiles = (K + BT - 1) / BT, blocks = tiles * (tiles + 1) / 2, cus = cnet::rt().prop.multiProcessorCount;
	const int chunks = (L + KC - 1) / KC;
	int best = 1;
	double least = 1e30;
	for (int s = 1; s <= 64 && (s == 1 || (chunks / s >= 4 && (double) s * K * K * 16 <= (double) (1 << 29))); ++s) {
		const int per = (chunks + s - 1) / s;
		if ((s - 1) * per >= chunks) continue;  // (the last share would be empty)
		const double us = std::ceil(blocks * s / cus) * per * chunk_us() + s * 8.0 * K * K * 2 / 3e6;
		if (us < least) least = us, best = s;
	}
	return best;
}

}  // namespace

namespace cnet {

double gram64_us(int K, int L) {
	const int s = gram_splits(K, L), chunks = (L + KC - 1) / KC;
	const double tiles = (K + BT - 1) / BT, cus = rt().prop.multiProcessorCount;
	return 11.0 + 1.24 * std::ceil(tiles * (tiles + 1) / 2 * s / cus) * ((chunks + s - 1) / s) * chunk_us() + (s + 1) * 8.0 * K * K / 3e6;
}

double times_gram_us(int M, int K) {
	const double blocks = (double) ((M + BT - 1) / BT) * ((K + BT - 1) / BT);
	return 9.0 + 1.24 * std::ceil(blocks / rt().prop.multiProcessorCount) * ((K + KC - 1) / KC) * chunk_us();
}

int gram64(int K, int L, const float *a_re, const float *a_im, long lda, const double *weight, const Gram64 &c) {
	const int splits = gram_splits(K, L), chunks = (L + KC - 1) / KC, per = (chunks + splits - 1) / splits * KC;
	const long tiles = (K + BT - 1) / BT, plane = (long) K * c.ld;
	if (tiles * (tiles + 1) / 2 > (1L << 30) || (K + 31) / 32 > 65535) return fail(CNET_ERR_UNSUPPORTED, "a Gram matrix of %d columns is too wide", K);
	double *part = c.re;
	if (splits > 1) {
		part = (double *) workspace((size_t) splits * 2 * plane * sizeof(double));
		if (!part) return rt().capturing ? CNET_ERR_UNSUPPORTED : CNET_ERR_OUT_OF_MEMORY;
	}
	const bool near = lda < NEAR;
	auto kern = weight ? (near ? gram_kernel<true, unsigned> : gram_kernel<true, size_t>) : (near ? gram_kernel<false, unsigned> : gram_kernel<false, size_t>);
	hipLaunchKernelGGL(kern, dim3((unsigned) (tiles * (tiles + 1) / 2), (unsigned) splits), dim3(TPB), 0, rt().stream, a_re, a_im, lda, weight, K, L, per,
			part, plane, c.ld);
	CNET_LAUNCH_CHECK();
	const unsigned turns = (unsigned) ((K + 31) / 32);
	hipLaunchKernelGGL(gram_join_kernel, dim3(turns, turns), dim3(JOIN_TPB), 0, rt().stream, part, splits, c.re, c.re + plane, plane, c.ld, K);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

int times_gram(int M, int K, const float *a_re, const float *a_im, long lda, const Gram64 &g, const GramOut &out) {
	const long blocks = (long) ((M + BT - 1) / BT) * ((K + BT - 1) / BT), plane = (long) K * g.ld;
	if (blocks > (1L << 30)) return fail(CNET_ERR_UNSUPPORTED, "a product of %d rows with a Gram matrix of %d columns is too large", M, K);
	const bool near = lda < NEAR && g.ld < NEAR;
	auto kern = out.part ? (near ? times_gram_kernel<true, unsigned> : times_gram_kernel<true, size_t>)
			: (near ? times_gram_kernel<false, unsigned> : times_gram_kernel<false, size_t>);
	hipLaunchKernelGGL(kern, dim3((unsigned) blocks), dim3(TPB), 0, rt().stream, a_re, a_im, lda, g.re, g.re + plane, g.ld, M, K, out);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

}  // namespace cnet
