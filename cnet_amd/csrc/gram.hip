// Products in double for the vocabulary head's way through Gram matrices (vocab.hip): C = A^H diag(weight) A, and C = conj(A) G with
// such a G.  The operands A are fp32 planes, G and all sums are double.
//
// Why double: what the head takes from a Gram matrix (a row's sum |z|^2, the gradients) is small where the rows of A lie in
// directions that the other operand hardly has, while the terms it is summed from are not.  Products of two fp32 numbers are exact
// in double, and 29 bits to spare cover every such difference that the logits themselves would still show (whose fp32 sums lose
// all digits long before).
//
// One workgroup of four wavefronts forms 64 x 64 of C, each 32 x 32 of it with v_mfma_f64_16x16x4_f64, K in chunks of 16 through two
// buffers of LDS; the next chunk is on its way in registers while the present one is multiplied.  Three real products per complex one
// (with a' = conj(a): Re = ar br - ai' bi, Im = (ar + ai')(br + bi) - ar br - ai' bi; the differences cost a few of the bits to spare).
// Bound by the matrix pipe (64 cycles an instruction, 128 flop a cycle and compute unit, half of what fp32 has).  With 64 cycles an instruction
// everything else has time: 21 bytes of LDS a cycle and compute unit, accesses of 4 and 8 bytes whatever the operands' alignment.
#include "common.hpp"
#include "rows.hpp"

#include <algorithm>
#include <cmath>

#include "gram.hpp"

namespace {

using namespace cnet::rows;
using cnet::Gram64;
using cnet::GramOut;

constexpr int TPB = 256;
constexpr int BT = cnet::GRAM_TILE, KC = cnet::GRAM_CHUNK;
// (66: with a row-major operand 16 lanes write 16 different k of one row, 132 words apart: all 64 banks; the reads go two ways)
constexpr int LD = BT + 2;

typedef double double4_t __attribute__((ext_vector_type(4)));

struct Stage {
	double v[2][2][KC][LD];  // [A, B][re, im][k][row of A / column of B]
};

// rows m0 .. of the block's part of A (or columns, KMAJOR), columns n0 .. of B, and the range of k
template <bool KMAJOR, class TB>
struct Tile {
	const float *a_re, *a_im;
	const TB *b_re, *b_im;
	const double *weight;  // KMAJOR: of the rows of A and B, or NULL
	long lda, ldb;
	int M, N, m0, n0, k_end;
};

struct Sums {
	double4_t p1[2][2], p2[2][2], p3[2][2];  // ar br, ai' bi, (ar + ai')(br + bi)
};

// K from k0 to t.k_end (k0 a multiple of KC).  What lies behind k_end is zero in both operands; rows and columns beyond M and N repeat
// the last ones, and nobody stores what comes of them.
template <bool KMAJOR, class TB>
__device__ __forceinline__ void tile_product(const Tile<KMAJOR, TB> &t, int k0, Stage (&st)[2], Sums &s) {
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1, r = lane & 15, q = lane >> 4;
#pragma unroll
	for (int i = 0; i < 2; ++i)
#pragma unroll
		for (int j = 0; j < 2; ++j) s.p1[i][j] = s.p2[i][j] = s.p3[i][j] = double4_t{0.0, 0.0, 0.0, 0.0};
	// element i of a thread: k-major operands: column tid % 64, k = tid / 64 + 4 i; row-major: k = tid % 16, row tid / 16 + 16 i
	const int col_b = min(t.n0 + tid % BT, t.N - 1);
	long a_at[4];
	if (KMAJOR) {
		a_at[0] = min(t.m0 + tid % BT, t.M - 1);
	} else {
#pragma unroll
		for (int i = 0; i < 4; ++i) a_at[i] = (long) min(t.m0 + tid / KC + 16 * i, t.M - 1) * t.lda;
	}
	float a_r[4], a_i[4];
	TB b_r[4], b_i[4];
	double g[4];
	auto fetch = [&](int k) {
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const int kb = min(k + tid / BT + 4 * i, t.k_end - 1), ka = KMAJOR ? kb : min(k + tid % KC, t.k_end - 1);
			const long a = KMAJOR ? (long) ka * t.lda + a_at[0] : a_at[i] + ka, b = (long) kb * t.ldb + col_b;
			a_r[i] = t.a_re[a];
			a_i[i] = t.a_im[a];
			b_r[i] = t.b_re[b];
			b_i[i] = t.b_im[b];
			g[i] = KMAJOR && t.weight ? t.weight[kb] : 1.0;
		}
	};
	auto put_stage = [&](Stage &to, int k) {
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const int kb = tid / BT + 4 * i, ka = KMAJOR ? kb : tid % KC, m = KMAJOR ? tid % BT : tid / KC + 16 * i;
			// (a row of weight 0 is left out whatever it holds)
			const bool in_b = k + kb < t.k_end && g[i] != 0.0, in_a = KMAJOR ? in_b : k + ka < t.k_end;
			const double x = (double) a_r[i], y = -(double) a_i[i];
			to.v[0][0][ka][m] = in_a ? (KMAJOR ? x * g[i] : x) : 0.0;
			to.v[0][1][ka][m] = in_a ? (KMAJOR ? y * g[i] : y) : 0.0;
			to.v[1][0][kb][tid % BT] = in_b ? (double) b_r[i] : 0.0;
			to.v[1][1][kb][tid % BT] = in_b ? (double) b_i[i] : 0.0;
		}
	};
	fetch(k0);
	int at = 0;
	for (int k = k0; k < t.k_end; k += KC, at ^= 1) {
		put_stage(st[at], k);  // (last read two chunks ago, before the barrier of the chunk between)
		__syncthreads();
		if (k + KC < t.k_end) fetch(k + KC);
		__builtin_amdgcn_sched_barrier(0);  // (the loads go out before the products, not after them)
#pragma unroll
		for (int step = 0; step < KC / 4; ++step) {
			double ar[2], ai[2], as[2], br[2], bi[2], bs[2];
#pragma unroll
			for (int i = 0; i < 2; ++i) {
				ar[i] = st[at].v[0][0][4 * step + q][32 * wm + 16 * i + r];
				ai[i] = st[at].v[0][1][4 * step + q][32 * wm + 16 * i + r];
				br[i] = st[at].v[1][0][4 * step + q][32 * wn + 16 * i + r];
				bi[i] = st[at].v[1][1][4 * step + q][32 * wn + 16 * i + r];
				as[i] = ar[i] + ai[i];
				bs[i] = br[i] + bi[i];
			}
#pragma unroll
			for (int i = 0; i < 2; ++i)
#pragma unroll
				for (int j = 0; j < 2; ++j) {
					s.p1[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(ar[i], br[j], s.p1[i][j], 0, 0, 0);
					s.p2[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(ai[i], bi[j], s.p2[i][j], 0, 0, 0);
					s.p3[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(as[i], bs[j], s.p3[i][j], 0, 0, 0);
				}
		}
	}
}

// calls f(row, column, i, j, e, re, im) for a lane's 16 elements of the block: element e of tile (i, j) is row 4 e + lane / 16, column lane % 16
template <class F>
__device__ __forceinline__ void each_element(const Sums &s, int m0, int n0, F f) {
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
	for (int i = 0; i < 2; ++i)
#pragma unroll
		for (int e = 0; e < 4; ++e)
#pragma unroll
			for (int j = 0; j < 2; ++j) {
				const double re = s.p1[i][j][e] - s.p2[i][j][e], im = s.p3[i][j][e] - s.p1[i][j][e] - s.p2[i][j][e];
				f(m0 + 32 * (wave >> 1) + 16 * i + 4 * e + (lane >> 4), n0 + 32 * (wave & 1) + 16 * j + (lane & 15), i, e, re, im);
			}
}

// C = A^H diag(weight) A [K][K] over the rows [split * per, ..) of A, blocks on and above the diagonal: blockIdx.x counts them column by
// column, blockIdx.y the shares of the rows, each with planes of its own in `part`.
__global__ __launch_bounds__(TPB, 2) void gram_kernel(const float *a_re, const float *a_im, long lda, const double *weight, int K, int L, int per,
		double *__restrict__ part, long plane, long ldc) {
	__shared__ Stage st[2];
	const int pid = blockIdx.x;
	int j = (int) ((sqrtf(8.0f * (float) pid + 1.0f) - 1.0f) * 0.5f);  // block column j starts at number j (j + 1) / 2
	while (j * (j + 1) / 2 > pid) --j;
	while ((j + 1) * (j + 2) / 2 <= pid) ++j;
	const int m0 = (pid - j * (j + 1) / 2) * BT, n0 = j * BT;
	const int k0 = blockIdx.y * per, k1 = min(L, k0 + per);
	const Tile<true, float> t = {a_re, a_im, a_re, a_im, weight, lda, lda, K, K, m0, n0, k1};
	Sums s;
	tile_product(t, k0, st, s);
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
__global__ __launch_bounds__(TPB) void gram_join_kernel(const double *part, int splits, double *c_re, double *c_im, long plane, long ldc, int K) {
	__shared__ double tile[2][32][33];
	const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
	if (c0 < r0) return;
	const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
	for (int k = ty; k < 32; k += 8)
		if (r0 + k < K && c0 + tx < K) {
			const long at = (long) (r0 + k) * ldc + c0 + tx;
			double re = part[at], im = part[at + plane];
#pragma unroll 4
			for (int s = 1; s < splits; ++s) {
				re += part[at + 2 * s * plane];
				im += part[at + (2 * s + 1) * plane];
			}
			if (r0 + k == c0 + tx) im = 0.0;
			tile[0][k][tx] = re;
			tile[1][k][tx] = im;
			if (r0 + k <= c0 + tx) {
				c_re[at] = re;
				c_im[at] = im;
			}
		}
	__syncthreads();
	for (int k = ty; k < 32; k += 8)
		if (c0 + k < K && r0 + tx < K && c0 + k > r0 + tx) {
			c_re[(long) (c0 + k) * ldc + r0 + tx] = tile[0][tx][k];
			c_im[(long) (c0 + k) * ldc + r0 + tx] = -tile[1][tx][k];
		}
}

// C = conj(A) G for M rows of A: as an fp32 gradient with its conjugate, added or not, and (part != NULL) with Re sum_j C_ij A_ij over the
// block's columns to part[row][block column], in double from the sums themselves.
// The blocks of an XCD (consecutive numbers go to the XCDs in turn) are a contiguous strip, walked in groups of four block rows, column
// by column, so that what its L2 holds of A (2 MB for K = 1024) meets one block column of G after the other.
template <bool PART>
__global__ __launch_bounds__(TPB, 2) void times_gram_kernel(const float *a_re, const float *a_im, long lda, const double *g_re, const double *g_im, long ldg,
		int M, int K, const GramOut out) {
	__shared__ Stage st[2];
	const int tiles_m = (M + BT - 1) / BT, tiles_n = (K + BT - 1) / BT, total = gridDim.x;
	constexpr int XCDS = 8, GROUP = 4;
	const int xcd = blockIdx.x % XCDS, pid = xcd * (total / XCDS) + min(xcd, total % XCDS) + blockIdx.x / XCDS;
	const int group = pid / (GROUP * tiles_n), rows = min(GROUP, tiles_m - group * GROUP), in = pid - group * GROUP * tiles_n;
	const int m0 = (group * GROUP + in % rows) * BT, n0 = in / rows * BT;
	const Tile<false, double> t = {a_re, a_im, g_re, g_im, nullptr, lda, ldg, M, K, m0, n0, K};
	Sums s;
	tile_product(t, 0, st, s);
	double sum[2][4];
#pragma unroll
	for (int i = 0; i < 2; ++i)
#pragma unroll
		for (int e = 0; e < 4; ++e) sum[i][e] = 0.0;
	auto give = [&](float *p, long at, double v) { p[at] = out.accumulate ? (float) ((double) p[at] + v) : (float) v; };
	each_element(s, m0, n0, [&](int row, int col, int i, int e, double x, double y) {
		if (row >= M || col >= K) return;
		if (PART) sum[i][e] += x * (double) a_re[row * lda + col] - y * (double) a_im[row * lda + col];
		if (!out.re) return;
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
			if ((lane & 15) == 0) met[wave & 1][32 * (wave >> 1) + 16 * i + 4 * e + (lane >> 4)] = v;
		}
	__syncthreads();
	const int row = m0 + (int) threadIdx.x;
	if (threadIdx.x < BT && row < M) out.part[(long) row * tiles_n + n0 / BT] = met[0][threadIdx.x] + met[1][threadIdx.x];
}

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
	return 8.0 + 1.1 * std::ceil(tiles * (tiles + 1) / 2 * s / cus) * ((chunks + s - 1) / s) * chunk_us() + (s + 1) * 16.0 * K * K / 3e6;
}

double times_gram_us(int M, int K) {
	const double blocks = (double) ((M + BT - 1) / BT) * ((K + BT - 1) / BT);
	return 4.0 + 1.1 * std::ceil(blocks / rt().prop.multiProcessorCount) * ((K + KC - 1) / KC) * chunk_us();
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
	hipLaunchKernelGGL(gram_kernel, dim3((unsigned) (tiles * (tiles + 1) / 2), (unsigned) splits), dim3(TPB), 0, rt().stream, a_re, a_im, lda, weight, K, L,
			per, part, plane, c.ld);
	CNET_LAUNCH_CHECK();
	const unsigned turns = (unsigned) ((K + 31) / 32);
	hipLaunchKernelGGL(gram_join_kernel, dim3(turns, turns), dim3(TPB), 0, rt().stream, part, splits, c.re, c.re + plane, plane, c.ld, K);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

int times_gram(int M, int K, const float *a_re, const float *a_im, long lda, const Gram64 &g, const GramOut &out) {
	const long blocks = (long) ((M + BT - 1) / BT) * ((K + BT - 1) / BT), plane = (long) K * g.ld;
	if (blocks > (1L << 30)) return fail(CNET_ERR_UNSUPPORTED, "a product of %d rows with a Gram matrix of %d columns is too large", M, K);
	if (out.part)
		hipLaunchKernelGGL(times_gram_kernel<true>, dim3((unsigned) blocks), dim3(TPB), 0, rt().stream, a_re, a_im, lda, g.re, g.re + plane, g.ld, M, K, out);
	else
		hipLaunchKernelGGL(times_gram_kernel<false>, dim3((unsigned) blocks), dim3(TPB), 0, rt().stream, a_re, a_im, lda, g.re, g.re + plane, g.ld, M, K, out);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

}  // namespace cnet
