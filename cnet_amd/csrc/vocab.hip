// What sits on the last block of a token model: the Linear to a large vocabulary with its CrossEntropy, whose logits are formed
// in pieces of the vocabulary and never kept, and the loss against a teacher's top entries.
//
// Both use the probabilities of CrossEntropy, p_k = |z_k|^2 / S with S = sum |z_k|^2 (impl/crossent.h:50-80 upstream), so that
//   dL/dz_k = conj(z_k) Q / S - q_k conj(z_k) / max(|z_k|^2, 1e-15)
// for targets q_k with the sum Q: one label (q = Q = 1), or the teacher's entries.
#include "common.hpp"
#include "rows.hpp"

#include <algorithm>
#include <cmath>

namespace cnet {
// cgemm.hip
int cgemm_pair(bool a_mcontig, bool b_ncontig, int nprob, int M, int N, int K, const float *const a_re[2], const float *const a_im[2], long lda,
		const float *const b_re[2], const float *const b_im[2], long ldb, const bool conj_b[2], float *const c_re[2], float *const c_im[2],
		long ldc, int accumulate, int tri, int mirror);
}  // namespace cnet

namespace {

using namespace cnet::rows;

constexpr int TPB = 256;
constexpr int WAVES = TPB / 64;
constexpr float LEAST = 1.0e-15f;  // of |z|^2 and of a probability whose logarithm is taken, as in CrossEntropy

// v, but at least LEAST; a NaN stays one, which fmax would drop
__device__ __forceinline__ float clamped(float v) { return v <= LEAST ? LEAST : v; }
__device__ __forceinline__ double clamped(double v) { return v <= (double) LEAST ? (double) LEAST : v; }

__device__ __forceinline__ void put(float *p, float v, int accumulate) { *p = accumulate ? *p + v : v; }

// ------------------------------------------------------------------------------------------------ distillation
struct DistillArgs {
	const float *z_re, *z_im;
	long ldz;
	const int *ids;
	const float *probs;
	int top;
	float *s, *loss;
	float *dz_re, *dz_im, *dzs_re, *dzs_im;
	long lddz;
	int rows, cols;
};

// One workgroup per row.  FWD: S and the loss; BWD: the gradient, with the S just formed or the one given.  The gradient is
// written for every column as if no entry named it, and the named ones are written again behind a barrier: the first entry of
// an index writes it, with the weights of all entries of that index.
template <bool FWD, bool BWD>
__global__ __launch_bounds__(TPB) void distill_kernel(const DistillArgs a) {
	__shared__ double lds_d[WAVES];
	__shared__ float lds_f[WAVES];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const long row = blockIdx.x;
	const float *zr = a.z_re + row * a.ldz, *zi = a.z_im + row * a.ldz;
	const int *ids = a.ids + row * a.top;
	const float *probs = a.probs + row * a.top;
	float S;
	if (FWD) {
		double sum = 0.0;
		for (int c = t; c < a.cols; c += TPB) sum = fma((double) zi[c], (double) zi[c], fma((double) zr[c], (double) zr[c], sum));
		sum = group_reduce<double, WAVES>(sum, SumD(), lds_d, 0, wave, lane);
		S = clamped((float) sum);
		float terms = 0.f;
		for (int j = t; j < a.top; j += TPB) {
			const int id = ids[j];
			const float q = probs[j];
			if (id < 0 || q == 0.f) continue;
			double p = (double) __builtin_nanf("");
			if (id < a.cols) p = clamped(((double) zr[id] * zr[id] + (double) zi[id] * zi[id]) / (double) S);
			terms += q * logf((float) (q / p));
		}
		terms = group_reduce<float, WAVES>(terms, SumF(), lds_f, 0, wave, lane);
		if (t == 0) {
			a.s[row] = S;
			a.loss[row] = terms;
		}
	} else {
		S = a.s[row];
	}
	if (!BWD) return;
	float total = 0.f;
	for (int j = t; j < a.top; j += TPB)
		if (ids[j] >= 0) total += probs[j];
	total = group_reduce<float, WAVES>(total, SumF(), lds_f, 0, wave, lane);
	const float share = total / S;
	float *or_ = a.dz_re + row * a.lddz, *oi = a.dz_im + row * a.lddz;
	float *sr = a.dzs_re ? a.dzs_re + row * a.lddz : nullptr, *si = a.dzs_re ? a.dzs_im + row * a.lddz : nullptr;
	auto store = [&](int c, float re, float im) {
		or_[c] = re;
		oi[c] = im;
		if (sr) {
			sr[c] = re;
			si[c] = -im;
		}
	};
	for (int c = t; c < a.cols; c += TPB) store(c, zr[c] * share, -(zi[c] * share));
	__syncthreads();
	for (int j = t; j < a.top; j += TPB) {
		const int id = ids[j];
		if (id < 0 || id >= a.cols) continue;
		float q = 0.f;
		bool first = true;
		for (int i = 0; i < a.top; ++i)
			if (ids[i] == id) {
				if (i < j) first = false;
				q += probs[i];
			}
		if (!first) continue;
		const double m = clamped((double) zr[id] * zr[id] + (double) zi[id] * zi[id]);
		const float k = (float) ((double) total / S - q / m);
		store(id, zr[id] * k, -(zi[id] * k));
	}
}

// ------------------------------------------------------------------------------------------------ vocabulary head
struct RowState {   // one entry per row of x, carried from piece to piece
	double *sum;    // sum |z|^2 so far
	float *best;    // largest |z|^2 so far, and its first index
	int *index;
	float *c_re, *c_im;  // conj(z_label) / m, the label's share of the gradient
};

// sum |z|^2 and the largest |z|^2 over the columns of one piece of the logits, added to what the earlier pieces left
__global__ __launch_bounds__(TPB) void head_piece_kernel(const float *__restrict__ zr, const float *__restrict__ zi, long ldz, int cols, int first_col,
		RowState st) {
	__shared__ double lds_d[WAVES];
	__shared__ ArgMax lds_a[WAVES];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const long row = blockIdx.x;
	zr += row * ldz;
	zi += row * ldz;
	double sum = 0.0;
	ArgMax best = {-1.0f, 0x7fffffff};
	for (int c = t; c < cols; c += TPB) {
		const float a = zr[c], b = zi[c];
		sum = fma((double) b, (double) b, fma((double) a, (double) a, sum));
		const float q = fmaf(a, a, b * b);
		if (q > best.v) best = ArgMax{q, first_col + c};
	}
	sum = group_reduce<double, WAVES>(sum, SumD(), lds_d, 0, wave, lane);
	best = group_reduce<ArgMax, WAVES>(best, ArgMaxOp(), lds_a, 0, wave, lane);
	if (t == 0) {
		if (first_col == 0) {
			st.sum[row] = sum;
			st.best[row] = best.v;
			st.index[row] = best.i;
		} else {
			st.sum[row] += sum;
			if (best.v > st.best[row]) {
				st.best[row] = best.v;
				st.index[row] = best.i;
			}
		}
	}
}

struct HeadArgs {
	const float *x_re, *x_im, *w_re, *w_im;
	long ldx, ldw;
	const int *labels;
	float *s, *loss;
	int *argmax;
	const float *y_re, *y_im;  // conj(z) w, not yet divided by S
	float *xs_re, *xs_im;      // x / S, for the weights' gradient
	long ldy;
	float *dx_re, *dx_im, *dxs_re, *dxs_im;
	long lddx;
	int accumulate_dx;
	int K, N;
};

// One workgroup per row: S, the label's logit (its products summed in double: the gradient goes with its inverse), loss, and the
// gradient at x: y / S minus the label's row of w times conj(z_label) / m.
template <bool BWD>
__global__ __launch_bounds__(TPB) void head_finish_kernel(const HeadArgs a, RowState st) {
	__shared__ double lds_d[WAVES];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const long row = blockIdx.x;
	const float S = clamped((float) st.sum[row]);
	int best = st.index[row];
	if (best < 0 || best >= a.N) best = 0;  // a row of NaN has no largest entry
	const int label = a.labels ? a.labels[row] : best;
	const bool known = label >= 0 && label < a.N;
	const float *xr = a.x_re + row * a.ldx, *xi = a.x_im + row * a.ldx;
	const float *wr = a.w_re + (known ? label : 0) * a.ldw, *wi = a.w_im + (known ? label : 0) * a.ldw;
	double re = 0.0, im = 0.0;
	if (known) {
		for (int c = t; c < a.K; c += TPB) {
			re += (double) xr[c] * wr[c] - (double) xi[c] * wi[c];
			im += (double) xr[c] * wi[c] + (double) xi[c] * wr[c];
		}
	}
	re = group_reduce<double, WAVES>(re, SumD(), lds_d, 0, wave, lane);
	im = group_reduce<double, WAVES>(im, SumD(), lds_d, 0, wave, lane);
	const double power = re * re + im * im, m = clamped(power);
	if (t == 0) {
		a.s[row] = S;
		if (a.loss) a.loss[row] = label < 0 ? 0.f : known ? -logf((float) clamped(power / (double) S)) : __builtin_nanf("");
		if (a.argmax) a.argmax[row] = best;
	}
	if (!BWD) return;
	const float inv = label < 0 ? 0.f : 1.0f / S;
	const float c_re = known ? (float) (re / m) : 0.f, c_im = known ? (float) (-im / m) : 0.f;
	if (t == 0) {
		st.c_re[row] = c_re;
		st.c_im[row] = c_im;
	}
	for (int c = t; c < a.K; c += TPB) {
		const long o = row * a.ldy + c, d = row * a.lddx + c;
		const float g_r = a.y_re[o] * inv - (c_re * wr[c] - c_im * wi[c]), g_i = a.y_im[o] * inv - (c_re * wi[c] + c_im * wr[c]);
		put(a.dx_re + d, g_r, a.accumulate_dx);
		put(a.dx_im + d, g_i, a.accumulate_dx);
		if (a.dxs_re) {
			put(a.dxs_re + d, g_r, a.accumulate_dx);
			put(a.dxs_im + d, -g_i, a.accumulate_dx);
		}
		a.xs_re[o] = xr[c] * inv;
		a.xs_im[o] = xi[c] * inv;
	}
}

struct ScatterArgs {
	const int *labels;
	const float *c_re, *c_im, *x_re, *x_im;
	long ldx;
	float *dw_re, *dw_im, *dws_re, *dws_im;
	long lddw;
	int B, K, N;
};

// dw[label[r]] -= c_r x_r for every row r, rows of the same label in order.  A workgroup owns SPAN rows of the vocabulary: it
// walks the labels in steps of TPB, and each of its threads owns columns.
constexpr int SPAN = 64;
__global__ __launch_bounds__(TPB) void head_scatter_kernel(const ScatterArgs a) {
	__shared__ int found[TPB], count[WAVES];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const int lo = blockIdx.x * SPAN, hi = min(a.N, lo + SPAN);
	for (int r0 = 0; r0 < a.B; r0 += TPB) {
		const int r = r0 + t;
		const int label = r < a.B ? a.labels[r] : -1;
		const bool mine = label >= lo && label < hi;
		const unsigned long long set = __ballot(mine);
		if (lane == 0) count[wave] = __popcll(set);
		__syncthreads();
		int at = __popcll(set & ((1ull << lane) - 1)), total = 0;
		for (int w = 0; w < WAVES; ++w) {
			if (w < wave) at += count[w];
			total += count[w];
		}
		if (mine) found[at] = r;
		__syncthreads();
		for (int k = 0; k < total; ++k) {
			const long row = found[k];
			const long dst = (long) a.labels[row] * a.lddw;
			const float c_re = a.c_re[row], c_im = a.c_im[row];
			for (int c = t; c < a.K; c += TPB) {
				const float x_r = a.x_re[row * a.ldx + c], x_i = a.x_im[row * a.ldx + c];
				const float d_r = c_re * x_r - c_im * x_i, d_i = c_re * x_i + c_im * x_r;
				a.dw_re[dst + c] -= d_r;
				a.dw_im[dst + c] -= d_i;
				if (a.dws_re) {
					a.dws_re[dst + c] -= d_r;
					a.dws_im[dst + c] += d_i;
				}
			}
		}
		__syncthreads();
	}
}

// the gradient of no rows at all
__global__ __launch_bounds__(TPB) void head_clear_kernel(float *p, long ld, int cols) {
	for (int c = threadIdx.x; c < cols; c += TPB) p[blockIdx.x * ld + c] = 0.f;
}

}  // namespace

using namespace cnet;

template <bool FWD, bool BWD>
static int distill(const DistillArgs &a) {
	hipLaunchKernelGGL((distill_kernel<FWD, BWD>), dim3((unsigned) a.rows), dim3(TPB), 0, rt().stream, a);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

// what the calls of the head keep between their launches, carved out of one buffer of the library
struct HeadBuffers {
	RowState st;
	float *piece, *y, *xs;  // planes re, im
	int piece_cols;         // columns of one piece, also its leading dimension
	long ldk;               // leading dimension of y and xs
};

// A piece of logits (two planes of B rows) is as wide as the memory-side cache holds: the pass over it, and the product that
// reads it, then find it there.
constexpr size_t PIECE_BYTES = (size_t) 192 << 20;

static int head_buffers(int B, int K, int N, bool bwd, HeadBuffers &b) {
	const long whole = ((long) N + 63) / 64 * 64;
	b.piece_cols = (int) std::min(whole, std::max(64L, (long) (PIECE_BYTES / (8 * (size_t) B)) / 64 * 64));
	b.ldk = ((long) K + 3) / 4 * 4;
	const size_t rows = ((size_t) B + 63) / 64 * 64;
	const size_t piece = 2 * (size_t) B * b.piece_cols, wide = bwd ? 2 * (size_t) B * b.ldk : 0;
	float *p = (float *) vocab_workspace((7 * rows + piece + 2 * wide) * sizeof(float));
	if (!p) return rt().capturing ? CNET_ERR_UNSUPPORTED : CNET_ERR_OUT_OF_MEMORY;
	b.st.sum = (double *) p;
	b.st.best = p + 2 * rows;
	b.st.index = (int *) (p + 3 * rows);
	b.st.c_re = p + 4 * rows;
	b.st.c_im = p + 5 * rows;
	b.piece = p + 7 * rows;
	b.y = b.piece + piece;
	b.xs = b.y + wide;
	return CNET_OK;
}

static int head(const HeadArgs &proto, int B, float *dw_re, float *dw_im, float *dws_re, float *dws_im, long lddw, int accumulate_dw, bool bwd) {
	HeadArgs a = proto;
	const int K = a.K, N = a.N;
	HeadBuffers b;
	int rc = head_buffers(B, K, N, bwd, b);
	if (rc) return rc;
	float *z_re = b.piece, *z_im = b.piece + (size_t) B * b.piece_cols;
	float *y_re = b.y, *y_im = b.y + (size_t) B * b.ldk;
	a.y_re = y_re;
	a.y_im = y_im;
	a.xs_re = b.xs;
	a.xs_im = b.xs + (size_t) B * b.ldk;
	a.ldy = b.ldk;
	const int np = b.piece_cols;
	auto logits = [&](int n0, int n) {
		return cnet_clinear_fwd(a.x_re, a.x_im, a.ldx, a.w_re + (size_t) n0 * a.ldw, a.w_im + (size_t) n0 * a.ldw, a.ldw, z_re, z_im, np, B, K, n, 0);
	};
	for (int n0 = 0; n0 < N; n0 += np) {
		const int n = std::min(np, N - n0);
		rc = logits(n0, n);
		if (rc) return rc;
		hipLaunchKernelGGL(head_piece_kernel, dim3((unsigned) B), dim3(TPB), 0, rt().stream, z_re, z_im, (long) np, n, n0, b.st);
		CNET_LAUNCH_CHECK();
		if (bwd) {  // y += conj(z) w: linear in z, so the division by S can wait until S is whole
			rc = cnet_cgemm_batched(0, 1, 1, 0, B, K, n, z_re, z_im, np, 0, a.w_re + (size_t) n0 * a.ldw, a.w_im + (size_t) n0 * a.ldw, a.ldw, 0, y_re,
					y_im, b.ldk, 0, 1, n0 > 0);
			if (rc) return rc;
		}
	}
	if (bwd) hipLaunchKernelGGL(head_finish_kernel<true>, dim3((unsigned) B), dim3(TPB), 0, rt().stream, a, b.st);
	else hipLaunchKernelGGL(head_finish_kernel<false>, dim3((unsigned) B), dim3(TPB), 0, rt().stream, a, b.st);
	CNET_LAUNCH_CHECK();
	if (!bwd) return CNET_OK;
	for (int n0 = 0; n0 < N; n0 += np) {
		const int n = std::min(np, N - n0);
		if (N > np) {
			rc = logits(n0, n);
			if (rc) return rc;
		}
		const size_t o = (size_t) n0 * lddw;
		if (dws_re) {  // dz* = z^T conj(x / S) is computed, dz written as its conjugate
			const float *ar[2] = {z_re, z_re}, *ai[2] = {z_im, z_im}, *br[2] = {a.xs_re, a.xs_re}, *bi[2] = {a.xs_im, a.xs_im};
			float *cr[2] = {dws_re + o, dw_re + o}, *ci[2] = {dws_im + o, dw_im + o};
			const bool cj[2] = {true, true};
			rc = cgemm_pair(true, true, 1, n, K, B, ar, ai, np, br, bi, b.ldk, cj, cr, ci, lddw, accumulate_dw, 0, 1);
		} else {
			rc = cnet_cgemm_batched(1, 1, 1, 0, n, K, B, z_re, z_im, np, 0, a.xs_re, a.xs_im, b.ldk, 0, dw_re + o, dw_im + o, lddw, 0, 1, accumulate_dw);
		}
		if (rc) return rc;
	}
	const ScatterArgs sc = {a.labels, b.st.c_re, b.st.c_im, a.x_re, a.x_im, a.ldx, dw_re, dw_im, dws_re, dws_im, lddw, B, K, N};
	hipLaunchKernelGGL(head_scatter_kernel, dim3((unsigned) ((N + SPAN - 1) / SPAN)), dim3(TPB), 0, rt().stream, sc);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

extern "C" {

int cnet_distill_fwd(const float *z_re, const float *z_im, int64_t ldz, const int32_t *ids, const float *probs, int top, float *s, float *loss,
		int rows, int cols) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 24) && cols > 0 && top > 0 && top <= CNET_DISTILL_MAX_TOP);
	if (!rows) return CNET_OK;
	CNET_CHECK_ARG(z_re && z_im && ids && probs && s && loss && ldz >= cols);
	return distill<true, false>(DistillArgs{z_re, z_im, (long) ldz, ids, probs, top, s, loss, nullptr, nullptr, nullptr, nullptr, 0, rows, cols});
}

int cnet_distill_bwd_sym(const float *z_re, const float *z_im, int64_t ldz, const float *s, const int32_t *ids, const float *probs, int top,
		float *dz_dz_re, float *dz_dz_im, float *dz_dzs_re, float *dz_dzs_im, int64_t lddz, int rows, int cols) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 24) && cols > 0 && top > 0 && top <= CNET_DISTILL_MAX_TOP);
	if (!rows) return CNET_OK;
	CNET_CHECK_ARG(z_re && z_im && ids && probs && s && ldz >= cols);
	CNET_CHECK_ARG(dz_dz_re && dz_dz_im && ((dz_dzs_re == nullptr) == (dz_dzs_im == nullptr)) && lddz >= cols);
	return distill<false, true>(DistillArgs{z_re, z_im, (long) ldz, ids, probs, top, const_cast<float *>(s), nullptr, dz_dz_re, dz_dz_im, dz_dzs_re,
			dz_dzs_im, (long) lddz, rows, cols});
}

int cnet_distill_fwd_bwd_sym(const float *z_re, const float *z_im, int64_t ldz, const int32_t *ids, const float *probs, int top, float *s, float *loss,
		float *dz_dz_re, float *dz_dz_im, float *dz_dzs_re, float *dz_dzs_im, int64_t lddz, int rows, int cols) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 24) && cols > 0 && top > 0 && top <= CNET_DISTILL_MAX_TOP);
	if (!rows) return CNET_OK;
	CNET_CHECK_ARG(z_re && z_im && ids && probs && s && loss && ldz >= cols);
	CNET_CHECK_ARG(dz_dz_re && dz_dz_im && ((dz_dzs_re == nullptr) == (dz_dzs_im == nullptr)) && lddz >= cols);
	return distill<true, true>(DistillArgs{z_re, z_im, (long) ldz, ids, probs, top, s, loss, dz_dz_re, dz_dz_im, dz_dzs_re, dz_dzs_im, (long) lddz, rows,
			cols});
}

int cnet_vocab_head_fwd(const float *x_re, const float *x_im, int64_t ldx, const float *w_re, const float *w_im, int64_t ldw, const int32_t *labels,
		float *s, float *loss, int32_t *argmax, int B, int K, int N) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(B >= 0 && B < (1 << 24) && K > 0 && N > 0 && N <= (1 << 30));
	if (!B) return CNET_OK;
	CNET_CHECK_ARG(x_re && x_im && w_re && w_im && s && (loss || argmax));
	CNET_CHECK_ARG(ldx >= K && ldw >= K);
	HeadArgs a = {};
	a.x_re = x_re;
	a.x_im = x_im;
	a.w_re = w_re;
	a.w_im = w_im;
	a.ldx = ldx;
	a.ldw = ldw;
	a.labels = labels;
	a.s = s;
	a.loss = loss;
	a.argmax = argmax;
	a.K = K;
	a.N = N;
	return head(a, B, nullptr, nullptr, nullptr, nullptr, 0, 0, false);
}

int cnet_vocab_head_fwd_bwd_sym(const float *x_re, const float *x_im, int64_t ldx, const float *w_re, const float *w_im, int64_t ldw,
		const int32_t *labels, float *s, float *loss, int32_t *argmax, float *dx_dz_re, float *dx_dz_im, float *dx_dzs_re, float *dx_dzs_im,
		int64_t lddx, int accumulate_dx, float *dw_dz_re, float *dw_dz_im, float *dw_dzs_re, float *dw_dzs_im, int64_t lddw, int accumulate_dw, int B,
		int K, int N) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(B >= 0 && B < (1 << 24) && K > 0 && N > 0 && N <= (1 << 30));
	CNET_CHECK_ARG(dw_dz_re && dw_dz_im && ((dw_dzs_re == nullptr) == (dw_dzs_im == nullptr)) && lddw >= K);
	if (!B) {
		if (accumulate_dw) return CNET_OK;
		for (float *p : {dw_dz_re, dw_dz_im, dw_dzs_re, dw_dzs_im})
			if (p) hipLaunchKernelGGL(head_clear_kernel, dim3((unsigned) N), dim3(TPB), 0, rt().stream, p, (long) lddw, K);
		CNET_LAUNCH_CHECK();
		return CNET_OK;
	}
	CNET_CHECK_ARG(x_re && x_im && w_re && w_im && labels && s && loss);
	CNET_CHECK_ARG(ldx >= K && ldw >= K);
	CNET_CHECK_ARG(dx_dz_re && dx_dz_im && ((dx_dzs_re == nullptr) == (dx_dzs_im == nullptr)) && lddx >= K);
	HeadArgs a = {};
	a.x_re = x_re;
	a.x_im = x_im;
	a.w_re = w_re;
	a.w_im = w_im;
	a.ldx = ldx;
	a.ldw = ldw;
	a.labels = labels;
	a.s = s;
	a.loss = loss;
	a.argmax = argmax;
	a.dx_re = dx_dz_re;
	a.dx_im = dx_dz_im;
	a.dxs_re = dx_dzs_re;
	a.dxs_im = dx_dzs_im;
	a.lddx = lddx;
	a.accumulate_dx = accumulate_dx;
	a.K = K;
	a.N = N;
	return head(a, B, dw_dz_re, dw_dz_im, dw_dzs_re, dw_dzs_im, lddw, accumulate_dw, true);
}

}  // extern "C"
