// What sits on the last block of a token model: the Linear to a large vocabulary with its CrossEntropy, whose logits are formed
// in pieces of the vocabulary and never kept, and the loss against a teacher's top entries.
//
// Both use the probabilities of CrossEntropy, p_k = |z_k|^2 / S with S = sum |z_k|^2 (impl/crossent.h:50-80 upstream), so that
//   dL/dz_k = conj(z_k) Q / S - q_k conj(z_k) / max(|z_k|^2, 1e-15)
// for targets q_k with the sum Q: one label (q = Q = 1), or the teacher's entries.
#include "common.hpp"
#include "gram.hpp"
#include "rows.hpp"

#include <algorithm>
#include <cmath>

namespace cnet {
// cgemm.hip
int cgemm_pair(bool a_mcontig, bool b_ncontig, int nprob, int M, int N, int K, const float *const a_re[2], const float *const a_im[2], long lda,
		const float *const b_re[2], const float *const b_im[2], long ldb, const bool conj_b[2], float *const c_re[2], float *const c_im[2],
		long ldc, int accumulate, int tri, int mirror);
int clinear_bwd_sym(bool one_launch, const float *g_dz_re, const float *g_dz_im, int64_t ldg, const float *x_re, const float *x_im, int64_t ldx,
		const float *w_re, const float *w_im, int64_t ldw, float *dx_dz_re, float *dx_dz_im, float *dx_dzs_re, float *dx_dzs_im, int64_t lddx,
		int accumulate_dx, float *dw_dz_re, float *dw_dz_im, float *dw_dzs_re, float *dw_dzs_im, int64_t lddw, int accumulate_dw, int B, int K, int N);
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

template <int V>
__device__ __forceinline__ void load_v(float *v, const float *p) {
	if (V == 4) {
		const float4 t = *reinterpret_cast<const float4 *>(p);
		v[0] = t.x;
		v[1 % V] = t.y;
		v[2 % V] = t.z;
		v[3 % V] = t.w;
	} else {
		v[0] = p[0];
	}
}
template <int V>
__device__ __forceinline__ void store_v(float *p, const float *v) {
	if (V == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1 % V], v[2 % V], v[3 % V]);
	else p[0] = v[0];
}

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

// A row's entries in LDS, each array filled up to a multiple of four: index, weight, and the row's values there
struct Entries {
	int *id;
	float *q, *re, *im;
	int count;  // with the filling
};
__host__ __device__ __forceinline__ int entry_slots(int top) { return (top + 3) / 4 * 4; }
__device__ __forceinline__ Entries entries_at(float *lds, int top) {
	const int n = entry_slots(top);
	return Entries{(int *) lds, lds + n, lds + 2 * n, lds + 3 * n, n};
}

// T threads fetch the entries of their row
template <int T>
__device__ __forceinline__ void fetch_entries(const DistillArgs &a, const Entries &e, long row, int t) {
	for (int j = t; j < e.count; j += T) {
		const int id = j < a.top ? a.ids[row * a.top + j] : -1;
		const bool there = id >= 0 && id < a.cols;
		const float q = id < 0 ? 0.f : a.probs[row * a.top + j];
		e.id[j] = id;
		e.q[j] = q;
		e.re[j] = there ? a.z_re[row * a.ldz + id] : 0.f;
		e.im[j] = there ? a.z_im[row * a.ldz + id] : 0.f;
	}
}

// the sum of the weights, formed by every wavefront for itself
__device__ __forceinline__ float total_weight(const Entries &e, int lane) {
	float total = 0.f;
	for (int j = lane; j < e.count; j += 64) total += e.q[j];
	return wave_reduce(total, SumF());
}

// one thread's part of the loss
template <int T>
__device__ __forceinline__ float loss_terms(const DistillArgs &a, const Entries &e, float S, int t) {
	float terms = 0.f;
	for (int j = t; j < a.top; j += T) {
		const float q = e.q[j];
		if (q == 0.f) continue;
		double p = (double) __builtin_nanf("");
		if (e.id[j] < a.cols) p = clamped(((double) e.re[j] * e.re[j] + (double) e.im[j] * e.im[j]) / (double) S);
		terms += q * logf((float) (q / p));
	}
	return terms;
}

__device__ __forceinline__ void distill_store(const DistillArgs &a, long row, int c, float re, float im) {
	const long o = row * a.lddz + c;
	a.dz_re[o] = re;
	a.dz_im[o] = im;
	if (a.dzs_re) {
		a.dzs_re[o] = re;
		a.dzs_im[o] = -im;
	}
}

// The gradient at the entries' own columns among [c0, c1), over what the pass over the whole row has left there: the first entry
// of an index writes it, with the weights of all entries of that index.
template <int T>
__device__ __forceinline__ void entry_gradients(const DistillArgs &a, const Entries &e, long row, float S, float total, int t, int c0, int c1) {
	for (int j = t; j < a.top; j += T) {
		const int id = e.id[j];
		if (id < c0 || id >= c1) continue;
		float q = 0.f;
		int first = j;
#pragma unroll 4
		for (int i = 0; i < e.count; i += 4) {
			const int4 n = *reinterpret_cast<const int4 *>(e.id + i);
			const float4 p = *reinterpret_cast<const float4 *>(e.q + i);
			q += n.x == id ? p.x : 0.f;
			q += n.y == id ? p.y : 0.f;
			q += n.z == id ? p.z : 0.f;
			q += n.w == id ? p.w : 0.f;
			const int at = n.x == id ? i : n.y == id ? i + 1 : n.z == id ? i + 2 : n.w == id ? i + 3 : j;
			first = min(first, at);
		}
		if (first != j) continue;
		const double m = clamped((double) e.re[j] * e.re[j] + (double) e.im[j] * e.im[j]);
		const float k = (float) ((double) total / S - q / m);
		distill_store(a, row, id, e.re[j] * k, -(e.im[j] * k));
	}
}

// The row in registers: T threads hold V x NIT columns each, so z is read once and the gradient written once, 16 bytes per element
// each way (24 with dz*), which is what bounds it: 8192 x 32768 takes 802 us among other work, 5.4 TB/s (a copy of 1 GiB: 5.1).  The entries and their
// values are fetched while the row is on its way.  T = 64: four rows to a workgroup (96 x 512: 4.9 us, a launch).
// LONG: the columns that the registers do not hold are read once more for the gradient (4096 x 50257, 36 of 100 columns: 786 us).
template <int T, int NIT, int V, bool LONG>
__global__ __launch_bounds__(T < TPB ? TPB : T) void distill_kernel(const DistillArgs a, const int policy) {
	constexpr int G = T / 64, ROWS = T < TPB ? TPB / T : 1;
	extern __shared__ __align__(16) float lds[];
	__shared__ double lds_d[ROWS * G];
	__shared__ float lds_f[ROWS * G];
	const int slot = threadIdx.x / T, t = threadIdx.x % T, lane = threadIdx.x & 63, wave = t >> 6;
	const bool live = (long) blockIdx.x * ROWS + slot < a.rows;
	const long row = live ? (long) blockIdx.x * ROWS + slot : a.rows - 1;
	const Entries e = entries_at(lds + slot * 4 * entry_slots(a.top), a.top);
	const float *zr = a.z_re + row * a.ldz, *zi = a.z_im + row * a.ldz;
	float re[NIT][V], im[NIT][V];
#pragma unroll
	for (int k = 0; k < NIT; ++k) {
		// (no branch around the loads: a column of the row is read in any case and the result chosen afterwards)
		const int c = (k * T + t) * V, at = min(c, a.cols - V);
		const bool in = c < a.cols;
		if (V == 4) {
			const float4 x = ld4(zr + at, policy), y = ld4(zi + at, policy);
			re[k][0] = in ? x.x : 0.f, re[k][1 % V] = in ? x.y : 0.f, re[k][2 % V] = in ? x.z : 0.f, re[k][3 % V] = in ? x.w : 0.f;
			im[k][0] = in ? y.x : 0.f, im[k][1 % V] = in ? y.y : 0.f, im[k][2 % V] = in ? y.z : 0.f, im[k][3 % V] = in ? y.w : 0.f;
		} else {
			const float x = zr[at], y = zi[at];
			re[k][0] = in ? x : 0.f;
			im[k][0] = in ? y : 0.f;
		}
	}
	fetch_entries<T>(a, e, row, t);
	float S;
	if (a.loss) {
		double sum = 0.0;
#pragma unroll
		for (int k = 0; k < NIT; ++k)
#pragma unroll
			for (int q = 0; q < V; ++q) sum = fma((double) im[k][q], (double) im[k][q], fma((double) re[k][q], (double) re[k][q], sum));
		if (LONG) {
#pragma unroll 2
			for (int c = (NIT * T + t) * V; c < a.cols; c += T * V) {
				float u[V], v[V];
				load_v<V>(u, zr + c);
				load_v<V>(v, zi + c);
#pragma unroll
				for (int q = 0; q < V; ++q) sum = fma((double) v[q], (double) v[q], fma((double) u[q], (double) u[q], sum));
			}
		}
		S = clamped((float) group_reduce<double, G>(sum, SumD(), lds_d, slot, wave, lane));
	} else {
		S = a.s[row];
	}
	if (G == 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the entries are this wavefront's own
	else if (!a.loss) __syncthreads();                                   // (the exchange of the sum has had its barriers)
	const float total = total_weight(e, lane);
	const bool none = total == 0.f;  // nothing to learn from (a row of padding): gradient 0 whatever the row holds, NaN and infinities too
	const float share = none ? 0.f : total / S;
	if (none) {
#pragma unroll
		for (int k = 0; k < NIT; ++k)
#pragma unroll
			for (int q = 0; q < V; ++q) re[k][q] = im[k][q] = 0.f;
	}
	// the gradient first, the loss while it is on its way to memory
	if (live && a.dz_re) {
#pragma unroll
		for (int k = 0; k < NIT; ++k) {
			const int c = (k * T + t) * V;
			if (c >= a.cols) continue;
			if (V == 4) {
				const long o = row * a.lddz + c;
				const float4 u = make_float4(re[k][0] * share, re[k][1 % V] * share, re[k][2 % V] * share, re[k][3 % V] * share);
				const float4 v = make_float4(im[k][0] * share, im[k][1 % V] * share, im[k][2 % V] * share, im[k][3 % V] * share);
				const float4 n = make_float4(-v.x, -v.y, -v.z, -v.w);
				st4(a.dz_re + o, u, policy);
				st4(a.dz_im + o, n, policy);
				if (a.dzs_re) {
					st4(a.dzs_re + o, u, policy);
					st4(a.dzs_im + o, v, policy);
				}
			} else {
				distill_store(a, row, c, re[k][0] * share, -(im[k][0] * share));
			}
		}
		if (LONG) {
#pragma unroll 2
			for (int c = (NIT * T + t) * V; c < a.cols; c += T * V) {
				const long o = row * a.lddz + c;
				float u[V], v[V], n[V];
				load_v<V>(u, zr + c);
				load_v<V>(v, zi + c);
#pragma unroll
				for (int q = 0; q < V; ++q) {
					u[q] = none ? 0.f : u[q] * share;
					v[q] = none ? 0.f : v[q] * share;
					n[q] = -v[q];
				}
				store_v<V>(a.dz_re + o, u);
				store_v<V>(a.dz_im + o, n);
				if (a.dzs_re) {
					store_v<V>(a.dzs_re + o, u);
					store_v<V>(a.dzs_im + o, v);
				}
			}
		}
	}
	if (a.loss) {
		const float loss = group_reduce<float, G>(loss_terms<T>(a, e, S, t), SumF(), lds_f, slot, wave, lane);
		if (t == 0 && live) {
			a.s[row] = S;
			a.loss[row] = loss;
		}
	}
	if (!a.dz_re) return;
	if (G == 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
	else __syncthreads();
	if (live && !none) entry_gradients<T>(a, e, row, S, total, t, 0, a.cols);
}

// Few long rows: a row is dealt out to workgroups of SLAB columns each, in two launches (its sum, in parts; its gradient).  Bound by
// the two launches: 3 x 100003 takes 8.5 us (116 with one workgroup per row).
constexpr int SLAB_COLS = 8;           // of one thread
constexpr int SLAB = TPB * SLAB_COLS;
__global__ __launch_bounds__(TPB) void distill_slab_sum_kernel(const DistillArgs a, double *__restrict__ part) {
	__shared__ double lds_d[WAVES];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const long row = blockIdx.y;
	const int c0 = blockIdx.x * SLAB;
	const float *zr = a.z_re + row * a.ldz, *zi = a.z_im + row * a.ldz;
	float re[SLAB_COLS], im[SLAB_COLS];
#pragma unroll
	for (int k = 0; k < SLAB_COLS; ++k) {
		const int at = min(c0 + k * TPB + t, a.cols - 1);
		re[k] = zr[at];
		im[k] = zi[at];
	}
	double sum = 0.0;
#pragma unroll
	for (int k = 0; k < SLAB_COLS; ++k)
		if (c0 + k * TPB + t < a.cols) sum = fma((double) im[k], (double) im[k], fma((double) re[k], (double) re[k], sum));
	sum = group_reduce<double, WAVES>(sum, SumD(), lds_d, 0, wave, lane);
	if (t == 0) part[row * gridDim.x + blockIdx.x] = sum;
}

__global__ __launch_bounds__(TPB) void distill_slab_kernel(const DistillArgs a, const double *__restrict__ part) {
	extern __shared__ __align__(16) float lds[];
	__shared__ double lds_d[WAVES];
	__shared__ float lds_f[WAVES];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const long row = blockIdx.y;
	const int c0 = blockIdx.x * SLAB, c1 = min(a.cols, c0 + SLAB);
	const Entries e = entries_at(lds, a.top);
	const float *zr = a.z_re + row * a.ldz, *zi = a.z_im + row * a.ldz;
	float re[SLAB_COLS], im[SLAB_COLS];
#pragma unroll
	for (int k = 0; k < SLAB_COLS; ++k) {
		const int at = min(c0 + k * TPB + t, a.cols - 1);
		re[k] = zr[at];
		im[k] = zi[at];
	}
	double sum = 0.0;
	if (a.loss)
		for (int k = t; k < (int) gridDim.x; k += TPB) sum += part[row * gridDim.x + k];
	fetch_entries<TPB>(a, e, row, t);
	sum = group_reduce<double, WAVES>(sum, SumD(), lds_d, 0, wave, lane);  // (its barriers are the entries' as well)
	const float S = a.loss ? clamped((float) sum) : a.s[row];
	const float total = total_weight(e, lane);
	const bool none = total == 0.f;  // as in distill_kernel
	if (a.dz_re) {
		const float share = total / S;
#pragma unroll
		for (int k = 0; k < SLAB_COLS; ++k) {
			const int c = c0 + k * TPB + t;
			if (c < a.cols) distill_store(a, row, c, none ? 0.f : re[k] * share, none ? 0.f : -(im[k] * share));
		}
	}
	if (a.loss && blockIdx.x == 0) {
		const float loss = group_reduce<float, WAVES>(loss_terms<TPB>(a, e, S, t), SumF(), lds_f, 0, wave, lane);
		if (t == 0) {
			a.s[row] = S;
			a.loss[row] = loss;
		}
	}
	if (!a.dz_re) return;
	if (none) return;
	__syncthreads();
	entry_gradients<TPB>(a, e, row, S, total, t, c0, c1);
}

// ------------------------------------------------------------------------------------------------ vocabulary head
struct RowState {   // one entry per row of x, carried from launch to launch
	double *sum;    // sum |z|^2 so far
	double *part;   // [row][slabs]: what it is added up from, through a Gram matrix
	int slabs;
	double *weight; // 1 / S, or 0 where the row is left out: what x^H x is weighted with
	float *best;    // largest |z|^2 so far, and its first index
	int *index;
	float *c_re, *c_im;  // conj(z_label) / m, the label's share of the gradient
};

// sum |z|^2 and the largest |z|^2 over the columns of one piece of the logits, added to what the earlier pieces left.  Reads the
// logits from the memory-side cache, where the product has left them (4096 rows of 6144 columns, 201 MB: 34 us, beside 1400 for the product)
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

// ---- The loss through the Gram matrix of w.  The loss knows the logits z = x w^T through sum |z|^2 alone, a quadratic form of x:
// with T = w^H w (K x K), y = conj(x) T is what the logits' gradient hands back to x (before its division by S and without the
// label's term) and S = sum_j y_j x_j; and dw is conj(w) P with P = x^H diag(1 / S) x (again without the label's term).  So neither S
// nor either gradient needs the logits: N K^2 + B K^2 products stand for B N K.
// Where x lies in directions that w hardly has (or a row of w in directions that the batch hardly has) these sums are small and
// their terms are not.  With D = sum |x_i|^2 T_ii, what their terms amount to, a sum of rounded terms is off by D / S roundings, where the sum
// over the logits is off by about sqrt(D / S).  T, y, S and P are therefore formed and kept in double (gram.hip), which is
// closer than logits in single precision wherever these have a digit left (D / S up to 1e14).
struct HeadArgs {
	const float *x_re, *x_im, *w_re, *w_im;
	long ldx, ldw;
	const int *labels;
	float *s, *loss;
	int *argmax;
	const float *y_re, *y_im;  // conj(z) w, not yet divided by S
	float *xs_re, *xs_im;      // without a Gram matrix: the rows that are trained on, as the weights' gradient reads them; zeros elsewhere
	long ldy;                  // leading dimension of y and xs
	float *dx_re, *dx_im, *dxs_re, *dxs_im;
	long lddx;
	int accumulate_dx;
	int B, K, N;
};

// what a row's label makes of it
struct LabelTerm {
	int label;          // -1: none in the vocabulary
	bool live;          // false: the row is left out
	float loss;
	float c_re, c_im;   // conj(z_label) / m
};

// The label's logit is formed from x and w with its products summed in double: the gradient goes with its inverse, and an unlikely
// label has one near zero, of which a sum in single precision leaves few digits.  W wavefronts.
template <int W>
__device__ __forceinline__ LabelTerm label_term(const HeadArgs &a, long row, int label, float S, double *lds, int t, int lane, int wave) {
	const bool known = label >= 0 && label < a.N;
	double re = 0.0, im = 0.0;
	if (known) {
		const float *xr = a.x_re + row * a.ldx, *xi = a.x_im + row * a.ldx;
		const float *wr = a.w_re + label * a.ldw, *wi = a.w_im + label * a.ldw;
		for (int c = t; c < a.K; c += 64 * W) {
			re += (double) xr[c] * wr[c] - (double) xi[c] * wi[c];
			im += (double) xr[c] * wi[c] + (double) xi[c] * wr[c];
		}
	}
	re = group_reduce<double, W>(re, SumD(), lds, 0, wave, lane);
	im = group_reduce<double, W>(im, SumD(), lds, 0, wave, lane);
	const double power = re * re + im * im, m = clamped(power);
	LabelTerm l;
	l.label = known ? label : -1;
	l.loss = label < 0 ? 0.f : known ? -logf((float) clamped(power / (double) S)) : __builtin_nanf("");
	l.live = label >= 0;
	l.c_re = known ? (float) (re / m) : 0.f;
	l.c_im = known ? (float) (-im / m) : 0.f;
	return l;
}

// What is left to do for a row once its sum |z|^2 is known, by G wavefronts: S, the label's logit, loss, and the gradient at x: y / S
// minus the label's row of w times conj(z_label) / m.  For the weights' gradient, GRAM: the row's weight; otherwise xs = x / sqrt(S), so
// that both of its operands come from it: a row that is left out is zero in either, whatever it holds (padding may hold anything).
template <int G, int V, bool BWD, bool GRAM>
__device__ __forceinline__ void finish_row(const HeadArgs &a, const RowState &st, long row, double sum, double *lds, int t, int lane, int wave) {
	const float S = clamped((float) sum);
	int best = a.labels && !a.argmax ? 0 : st.index[row];
	if (best < 0 || best >= a.N) best = 0;  // a row of NaN has no largest entry
	const LabelTerm l = label_term<G>(a, row, a.labels ? a.labels[row] : best, S, lds, t, lane, wave);
	if (t == 0) {
		a.s[row] = S;
		if (a.loss) a.loss[row] = l.loss;
		if (a.argmax) a.argmax[row] = best;
	}
	if (!BWD) return;
	if (t == 0) {
		st.c_re[row] = l.c_re;
		st.c_im[row] = l.c_im;
		if (GRAM) st.weight[row] = l.live ? 1.0 / (double) S : 0.0;
	}
	const float *xr = a.x_re + row * a.ldx, *xi = a.x_im + row * a.ldx;
	const long label_row = (l.label < 0 ? 0 : l.label) * a.ldw;
	const float inv = 1.0f / S, root = (float) (1.0 / sqrt((double) S));
	for (int c = t * V; c < a.ldy; c += 64 * G * V) {
		const long o = row * a.ldy + c, d = row * a.lddx + c;
		float s_r[V] = {}, s_i[V] = {};
		if (c < a.K) {
			float g_r[V] = {}, g_i[V] = {};
			if (l.live) {
				float w_r[V], w_i[V];
				load_v<V>(g_r, a.y_re + o);
				load_v<V>(g_i, a.y_im + o);
				load_v<V>(w_r, a.w_re + label_row + c);
				load_v<V>(w_i, a.w_im + label_row + c);
				if (!GRAM) {
					load_v<V>(s_r, xr + c);
					load_v<V>(s_i, xi + c);
				}
#pragma unroll
				for (int k = 0; k < V; ++k) {
					g_r[k] = g_r[k] * inv - (l.c_re * w_r[k] - l.c_im * w_i[k]);
					g_i[k] = g_i[k] * inv - (l.c_re * w_i[k] + l.c_im * w_r[k]);
					s_r[k] *= root;
					s_i[k] *= root;
				}
			}
			auto give = [&](float *p, const float *v, float sign) {
				float u[V];
#pragma unroll
				for (int k = 0; k < V; ++k) u[k] = 0.f;
				if (a.accumulate_dx) load_v<V>(u, p + d);
#pragma unroll
				for (int k = 0; k < V; ++k) u[k] = a.accumulate_dx ? u[k] + sign * v[k] : sign * v[k];
				store_v<V>(p + d, u);
			};
			give(a.dx_re, g_r, 1.f);
			give(a.dx_im, g_i, 1.f);
			if (a.dxs_re) {
				give(a.dxs_re, g_r, 1.f);
				give(a.dxs_im, g_i, -1.f);
			}
		}
		if (!GRAM) {
			store_v<V>(a.xs_re + o, s_r);
			store_v<V>(a.xs_im + o, s_i);
		}
	}
}

// T threads per row (64: four rows to a workgroup).  GRAM: the sum is added up from its parts.  Rows beyond B, which fill up the last
// chunk of the weights' product, become zero in xs.
// Bound by memory: y and the labels' rows of w are read, dx written; 8192 x 1024, 201 MB, takes 42 us, 4.8 TB/s.
template <int T, int V, bool BWD, bool GRAM>
__global__ __launch_bounds__(TPB) void head_finish_kernel(const HeadArgs a, RowState st, int rows) {
	constexpr int G = T / 64, ROWS = TPB / T;
	__shared__ double lds_d[WAVES];
	const int slot = threadIdx.x / T, t = threadIdx.x % T, lane = threadIdx.x & 63, wave = t >> 6;
	const long row = (long) blockIdx.x * ROWS + slot;
	if (row >= rows) return;
	if (BWD && row >= a.B) {
		for (int c = t; c < a.ldy; c += T) a.xs_re[row * a.ldy + c] = a.xs_im[row * a.ldy + c] = 0.f;
		return;
	}
	double sum;
	if (GRAM) {  // (every wavefront for itself, and lane 0's for all of them)
		sum = 0.0;
		for (int k = lane; k < st.slabs; k += 64) sum += st.part[row * st.slabs + k];
		sum = __shfl(wave_reduce(sum, SumD()), 0);
	} else {
		sum = st.sum[row];
	}
	finish_row<G, V, BWD, GRAM>(a, st, row, sum, lds_d + slot * G, t, lane, wave);
}

// The logits of one row as a whole (two planes of leading dimension ldz, a multiple of four): S, the largest, the label's logit,
// loss; and, BWD, the logits overwritten with their gradient.  T threads per row.  The logits are few enough to be in the caches still:
// a launch (96 rows of 512: 5 us).
// st.c_re != NULL: the label's term is kept out of them, and goes to dx here and to dw behind the products.
template <int T, bool BWD>
__global__ __launch_bounds__(T) void head_row_kernel(const HeadArgs a, RowState st, float *__restrict__ z_re, float *__restrict__ z_im, long ldz) {
	constexpr int W = T / 64;
	__shared__ double lds_d[W];
	__shared__ ArgMax lds_a[W];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const long row = blockIdx.x;
	float *zr = z_re + row * ldz, *zi = z_im + row * ldz;
	// xs: the row as it is, zero if it is left out (whatever it holds) or beyond B
	auto keep = [&](bool live) {
		for (int c = t; c < a.ldy; c += T) {
			const bool in = live && c < a.K;
			a.xs_re[row * a.ldy + c] = in ? a.x_re[row * a.ldx + c] : 0.f;
			a.xs_im[row * a.ldy + c] = in ? a.x_im[row * a.ldx + c] : 0.f;
		}
	};
	const float zero[4] = {0.f, 0.f, 0.f, 0.f};
	if (BWD && row >= a.B) {
		for (int c = 4 * t; c < a.N; c += 4 * T) {
			store_v<4>(zr + c, zero);
			store_v<4>(zi + c, zero);
		}
		keep(false);
		return;
	}
	double sum = 0.0;
	ArgMax top = {-1.0f, 0x7fffffff};
	for (int c = 4 * t; c < a.N; c += 4 * T) {
		float u[4], v[4];
		load_v<4>(u, zr + c);
		load_v<4>(v, zi + c);
#pragma unroll
		for (int k = 0; k < 4; ++k)
			if (c + k < a.N) {
				sum = fma((double) v[k], (double) v[k], fma((double) u[k], (double) u[k], sum));
				const float q = fmaf(u[k], u[k], v[k] * v[k]);
				if (q > top.v) top = ArgMax{q, c + k};
			}
	}
	sum = group_reduce<double, W>(sum, SumD(), lds_d, 0, wave, lane);
	top = group_reduce<ArgMax, W>(top, ArgMaxOp(), lds_a, 0, wave, lane);
	const float S = clamped((float) sum);
	const int best = top.i < 0 || top.i >= a.N ? 0 : top.i;  // a row of NaN has no largest entry
	const LabelTerm l = label_term<W>(a, row, a.labels ? a.labels[row] : best, S, lds_d, t, lane, wave);
	if (t == 0) {
		a.s[row] = S;
		if (a.loss) a.loss[row] = l.loss;
		if (a.argmax) a.argmax[row] = best;
	}
	if (!BWD) return;
	keep(l.live);
	const float inv = 1.0f / S;
	const bool apart = st.c_re != nullptr;
	if (apart) {
		if (t == 0) {
			st.c_re[row] = l.c_re;
			st.c_im[row] = l.c_im;
		}
		for (int c = t; c < a.K; c += T) {
			float d_r = 0.f, d_i = 0.f;
			if (l.label >= 0) {
				const float w_r = a.w_re[l.label * a.ldw + c], w_i = a.w_im[l.label * a.ldw + c];
				d_r = l.c_im * w_i - l.c_re * w_r;
				d_i = -(l.c_re * w_i + l.c_im * w_r);
			}
			const long d = row * a.lddx + c;
			put(a.dx_re + d, d_r, a.accumulate_dx);
			put(a.dx_im + d, d_i, a.accumulate_dx);
			if (a.dxs_re) {
				put(a.dxs_re + d, d_r, a.accumulate_dx);
				put(a.dxs_im + d, -d_i, a.accumulate_dx);
			}
		}
	}
	for (int c = 4 * t; c < a.N; c += 4 * T) {
		if (!l.live) {
			store_v<4>(zr + c, zero);
			store_v<4>(zi + c, zero);
			continue;
		}
		float u[4], v[4];
		load_v<4>(u, zr + c);
		load_v<4>(v, zi + c);
#pragma unroll
		for (int k = 0; k < 4; ++k) {
			u[k] *= inv;
			v[k] *= -inv;
			if (!apart && c + k == l.label) {
				u[k] -= l.c_re;
				v[k] -= l.c_im;
			}
		}
		store_v<4>(zr + c, u);
		store_v<4>(zi + c, v);
	}
}

// ---- A few rows against the whole vocabulary (the next tokens of a batch of sequences): w is read once, and nothing of the logits
// leaves the registers.  A wavefront forms the logits of 16 entries for up to 16 MT rows with v_mfma_f32_16x16x4_f32, K in chunks of
// 64.  Lane (r, q), r = lane % 16, q = lane / 16, holds entry r of w at k = 16 q .. 16 q + 15 of the chunk: 64 bytes in a row, so
// that every line of w is fetched whole by one lane quarter after the other, and step j of the chunk multiplies the lanes' j-th
// values (the four k of a matrix instruction are 16 apart; x is laid out in LDS to match).  The next chunk of w is on its way in
// registers, and that of x for all four wavefronts, while the present one is multiplied.
// Bound by reading w up to 16 rows, by the matrix pipe beyond (four real products per complex one): 32768 entries of 1024 take 68 us
// for one row, 3.9 TB/s (a sum over 1 GiB: 3.9; 56 us where calls follow each other closely and find part of w in the memory-side
// cache), and 120 us for 48, 107 TFLOP/s (the tiles are two wavefronts per SIMD, so waits show).
typedef float floatx4 __attribute__((ext_vector_type(4)));

struct ScoreTile {   // what a workgroup leaves for every row
	double sum;
	float best;
	int index;
};

// four floats from element k of a row of K on; GUARD: what lies behind K is zero and not read
template <bool V4, bool GUARD>
__device__ __forceinline__ floatx4 load_quad(const float *p, int k, int K) {
	if (GUARD) {
		floatx4 v;
#pragma unroll
		for (int j = 0; j < 4; ++j) v[j] = k + j < K ? p[k + j] : 0.f;
		return v;
	}
	if (V4) return *reinterpret_cast<const floatx4 *>(p + k);
	return floatx4{p[k], p[k + 1], p[k + 2], p[k + 3]};
}

constexpr int CHUNK_K = 64;
// rows of x in LDS: [buffer][plane][four k][row] (an odd pitch: the 16 k groups of a row go to different banks)
template <int MT>
struct ScoreRows {
	floatx4 v[2][2][CHUNK_K / 4][16 * MT + 1];
};

// The logits of 16 MT rows at the lanes' entries: rr sums xr wr, ii xi wi, ri xr wi + xi wr.  w_re, w_im: the lane's entry; x_at[i]: offset
// of the row of x that the thread lays out as number (t + TPB i) / 16.
template <int MT, bool V4>
__device__ __forceinline__ void score_tile(const HeadArgs &a, const float *w_re, const float *w_im, const long (&x_at)[MT], ScoreRows<MT> &xs,
		floatx4 (&rr)[MT], floatx4 (&ii)[MT], floatx4 (&ri)[MT]) {
	const int t = threadIdx.x, lane = t & 63, r = lane & 15, q = lane >> 4;
#pragma unroll
	for (int m = 0; m < MT; ++m) rr[m] = ii[m] = ri[m] = floatx4{0.f, 0.f, 0.f, 0.f};
	floatx4 w[2][4], w_next[2][4], x_next[2 * MT];
	const int chunks = (a.K + CHUNK_K - 1) / CHUNK_K;
	auto fetch = [&](int c) {
		const int k0 = c * CHUNK_K;
		if (k0 + CHUNK_K <= a.K) {
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				w_next[0][j] = load_quad<V4, false>(w_re, k0 + 16 * q + 4 * j, a.K);
				w_next[1][j] = load_quad<V4, false>(w_im, k0 + 16 * q + 4 * j, a.K);
			}
#pragma unroll
			for (int i = 0; i < 2 * MT; ++i) x_next[i] = load_quad<V4, false>((i < MT ? a.x_re : a.x_im) + x_at[i % MT], k0 + 4 * (t % 16), a.K);
		} else {
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				w_next[0][j] = load_quad<V4, true>(w_re, k0 + 16 * q + 4 * j, a.K);
				w_next[1][j] = load_quad<V4, true>(w_im, k0 + 16 * q + 4 * j, a.K);
			}
#pragma unroll
			for (int i = 0; i < 2 * MT; ++i) x_next[i] = load_quad<V4, true>((i < MT ? a.x_re : a.x_im) + x_at[i % MT], k0 + 4 * (t % 16), a.K);
		}
	};
	fetch(0);
	for (int c = 0; c < chunks; ++c) {
#pragma unroll
		for (int p = 0; p < 2; ++p)
#pragma unroll
			for (int j = 0; j < 4; ++j) w[p][j] = w_next[p][j];
		// (the buffer was last read two chunks ago, before the barrier of the chunk between)
#pragma unroll
		for (int i = 0; i < 2 * MT; ++i) xs.v[c & 1][i / MT][t % 16][(t + TPB * (i % MT)) / 16] = x_next[i];
		__syncthreads();
		if (c + 1 < chunks) fetch(c + 1);
		__builtin_amdgcn_sched_barrier(0);  // (the loads go out before the products, not after them)
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			floatx4 xr[MT], xi[MT];
#pragma unroll
			for (int m = 0; m < MT; ++m) {
				xr[m] = xs.v[c & 1][0][4 * q + j][16 * m + r];
				xi[m] = xs.v[c & 1][1][4 * q + j][16 * m + r];
			}
#pragma unroll
			for (int e = 0; e < 4; ++e) {
#pragma unroll
				for (int m = 0; m < MT; ++m) rr[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(xr[m][e], w[0][j][e], rr[m], 0, 0, 0);
#pragma unroll
				for (int m = 0; m < MT; ++m) ii[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(xi[m][e], w[1][j][e], ii[m], 0, 0, 0);
#pragma unroll
				for (int m = 0; m < MT; ++m) ri[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(xr[m][e], w[1][j][e], ri[m], 0, 0, 0);
#pragma unroll
				for (int m = 0; m < MT; ++m) ri[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(xi[m][e], w[0][j][e], ri[m], 0, 0, 0);
			}
		}
	}
}

template <int MT, bool V4>
__global__ __launch_bounds__(TPB) void head_score_kernel(const HeadArgs a, int B, ScoreTile *__restrict__ part) {
	constexpr int ROWS = 16 * MT;
	__shared__ ScoreRows<MT> xs;
	__shared__ ScoreTile met[WAVES][ROWS];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6, r = lane & 15, q = lane >> 4;
	const int n0 = (blockIdx.x * WAVES + wave) * 16;
	// lanes beyond the last entry or row read the last one again; their results are masked
	const long entry = (long) min(n0 + r, a.N - 1) * a.ldw;
	long x_at[MT];
#pragma unroll
	for (int i = 0; i < MT; ++i) x_at[i] = min((t + TPB * i) / 16, B - 1) * a.ldx;
	floatx4 rr[MT], ii[MT], ri[MT];
	score_tile<MT, V4>(a, a.w_re + entry, a.w_im + entry, x_at, xs, rr, ii, ri);
	// element i of a lane: entry n0 + r, row 16 m + 4 q + i; the 16 lanes of a quarter are combined in a fixed order
	const bool in = n0 + r < a.N;
#pragma unroll
	for (int m = 0; m < MT; ++m)
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const float z_r = rr[m][i] - ii[m][i], z_i = ri[m][i];
			double sum = in ? fma((double) z_i, (double) z_i, (double) z_r * z_r) : 0.0;
			ArgMax best = {in ? fmaf(z_r, z_r, z_i * z_i) : -1.f, n0 + r};
			if (!(best.v >= 0.f)) best.v = -1.f;  // a NaN is no entry's largest, and would be kept by whoever compares with it
			sum += exchange<double, 0>(sum);
			sum += exchange<double, 1>(sum);
			sum += exchange<double, 2>(sum);
			sum += exchange<double, 3>(sum);
			best = ArgMaxOp()(best, exchange<ArgMax, 0>(best));
			best = ArgMaxOp()(best, exchange<ArgMax, 1>(best));
			best = ArgMaxOp()(best, exchange<ArgMax, 2>(best));
			best = ArgMaxOp()(best, exchange<ArgMax, 3>(best));
			if (r == 0) met[wave][16 * m + 4 * q + i] = ScoreTile{sum, best.v, best.i};
		}
	__syncthreads();
	if (t < B) {
		ScoreTile x = met[0][t];
#pragma unroll
		for (int w = 1; w < WAVES; ++w) {
			const ScoreTile y = met[w][t];
			x.sum += y.sum;
			if (y.best > x.best) {  // (the entries of a later wavefront are larger numbers)
				x.best = y.best;
				x.index = y.index;
			}
		}
		part[(long) t * gridDim.x + blockIdx.x] = x;
	}
}

// One workgroup per row: its tiles, then its label (32768 entries: 5 us, a launch)
__global__ __launch_bounds__(TPB) void head_score_finish_kernel(const HeadArgs a, const ScoreTile *__restrict__ part, int tiles) {
	__shared__ double lds_d[WAVES];
	__shared__ ArgMax lds_a[WAVES];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const long row = blockIdx.x;
	double sum = 0.0;
	ArgMax top = {-1.0f, 0x7fffffff};
	for (int k = t; k < tiles; k += TPB) {
		const ScoreTile x = part[row * tiles + k];
		sum += x.sum;
		if (x.best > top.v) top = ArgMax{x.best, x.index};
	}
	sum = group_reduce<double, WAVES>(sum, SumD(), lds_d, 0, wave, lane);
	top = group_reduce<ArgMax, WAVES>(top, ArgMaxOp(), lds_a, 0, wave, lane);
	const float S = clamped((float) sum);
	const int best = top.i < 0 || top.i >= a.N ? 0 : top.i;  // a row of NaN has no largest entry
	const LabelTerm l = label_term<WAVES>(a, row, a.labels ? a.labels[row] : best, S, lds_d, t, lane, wave);
	if (t == 0) {
		a.s[row] = S;
		if (a.loss) a.loss[row] = l.loss;
		if (a.argmax) a.argmax[row] = best;
	}
}

struct ScatterArgs {
	const int *row_of, *label_of;  // the rows in order of their labels
	const float *c_re, *c_im, *x_re, *x_im;
	long ldx;
	float *dw_re, *dw_im, *dws_re, *dws_im;
	long lddw;
	float *part;  // [chunk][began before, begins here][re, im][ldk]
	long ldk;
	int B, K, N;
};

// ---- The label's term of the weights' gradient: dw[label[r]] -= c_r x_r for every row r.  Labels of a text repeat (the most
// frequent token of a batch of 8192 names hundreds of rows), so the rows are put in order of their labels first and then worked
// off in chunks of equal length, whatever the labels.  The order is the stable one, so a label's rows are added in order.
constexpr int ORDER_ROWS = 8192;  // rows ordered together (their labels fill 32 KB of LDS); longer batches go block by block
constexpr int CHUNK = 16;         // ordered rows of one workgroup
constexpr int RANK_ROWS = 32;     // rows of one workgroup of head_order_kernel

// Orders the rows [y ORDER_ROWS, ..) by (label, row), rows without a label of the vocabulary last: workgroup (x, y) counts for each of
// 32 rows how many come before it, its 32 half wavefronts sharing the labels to compare with (8192 rows: 67 million comparisons over
// 256 workgroups, 12 us; a sorting network in one workgroup took 80).  row_of = -1 and label_of = N where there
// is no label.
__global__ __launch_bounds__(1024) void head_order_kernel(const int *__restrict__ labels, int B, int N, int *__restrict__ row_of,
		int *__restrict__ label_of) {
	__shared__ __align__(16) int keys[ORDER_ROWS];
	constexpr int SHARES = 1024 / RANK_ROWS;
	__shared__ int count[SHARES][RANK_ROWS];
	const int first = blockIdx.y * ORDER_ROWS, n = min(ORDER_ROWS, B - first), n4 = (n + 3) / 4 * 4;
	const int lane = threadIdx.x % RANK_ROWS, share = threadIdx.x / RANK_ROWS, lo = blockIdx.x * RANK_ROWS, i = lo + lane;
	if (lo >= n) return;
	for (int k = threadIdx.x; k < n4; k += 1024) {
		const int label = k < n ? labels[first + k] : -1;
		keys[k] = k >= n ? 0x7fffffff : label >= 0 && label < N ? label : N;
	}
	__syncthreads();
	const int key = keys[min(i, n - 1)];
	const int per = ((n4 / 4 + SHARES - 1) / SHARES) * 4, j0 = min(n4, share * per), j1 = min(n4, j0 + per);
	int before = 0;
#pragma unroll 4
	for (int j = j0; j < j1; j += 4) {
		const int4 other = *reinterpret_cast<const int4 *>(keys + j);
		// an equal label counts where its row comes first: j + d < i
		if (j >= lo && j < lo + RANK_ROWS) {
			before += (other.x < key + (j < i)) + (other.y < key + (j + 1 < i)) + (other.z < key + (j + 2 < i)) + (other.w < key + (j + 3 < i));
		} else {
			const int limit = key + (j < lo);
			before += (other.x < limit) + (other.y < limit) + (other.z < limit) + (other.w < limit);
		}
	}
	count[share][lane] = before;
	__syncthreads();
	if (share || i >= n) return;
	int rank = 0;
#pragma unroll
	for (int k = 0; k < SHARES; ++k) rank += count[k][lane];
	label_of[first + rank] = key;
	row_of[first + rank] = key < N ? first + i : -1;
}

// V columns of one label's row of the gradient: its planes, and the label's sum subtracted from them
template <int V>
struct LabelRow {
	float v[4][V];
	__device__ __forceinline__ void load(const ScatterArgs &a, int label, int c) {
		const long o = (long) label * a.lddw + c;
		load_v<V>(v[0], a.dw_re + o);
		load_v<V>(v[1], a.dw_im + o);
		if (a.dws_re) {
			load_v<V>(v[2], a.dws_re + o);
			load_v<V>(v[3], a.dws_im + o);
		}
	}
	__device__ __forceinline__ void subtract(const ScatterArgs &a, int label, int c, const float *re, const float *im) {
		const long o = (long) label * a.lddw + c;
#pragma unroll
		for (int k = 0; k < V; ++k) {
			v[0][k] -= re[k];
			v[1][k] -= im[k];
			v[2][k] -= re[k];
			v[3][k] += im[k];
		}
		store_v<V>(a.dw_re + o, v[0]);
		store_v<V>(a.dw_im + o, v[1]);
		if (a.dws_re) {
			store_v<V>(a.dws_re + o, v[2]);
			store_v<V>(a.dws_im + o, v[3]);
		}
	}
};

// Workgroup (x, y): the ordered rows [CHUNK x, CHUNK x + CHUNK) of the block that starts at `first`, V columns per thread.  A run of
// one label that lies inside the chunk is subtracted at once; the part of a run that reaches over the chunk's ends goes to
// part[x][0] (it began before) or part[x][1] (it begins here).
// Reads x and what it changes of dw: 8192 rows of 1024, 36 us; 1000 of 333, 8 us.
template <int V>
__global__ __launch_bounds__(TPB) void head_label_kernel(const ScatterArgs a, int first) {
	__shared__ int label_at[CHUNK + 2], row_at[CHUNK];  // label_at[k + 1]: ordered row k of the chunk, and its neighbours
	__shared__ float c_at[2][CHUNK];
	const int t = threadIdx.x, c = (blockIdx.y * TPB + t) * V;
	const int p0 = first + blockIdx.x * CHUNK, block_end = min(a.B, first + ORDER_ROWS);
	if (t < CHUNK + 2) {
		const int p = p0 + t - 1;
		const int l = p >= first && p < block_end ? a.label_of[p] : -1;
		label_at[t] = l >= a.N ? -1 : l;
		if (t > 0 && t <= CHUNK) {
			const int r = l >= 0 && l < a.N ? a.row_of[p] : 0;
			row_at[t - 1] = r;
			c_at[0][t - 1] = a.c_re[r];
			c_at[1][t - 1] = a.c_im[r];
		}
	}
	__syncthreads();
	if (c >= a.K) return;
	float re[V], im[V];
	int begin = 0;
	constexpr int AHEAD = V == 4 ? 4 : 8;  // rows of x, and of the gradient they may end up in, in flight
#pragma unroll
	for (int k0 = 0; k0 < CHUNK; k0 += AHEAD) {
		float x_r[AHEAD][V], x_i[AHEAD][V];
		LabelRow<V> dst[AHEAD];
#pragma unroll
		for (int u = 0; u < AHEAD; ++u) {  // (a place without a label reads row 0 and is not used)
			load_v<V>(x_r[u], a.x_re + (long) row_at[k0 + u] * a.ldx + c);
			load_v<V>(x_i[u], a.x_im + (long) row_at[k0 + u] * a.ldx + c);
			dst[u].load(a, max(label_at[k0 + u + 1], 0), c);
		}
#pragma unroll
		for (int u = 0; u < AHEAD; ++u) {
			const int k = k0 + u, label = label_at[k + 1];
			if (label < 0) return;  // rows without a label are last
			if (k == 0 || label_at[k] != label) {
				begin = k;
#pragma unroll
				for (int q = 0; q < V; ++q) re[q] = im[q] = 0.f;
			}
			const float c_re = c_at[0][k], c_im = c_at[1][k];
#pragma unroll
			for (int q = 0; q < V; ++q) {
				re[q] += c_re * x_r[u][q] - c_im * x_i[u][q];
				im[q] += c_re * x_i[u][q] + c_im * x_r[u][q];
			}
			const bool same = label_at[k + 2] == label;
			if (same && k + 1 < CHUNK) continue;
			const bool began = begin == 0 && label_at[0] == label;
			if (!began && !same) {
				dst[u].subtract(a, label, c, re, im);
			} else {
				float *part = a.part + ((long) blockIdx.x * 2 + (began ? 0 : 1)) * 2 * a.ldk + c;
				store_v<V>(part, re);
				store_v<V>(part + a.ldk, im);
			}
		}
	}
}

// The runs that reach over chunks: the chunk that such a run begins in adds up its parts in order (8192 rows: 15 us)
template <int V>
__global__ __launch_bounds__(TPB) void head_label_join_kernel(const ScatterArgs a, int first) {
	const int c = (blockIdx.y * TPB + threadIdx.x) * V;
	const int p0 = first + blockIdx.x * CHUNK, block_end = min(a.B, first + ORDER_ROWS), p1 = p0 + CHUNK;
	if (p1 >= block_end || c >= a.K) return;
	const int label = a.label_of[p1 - 1];
	if (label >= a.N || a.label_of[p1] != label) return;            // nothing reaches over this chunk's end
	if (p0 > first && a.label_of[p0 - 1] == label) return;         // it began earlier
	int chunks = 1;                                                 // further chunks that hold a part of it
	while (p1 + chunks * CHUNK < block_end && a.label_of[p1 + chunks * CHUNK] == label) ++chunks;
	const float *part = a.part + ((long) blockIdx.x * 2 + 1) * 2 * a.ldk + c;
	LabelRow<V> dst;
	dst.load(a, label, c);
	float re[V], im[V];
	load_v<V>(re, part);
	load_v<V>(im, part + a.ldk);
#pragma unroll 4
	for (int k = 1; k <= chunks; ++k) {
		float x[V], y[V];
		const float *more = part + (k * 2 - 1) * 2 * a.ldk;
		load_v<V>(x, more);
		load_v<V>(y, more + a.ldk);
#pragma unroll
		for (int q = 0; q < V; ++q) {
			re[q] += x[q];
			im[q] += y[q];
		}
	}
	dst.subtract(a, label, c, re, im);
}

// Copies of both operands: dst[plane][r][c] = src_plane[r][c] inside rows x cols, zero outside.  The first blocks x copy x, the
// others w; blockIdx.y = plane.  One thread per four columns of dst.  1000 + 5003 rows of 333: 8 us.
struct PackArgs {
	const float *re[2], *im[2];
	long lds[2];
	float *dst[2];
	int rows[2], rows_d[2], blocks_x, cols, ldd;
};
__global__ __launch_bounds__(TPB) void head_pack_kernel(const PackArgs a) {
	const bool w = blockIdx.x >= (unsigned) a.blocks_x;
	const int groups = a.ldd / 4;
	const long rows_d = w ? a.rows_d[1] : a.rows_d[0], idx = (long) (blockIdx.x - (w ? a.blocks_x : 0)) * TPB + threadIdx.x;
	if (idx >= rows_d * groups) return;
	const long r = idx / groups;
	const int c0 = (int) (idx - r * groups) * 4;
	const float *s = (w ? (blockIdx.y ? a.im[1] : a.re[1]) : (blockIdx.y ? a.im[0] : a.re[0])) + r * (w ? a.lds[1] : a.lds[0]);
	float v[4] = {0.f, 0.f, 0.f, 0.f};
	if (r < (w ? a.rows[1] : a.rows[0])) {
#pragma unroll
		for (int k = 0; k < 4; ++k)
			if (c0 + k < a.cols) v[k] = s[c0 + k];
	}
	store_v<4>((w ? a.dst[1] : a.dst[0]) + (blockIdx.y * rows_d + r) * a.ldd + c0, v);
}

// the gradient of no rows at all
__global__ __launch_bounds__(TPB) void head_clear_kernel(float *p, long ld, int rows, int cols) {
	for (long r = blockIdx.x; r < rows; r += gridDim.x)
		for (int c = threadIdx.x; c < cols; c += TPB) p[r * ld + c] = 0.f;
}

}  // namespace

using namespace cnet;

// loss == NULL: the backward pass alone, dz_re == NULL: the forward pass alone
static int distill(const DistillArgs &a) {
	const bool vec = a.cols % 4 == 0 && a.ldz % 4 == 0 && aligned16(a.z_re) && aligned16(a.z_im) && (!a.dz_re || a.lddz % 4 == 0) && aligned16(a.dz_re) &&
			aligned16(a.dz_im) && aligned16(a.dzs_re) && aligned16(a.dzs_im);
	const size_t entries = (size_t) 4 * entry_slots(a.top) * sizeof(float);
	const int cus = rt().prop.multiProcessorCount;
	// rows that are longer than 8192 columns and fewer than a quarter of the compute units are dealt out; of the others, a workgroup
	// holds one of up to 32768 columns, and as much of a longer one
	if (a.cols > 8192 && 4L * a.rows < cus) {
		const int slabs = (a.cols + SLAB - 1) / SLAB;
		double *part = (double *) workspace((size_t) a.rows * slabs * sizeof(double));
		if (!part) return rt().capturing ? CNET_ERR_UNSUPPORTED : CNET_ERR_OUT_OF_MEMORY;
		const dim3 grid((unsigned) slabs, (unsigned) a.rows);
		if (a.loss) hipLaunchKernelGGL(distill_slab_sum_kernel, grid, dim3(TPB), 0, rt().stream, a, part);
		hipLaunchKernelGGL(distill_slab_kernel, grid, dim3(TPB), entries, rt().stream, a, part);
		CNET_LAUNCH_CHECK();
		return CNET_OK;
	}
	// (8192 x 32768, read once and written once, repeated on the same planes: 772 us with the streaming hint on both sides, 801 on the stores, 862 on the loads, 824
	// with none; 5.6 TB/s)
	const int policy = stream_policy(a.dz_re ? ST_BOTH : ST_LOADS, !a.dz_re ? 2 : a.dzs_re ? 6 : 4, (long) a.rows * a.cols);
#define CNET_DISTILL(T, E, LONG)                                                                                                                     \
	do {                                                                                                                                       \
		const dim3 grid((unsigned) ((a.rows + (T < TPB ? TPB / T : 1) - 1) / (T < TPB ? TPB / T : 1))), block(T < TPB ? TPB : T);                \
		if (vec) hipLaunchKernelGGL((distill_kernel<T, E / 4, 4, LONG>), grid, block, entries * (T < TPB ? TPB / T : 1), rt().stream, a, policy);       \
		else hipLaunchKernelGGL((distill_kernel<T, E, 1, LONG>), grid, block, entries * (T < TPB ? TPB / T : 1), rt().stream, a, policy);               \
	} while (0)
	if (a.cols <= 512 && a.top <= 64) CNET_DISTILL(64, 8, false);
	else if (a.cols <= 2048) CNET_DISTILL(256, 8, false);
	else if (a.cols <= 4096) CNET_DISTILL(256, 16, false);
	else if (a.cols <= 8192) CNET_DISTILL(256, 32, false);
	else if (a.cols <= 16384) CNET_DISTILL(1024, 16, false);
	else if (a.cols <= 32768) CNET_DISTILL(1024, 32, false);
	else CNET_DISTILL(1024, 32, true);
#undef CNET_DISTILL
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

// what the calls of the head keep between their launches, carved out of one buffer of the library
struct HeadBuffers {
	RowState st;
	float *piece, *y, *xs;         // planes re, im
	Gram64 gram;                   // T, then P
	float *x, *w;                  // copies of the operands (HeadPad)
	int *row_of, *label_of;
	float *label_part;
	int piece_cols;                // columns of one piece, also its leading dimension
	long ldk;                      // leading dimension of y and xs
};

struct HeadPlan {
	bool bwd, whole, gram, pieces;
	bool label;  // the label's terms go to dx and dw by themselves
	int piece_cols;
};

// A piece of logits (two planes of B rows) is as wide as the memory-side cache holds: the pass over it, and the product that
// reads it, then find it there.
static long piece_bytes() {
	static const long mb = [] {
		const char *e = getenv("CNET_HEAD_PIECE_MB");  // tuning override
		return e && atol(e) > 0 ? atol(e) : 192L;
	}();
	return mb << 20;
}

// Whether the label's terms go to dx and dw by themselves where the logits lie whole: three launches, 15 us, for digits.  dx off by,
// among the others / apart: 300 x 1500 x 40000 1.6e-6 / 6e-8 (3761 -> 3784 us), 531 x 1000 x 4000 8e-7 / 5e-8; what
// is left among the others (sums of 1024, or calls of less than about 130 us, whose sums the wavefronts share) stays within 5e-7
// (1000 x 600 x 900, 89 x 1063 x 2620 4e-7, 300 x 128 x 4000 3e-7).
static bool label_apart(int B, int K, int N) {
	const int longest = std::max(B, N);
	return longest > 4096 || (longest > 1024 && (double) B * N * K > (double) (1 << 28));
}

// Which way the call goes, by what its launches take: an fp32 product of m complex multiplications about 8 us + 8 m flop at 115
// TFLOP/s, the products in double by their matrix instructions, any other kernel about 3 us, plus its bytes.  Steps without the argmax, the
// logits as a whole / through the Gram matrices, both measured: 1188 x 125 -> 1869 155 / 108 us, 1155 x 551 -> 862 202 / 243, 7365 x 490 -> 633
// 601 / 524, 1624 x 1537 -> 305 269 / 1071, 2333 x 594 -> 5021 1471 / 636, 2183 x 1696 -> 8441 5689 / 4816, 331 x 675 -> 1215 138 / 280.
//   whole   the logits in one piece, turned into their gradient where they lie; dx and dw from it: three products, one kernel.  The
//           label's large entry among them costs the products' sums digits as they get long (label_apart)
//   pieces  the logits piece by piece, and a second time for dw; the label's term by itself
//   gram    T over N, y over K, P = x^H (x / S) over B, dw from it over K, all in double; the label's term by itself.  The argmax needs
//           the logits all the same.
static HeadPlan head_plan(int B, int K, int N, bool bwd, bool argmax) {
	static const int forced = [] {
		const char *e = getenv("CNET_HEAD_GRAM");  // tuning override: 0 / 1 never / always through the Gram matrix
		return e ? atoi(e) : -1;
	}();
	HeadPlan p;
	p.bwd = bwd;
	const long all = ((long) N + 63) / 64 * 64;
	p.piece_cols = (int) std::min(all, std::max(64L, piece_bytes() / (8 * (long) B) / 64 * 64));
	const int pieces = (N + p.piece_cols - 1) / p.piece_cols;
	const double b = B, k = K, n = N;
	auto product = [](double m) { return 8.0 + m * 8 / 115e6; };
	auto bytes = [](double v) { return 3.0 + v / 4e6; };
	const double label = bwd ? 20 + bytes(60 * b * k) : 0;
	const double scan = pieces * (product(b * n * k / pieces) + bytes(8 * b * n / pieces));
	double direct, gram = gram64_us(K, N) + times_gram_us(B, K) + (argmax ? scan : 0.0) + bytes(bwd ? 24 * b * k : 0.0);
	if (pieces == 1) direct = scan + (bwd ? bytes(16 * b * n) + 2 * product(b * n * k) + (label_apart(B, K, N) ? label : 0) : 0);
	else direct = scan + bytes(24 * b * k) + (bwd ? pieces * 3 * product(b * n * k / pieces) + label : 0);
	if (bwd) gram += gram64_us(K, B) + times_gram_us(N, K) + label;
	p.gram = (bwd || !argmax) && (forced >= 0 ? forced != 0 : gram < direct);
	p.whole = !p.gram && pieces == 1;
	p.label = bwd && (!p.whole || label_apart(B, K, N));
	p.pieces = !p.whole && (argmax || !p.gram);
	return p;
}

// Widths that do not suit the matrix kernels (128-bit transfers, whole chunks of 16 along the summed axis) cost them a copy of w in
// front of every product, or a second launch over the whole result for the rest of a chunk (300 x 1500 -> 40000: 0.9 ms for the
// last 12 of 300 rows).  A large head therefore copies x and w once, zeros filling the last chunks, and its own buffers
// have rows to spare.
struct HeadPad {
	bool copy;  // of x and w
	int B, K, N;
};
static HeadPad head_pad(const HeadArgs &a, int B, const HeadPlan &plan) {
	auto up = [](int v) { return (v + 15) / 16 * 16; };
	HeadPad p = {false, B, a.K, a.N};
	if ((double) a.N * a.K < (double) (1 << 18) || (plan.gram && !plan.pieces)) return p;  // (the products in double take any layout)
	if (plan.bwd && !plan.gram) p.B = up(B);
	const bool odd = a.K % 16 || a.ldx % 4 || a.ldw % 4 || !aligned16(a.x_re) || !aligned16(a.x_im) || !aligned16(a.w_re) || !aligned16(a.w_im);
	if (odd && 8.0 * up(a.N) * up(a.K) <= (double) (1L << 31)) {
		p.copy = true;
		p.K = up(a.K);
		p.N = up(a.N);
	}
	return p;
}

static int head_buffers(const HeadPad &pad, const HeadPlan &plan, int K, HeadBuffers &b) {
	b.piece_cols = plan.piece_cols;
	b.ldk = ((long) pad.K + 3) / 4 * 4;
	const size_t rows = ((size_t) pad.B + 63) / 64 * 64;
	const size_t piece = plan.pieces || plan.whole ? 2 * (size_t) pad.B * b.piece_cols : 0;
	const size_t wide = plan.bwd ? 2 * (size_t) pad.B * b.ldk : 0, xs = plan.gram ? 0 : wide;
	b.gram.ld = K;
	b.st.slabs = (K + GRAM_TILE - 1) / GRAM_TILE;
	const size_t square = plan.gram ? 4 * (size_t) K * K : 0, part = plan.gram ? 2 * (size_t) b.st.slabs * rows : 0, weight = plan.gram ? 2 * rows : 0;
	const bool label = plan.label;
	const size_t order = label ? rows : 0, label_part = label ? (size_t) (std::min(pad.B, ORDER_ROWS) + CHUNK - 1) / CHUNK * 4 * b.ldk : 0;
	const size_t copy_x = pad.copy ? 2 * (size_t) pad.B * b.ldk : 0, copy_w = pad.copy ? 2 * (size_t) pad.N * b.ldk : 0;
	float *p = (float *) vocab_workspace((6 * rows + square + part + weight + piece + wide + xs + 2 * order + label_part + copy_x + copy_w) * sizeof(float));
	if (!p) return rt().capturing ? CNET_ERR_UNSUPPORTED : CNET_ERR_OUT_OF_MEMORY;
	auto take = [&](size_t floats) {
		float *q = p;
		p += floats;
		return q;
	};
	b.st.sum = (double *) take(2 * rows);
	b.gram.re = (double *) take(square);
	b.st.part = (double *) take(part);
	b.st.weight = (double *) take(weight);
	b.st.best = take(rows);
	b.st.index = (int *) take(rows);
	b.st.c_re = take(rows);
	b.st.c_im = take(rows);
	b.piece = take(piece);
	b.y = take(wide);
	b.xs = take(xs);
	b.label_part = take(label_part);
	b.row_of = (int *) take(order);
	b.label_of = (int *) take(order);
	b.x = take(copy_x);
	b.w = take(copy_w);
	return CNET_OK;
}

// C = conj(A) B, A row-major or k-major, B k-major
static int conj_product(int a_kmajor, int M, int N, int K, const float *a_re, const float *a_im, long lda, const float *b_re, const float *b_im, long ldb,
		float *c_re, float *c_im, long ldc, int accumulate) {
	return cnet_cgemm_batched(a_kmajor, 1, 1, 0, M, N, K, a_re, a_im, lda, 0, b_re, b_im, ldb, 0, c_re, c_im, ldc, 0, 1, accumulate);
}

// a gradient's pair of planes from C = conj(A) B: with the dz* half wanted, A conj(B) is formed for that half and mirrored into
// the other
static int conj_product_pair(bool a_kmajor, int M, int N, int K, const float *a_re, const float *a_im, long lda, const float *b_re, const float *b_im,
		long ldb, float *c_re, float *c_im, float *cs_re, float *cs_im, long ldc, int accumulate) {
	if (!cs_re) return conj_product(a_kmajor, M, N, K, a_re, a_im, lda, b_re, b_im, ldb, c_re, c_im, ldc, accumulate);
	const float *ar[2] = {a_re, a_re}, *ai[2] = {a_im, a_im}, *br[2] = {b_re, b_re}, *bi[2] = {b_im, b_im};
	float *cr[2] = {cs_re, c_re}, *ci[2] = {cs_im, c_im};
	const bool cj[2] = {true, true};
	return cgemm_pair(a_kmajor, true, 1, M, N, K, ar, ai, lda, br, bi, ldb, cj, cr, ci, ldc, accumulate, 0, 1);
}

static int head_labels(const HeadArgs &a, const HeadBuffers &b, int B, float *dw_re, float *dw_im, float *dws_re, float *dws_im, long lddw) {
	const dim3 blocks((unsigned) ((std::min(B, ORDER_ROWS) + RANK_ROWS - 1) / RANK_ROWS), (unsigned) ((B + ORDER_ROWS - 1) / ORDER_ROWS));
	hipLaunchKernelGGL(head_order_kernel, blocks, dim3(1024), 0, rt().stream, a.labels, B, a.N, b.row_of, b.label_of);
	CNET_LAUNCH_CHECK();
	const ScatterArgs sc = {b.row_of, b.label_of, b.st.c_re, b.st.c_im, a.x_re, a.x_im, a.ldx, dw_re, dw_im, dws_re, dws_im, lddw, b.label_part, b.ldk,
			B, a.K, a.N};
	const bool vec = a.K % 4 == 0 && a.ldx % 4 == 0 && lddw % 4 == 0 && aligned16(a.x_re) && aligned16(a.x_im) && aligned16(dw_re) && aligned16(dw_im) &&
			aligned16(dws_re) && aligned16(dws_im);
	const int per_group = TPB * (vec ? 4 : 1);
	for (int first = 0; first < B; first += ORDER_ROWS) {
		const dim3 grid((unsigned) ((std::min(B - first, ORDER_ROWS) + CHUNK - 1) / CHUNK), (unsigned) ((a.K + per_group - 1) / per_group));
		if (vec) {
			hipLaunchKernelGGL(head_label_kernel<4>, grid, dim3(TPB), 0, rt().stream, sc, first);
			hipLaunchKernelGGL(head_label_join_kernel<4>, grid, dim3(TPB), 0, rt().stream, sc, first);
		} else {
			hipLaunchKernelGGL(head_label_kernel<1>, grid, dim3(TPB), 0, rt().stream, sc, first);
			hipLaunchKernelGGL(head_label_join_kernel<1>, grid, dim3(TPB), 0, rt().stream, sc, first);
		}
		CNET_LAUNCH_CHECK();
	}
	return CNET_OK;
}

// rows that head_score_kernel takes, where their logits are too many for the small-C kernel (4 tiles of 16 x 16 per compute unit, in a
// few microseconds with the pass over them)
constexpr int SCORE_ROWS = 64;

static int head_score(const HeadArgs &a, int B) {
	const int tiles = (a.N + 16 * WAVES - 1) / (16 * WAVES);
	ScoreTile *part = (ScoreTile *) vocab_workspace((size_t) tiles * B * sizeof(ScoreTile));
	if (!part) return rt().capturing ? CNET_ERR_UNSUPPORTED : CNET_ERR_OUT_OF_MEMORY;
	const bool v4 = a.ldx % 4 == 0 && a.ldw % 4 == 0 && aligned16(a.x_re) && aligned16(a.x_im) && aligned16(a.w_re) && aligned16(a.w_im);
#define CNET_SCORE(MT)                                                                                                          \
	do {                                                                                                                        \
		if (v4) hipLaunchKernelGGL((head_score_kernel<MT, true>), dim3((unsigned) tiles), dim3(TPB), 0, rt().stream, a, B, part);  \
		else hipLaunchKernelGGL((head_score_kernel<MT, false>), dim3((unsigned) tiles), dim3(TPB), 0, rt().stream, a, B, part);    \
	} while (0)
	if (B <= 16) CNET_SCORE(1);
	else if (B <= 32) CNET_SCORE(2);
	else if (B <= 48) CNET_SCORE(3);
	else CNET_SCORE(4);
#undef CNET_SCORE
	CNET_LAUNCH_CHECK();
	hipLaunchKernelGGL(head_score_finish_kernel, dim3((unsigned) B), dim3(TPB), 0, rt().stream, a, part, tiles);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

template <int T, int V>
static void launch_finish(const HeadArgs &a, const RowState &st, bool bwd, bool gram, int rows) {
	const dim3 grid((unsigned) ((rows + TPB / T - 1) / (TPB / T)));
	if (bwd && gram) hipLaunchKernelGGL((head_finish_kernel<T, V, true, true>), grid, dim3(TPB), 0, rt().stream, a, st, rows);
	else if (bwd) hipLaunchKernelGGL((head_finish_kernel<T, V, true, false>), grid, dim3(TPB), 0, rt().stream, a, st, rows);
	else if (gram) hipLaunchKernelGGL((head_finish_kernel<T, V, false, true>), grid, dim3(TPB), 0, rt().stream, a, st, rows);
	else hipLaunchKernelGGL((head_finish_kernel<T, V, false, false>), grid, dim3(TPB), 0, rt().stream, a, st, rows);
}

// the pass over the rows behind the products that give y
static int head_finish(const HeadArgs &a, const RowState &st, bool bwd, bool gram, int rows) {
	auto m4 = [](long v) { return v % 4 == 0; };
	const bool vec = m4(a.K) && m4(a.ldx) && m4(a.ldw) && (!bwd || m4(a.lddx)) && aligned16(a.x_re) && aligned16(a.x_im) && aligned16(a.w_re) &&
			aligned16(a.w_im) && aligned16(a.dx_re) && aligned16(a.dx_im) && aligned16(a.dxs_re) && aligned16(a.dxs_im);
	// a wavefront per row up to 512 columns (or what 128-bit accesses make of them), a workgroup beyond
	if (vec && a.K <= 512) launch_finish<64, 4>(a, st, bwd, gram, rows);
	else if (vec) launch_finish<256, 4>(a, st, bwd, gram, rows);
	else if (a.K <= 256) launch_finish<64, 1>(a, st, bwd, gram, rows);
	else launch_finish<256, 1>(a, st, bwd, gram, rows);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

static int head(const HeadArgs &proto, int B, float *dw_re, float *dw_im, float *dws_re, float *dws_im, long lddw, int accumulate_dw, bool bwd) {
	HeadArgs a = proto;
	a.B = B;
	const int K = a.K, N = a.N;
	if (!bwd && B <= SCORE_ROWS && (long) ((B + 15) / 16) * ((N + 15) / 16) > 4L * rt().prop.multiProcessorCount) return head_score(a, B);
	const HeadPlan plan = head_plan(B, K, N, bwd, a.argmax || !a.labels);
	const HeadPad pad = head_pad(a, B, plan);
	HeadBuffers b;
	int rc = head_buffers(pad, plan, K, b);
	if (rc) return rc;
	const int np = b.piece_cols, Kp = pad.K;  // Kp: K, or K filled up with zeros where the operands are copies
	const long ldk = b.ldk;
	if (pad.copy) {
		auto blocks = [&](int rows) { return (unsigned) (((long) rows * (ldk / 4) + TPB - 1) / TPB); };
		const PackArgs pk = {{a.x_re, a.w_re}, {a.x_im, a.w_im}, {a.ldx, a.ldw}, {b.x, b.w}, {B, N}, {pad.B, pad.N}, (int) blocks(pad.B), K, (int) ldk};
		hipLaunchKernelGGL(head_pack_kernel, dim3(blocks(pad.B) + blocks(pad.N), 2), dim3(TPB), 0, rt().stream, pk);
		CNET_LAUNCH_CHECK();
		a.x_re = b.x;
		a.x_im = b.x + (size_t) pad.B * ldk;
		a.w_re = b.w;
		a.w_im = b.w + (size_t) pad.N * ldk;
		a.ldx = a.ldw = ldk;
	}
	float *z_re = b.piece, *z_im = b.piece + (size_t) pad.B * np;
	float *y_re = b.y, *y_im = b.y + (size_t) pad.B * ldk;
	a.y_re = y_re;
	a.y_im = y_im;
	a.xs_re = b.xs;
	a.xs_im = b.xs + (size_t) pad.B * ldk;
	a.ldy = ldk;
	auto w_at = [&](const float *w, int n0) { return w + (size_t) n0 * a.ldw; };
	if (plan.whole) {
		rc = cnet_clinear_fwd(a.x_re, a.x_im, a.ldx, a.w_re, a.w_im, a.ldw, z_re, z_im, np, B, Kp, N, 0);
		if (rc) return rc;
		// a row of its own workgroup: many threads where the rows are long
		const dim3 grid((unsigned) (bwd ? pad.B : B));
		RowState st = b.st;
		if (!plan.label) st.c_re = st.c_im = nullptr;
		if (N > 4096) {
			if (bwd) hipLaunchKernelGGL((head_row_kernel<1024, true>), grid, dim3(1024), 0, rt().stream, a, st, z_re, z_im, (long) np);
			else hipLaunchKernelGGL((head_row_kernel<1024, false>), grid, dim3(1024), 0, rt().stream, a, st, z_re, z_im, (long) np);
		} else {
			if (bwd) hipLaunchKernelGGL((head_row_kernel<TPB, true>), grid, dim3(TPB), 0, rt().stream, a, st, z_re, z_im, (long) np);
			else hipLaunchKernelGGL((head_row_kernel<TPB, false>), grid, dim3(TPB), 0, rt().stream, a, st, z_re, z_im, (long) np);
		}
		CNET_LAUNCH_CHECK();
		if (!bwd) return CNET_OK;
		if (pad.B == B && !plan.label)  // both in one launch where they are small
			return clinear_bwd_sym(true, z_re, z_im, np, a.xs_re, a.xs_im, ldk, a.w_re, a.w_im, a.ldw, a.dx_re, a.dx_im, a.dxs_re, a.dxs_im, a.lddx,
					a.accumulate_dx, dw_re, dw_im, dws_re, dws_im, lddw, accumulate_dw, B, K, N);
		rc = cnet_clinear_bwd_input_sym(z_re, z_im, np, a.w_re, a.w_im, a.ldw, a.dx_re, a.dx_im, a.dxs_re, a.dxs_im, a.lddx, B, K, N,
				a.accumulate_dx || plan.label);
		if (rc) return rc;
		rc = cnet_clinear_bwd_weight_sym(z_re, z_im, np, a.xs_re, a.xs_im, ldk, dw_re, dw_im, dws_re, dws_im, lddw, pad.B, K, N, accumulate_dw);
		return rc || !plan.label ? rc : head_labels(a, b, B, dw_re, dw_im, dws_re, dws_im, lddw);
	}
	for (int n0 = 0; plan.pieces && n0 < N; n0 += np) {
		const int n = std::min(np, N - n0);
		rc = cnet_clinear_fwd(a.x_re, a.x_im, a.ldx, w_at(a.w_re, n0), w_at(a.w_im, n0), a.ldw, z_re, z_im, np, B, Kp, n, 0);
		if (rc) return rc;
		hipLaunchKernelGGL(head_piece_kernel, dim3((unsigned) B), dim3(TPB), 0, rt().stream, z_re, z_im, (long) np, n, n0, b.st);
		CNET_LAUNCH_CHECK();
		if (bwd && !plan.gram) {  // y += conj(z) w: linear in z, so the division by S can wait until S is whole
			rc = conj_product(0, B, K, n, z_re, z_im, np, w_at(a.w_re, n0), w_at(a.w_im, n0), a.ldw, y_re, y_im, ldk, n0 > 0);
			if (rc) return rc;
		}
	}
	if (plan.gram) {
		rc = gram64(K, N, a.w_re, a.w_im, a.ldw, nullptr, b.gram);
		if (rc) return rc;
		rc = times_gram(B, K, a.x_re, a.x_im, a.ldx, b.gram, GramOut{bwd ? y_re : nullptr, bwd ? y_im : nullptr, nullptr, nullptr, ldk, 0, b.st.part});
		if (rc) return rc;
	}
	rc = head_finish(a, b.st, bwd, plan.gram, bwd ? pad.B : B);
	if (rc) return rc;
	if (!bwd) return CNET_OK;
	if (plan.gram) {
		rc = gram64(K, B, a.x_re, a.x_im, a.ldx, b.st.weight, b.gram);
		if (rc) return rc;
		rc = times_gram(N, K, a.w_re, a.w_im, a.ldw, b.gram, GramOut{dw_re, dw_im, dws_re, dws_im, lddw, accumulate_dw, nullptr});
		if (rc) return rc;
	}
	for (int n0 = 0; !plan.gram && n0 < N; n0 += np) {  // the logits again, over sqrt(S) and zero where a row is left out
		const int n = std::min(np, N - n0);
		rc = cnet_clinear_fwd(a.xs_re, a.xs_im, ldk, w_at(a.w_re, n0), w_at(a.w_im, n0), a.ldw, z_re, z_im, np, pad.B, Kp, n, 0);
		if (rc) return rc;
		const size_t o = (size_t) n0 * lddw;
		rc = conj_product_pair(true, n, K, pad.B, z_re, z_im, np, a.xs_re, a.xs_im, ldk, dw_re + o, dw_im + o, dws_re ? dws_re + o : nullptr,
				dws_re ? dws_im + o : nullptr, lddw, accumulate_dw);
		if (rc) return rc;
	}
	return head_labels(a, b, B, dw_re, dw_im, dws_re, dws_im, lddw);
}

extern "C" {

int cnet_distill_fwd(const float *z_re, const float *z_im, int64_t ldz, const int32_t *ids, const float *probs, int top, float *s, float *loss,
		int rows, int cols) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 22) && cols > 0 && cols < (1 << 30) && top > 0 && top <= CNET_DISTILL_MAX_TOP);
	if (!rows) return CNET_OK;
	CNET_CHECK_ARG(z_re && z_im && ids && probs && s && loss && ldz >= cols);
	return distill(DistillArgs{z_re, z_im, (long) ldz, ids, probs, top, s, loss, nullptr, nullptr, nullptr, nullptr, 0, rows, cols});
}

int cnet_distill_bwd_sym(const float *z_re, const float *z_im, int64_t ldz, const float *s, const int32_t *ids, const float *probs, int top,
		float *dz_dz_re, float *dz_dz_im, float *dz_dzs_re, float *dz_dzs_im, int64_t lddz, int rows, int cols) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 22) && cols > 0 && cols < (1 << 30) && top > 0 && top <= CNET_DISTILL_MAX_TOP);
	if (!rows) return CNET_OK;
	CNET_CHECK_ARG(z_re && z_im && ids && probs && s && ldz >= cols);
	CNET_CHECK_ARG(dz_dz_re && dz_dz_im && ((dz_dzs_re == nullptr) == (dz_dzs_im == nullptr)) && lddz >= cols);
	return distill(DistillArgs{z_re, z_im, (long) ldz, ids, probs, top, const_cast<float *>(s), nullptr, dz_dz_re, dz_dz_im, dz_dzs_re,
			dz_dzs_im, (long) lddz, rows, cols});
}

int cnet_distill_fwd_bwd_sym(const float *z_re, const float *z_im, int64_t ldz, const int32_t *ids, const float *probs, int top, float *s, float *loss,
		float *dz_dz_re, float *dz_dz_im, float *dz_dzs_re, float *dz_dzs_im, int64_t lddz, int rows, int cols) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 22) && cols > 0 && cols < (1 << 30) && top > 0 && top <= CNET_DISTILL_MAX_TOP);
	if (!rows) return CNET_OK;
	CNET_CHECK_ARG(z_re && z_im && ids && probs && s && loss && ldz >= cols);
	CNET_CHECK_ARG(dz_dz_re && dz_dz_im && ((dz_dzs_re == nullptr) == (dz_dzs_im == nullptr)) && lddz >= cols);
	return distill(DistillArgs{z_re, z_im, (long) ldz, ids, probs, top, s, loss, dz_dz_re, dz_dz_im, dz_dzs_re, dz_dzs_im, (long) lddz, rows,
			cols});
}

int cnet_vocab_head_fwd(const float *x_re, const float *x_im, int64_t ldx, const float *w_re, const float *w_im, int64_t ldw, const int32_t *labels,
		float *s, float *loss, int32_t *argmax, int B, int K, int N) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(B >= 0 && B < (1 << 24) && K > 0 && K < (1 << 30) && N > 0 && N < (1 << 28));
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
	CNET_CHECK_ARG(B >= 0 && B < (1 << 24) && K > 0 && K < (1 << 30) && N > 0 && N < (1 << 28));
	CNET_CHECK_ARG(dw_dz_re && dw_dz_im && ((dw_dzs_re == nullptr) == (dw_dzs_im == nullptr)) && lddw >= K);
	if (!B) {
		if (accumulate_dw) return CNET_OK;
		for (float *p : {dw_dz_re, dw_dz_im, dw_dzs_re, dw_dzs_im})
			if (p) hipLaunchKernelGGL(head_clear_kernel, dim3((unsigned) std::min(N, 65535)), dim3(TPB), 0, rt().stream, p, (long) lddw, N, K);
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
