// Norms around a block of layers, with the weights, the residual path and the scale that go with them.
//
//   in front of a block   y = v .* n,            n = x s,   s = 1 / max(sqrt(mean |x|^2 + eps), 1e-15)   (one s per row)
//   behind it             h = u + scale v .* (f s1)         f: what the block computed, u: the residual path
//   and for the next one  y = w .* (h s2)
//
// Backward, for a conjugate gradient pair, all as dL/dz: with g = dL/dy and p = g v (= dL/dn),
//   dx = s (p - conj(n) t),  t = mean Re(p n),     dv = g n  (summed over the rows when they share v);
// where the clamp holds, s does not depend on x, and t is zero.
// the join adds what the next norm hands back to the gradient of h, dh = gh + back(g), gives it to u as it is, and goes on with
// f under the gradient scale dh.
#include "common.hpp"
#include "rows.hpp"

#include <algorithm>
#include <cmath>

namespace {

using namespace cnet::rows;

constexpr int TPB = 256;

struct Planes {
	const float *re, *im;
	long ld;
};
struct Out4 {
	float *re, *im, *sre, *sim;  // dz and, where wanted, dz*
	long ld;
};

struct FwdArgs {
	Planes x, v, u, w;  // x: the operand of the (first) norm; v, w: ld == 0 for one row shared by all; u: the residual path
	float *y_re, *y_im, *h_re, *h_im;
	long ldy, ldh;
	float *s, *s2;
	float scale, eps;
	double inv_cols;
	int rows, cols;
};

struct BwdArgs {
	Planes x, v, h, w, g, gh;  // x: the operand of the (first) norm; gh: dL/d its result along the residual path; h, w, g = dL/dy: the next norm's
	const float *s, *s2;
	Out4 du, dx, dv;   // dv: only with a gate of its own for every row (the shared one goes through `partial`)
	float *partial;    // [slab][planes][cols]: dv re, im (unless every row has a gate of its own), dw re, im
	int planes, rows_per_slab;
	float scale;
	int rows, cols, accumulate, accumulate_w;
};

// |z|^2 added to a sum in double: a square of single precision leaves its range at 1.8e19, and a finite row would come out as zeros
__device__ __forceinline__ double add_power(double sum, float re, float im) {
	return fma((double) im, (double) im, fma((double) re, (double) re, sum));
}

constexpr float LEAST = 1.0e-15f;  // of a row's rms
// whether this s is the clamp's, and so the same for every x nearby
__device__ __forceinline__ bool at_clamp(float s) { return s >= 1.0f / LEAST; }

// (the clamp lets a NaN through, which fmaxf would not: the whole row is then NaN)
__device__ __forceinline__ float inv_rms(double sum, double inv_cols, float eps) {
	const double mean = sum * inv_cols + (double) eps;
	if (!(mean < 1.0e37)) return (float) (1.0 / sqrt(mean));  // beyond single precision: few rows ever, so the long way
	const float rms = sqrtf((float) mean);
	return 1.0f / (rms <= LEAST ? LEAST : rms);
}

__device__ __forceinline__ void put(float *p, float v, int accumulate) { *p = accumulate ? *p + v : v; }

// V consecutive columns from c on (V = 4: the row is a multiple of four).  A thread beyond the row's end gets the row's last columns:
// the load has no branch around it, behind which everything already on its way would have to be waited for (16384 x 128 backward:
// 58 us so, 32 without), and whoever uses the values for a sum masks them there, when they have arrived.
template <int V>
__device__ __forceinline__ void load_cols(float *v, const float *p, int c, int cols, int policy = 0) {
	const int at = min(c, cols - V);
	if (V == 4) {
		const float4 x = ld4(p + at, policy);
		v[0] = x.x;
		v[1 % V] = x.y;
		v[2 % V] = x.z;
		v[3 % V] = x.w;
	} else {
		v[0] = p[at];
	}
}
template <int V>
__device__ __forceinline__ void store_cols(float *p, const float *v, int c, int cols, int accumulate, int policy) {
	if (c >= cols) return;
	if (V == 4) {
		float4 x = make_float4(v[0], v[1 % V], v[2 % V], v[3 % V]);
		if (accumulate) {
			const float4 o = *reinterpret_cast<const float4 *>(p + c);
			x.x += o.x, x.y += o.y, x.z += o.z, x.w += o.w;
		}
		st4(p + c, x, policy);
	} else {
		put(p + c, v[0], accumulate);
	}
}
// a gradient (dz) into its planes, and its conjugate where the dz* half is wanted
template <int V>
__device__ __forceinline__ void store_grad(const Out4 &o, long row, float *re, float *im, int c, int cols, int accumulate, int policy) {
	const long at = row * o.ld;
	store_cols<V>(o.re + at, re, c, cols, accumulate, policy);
	store_cols<V>(o.im + at, im, c, cols, accumulate, policy);
	if (o.sre) {
#pragma unroll
		for (int k = 0; k < V; ++k) im[k] = -im[k];
		store_cols<V>(o.sre + at, re, c, cols, accumulate, policy);
		store_cols<V>(o.sim + at, im, c, cols, accumulate, policy);
	}
}

// T threads hold a row in registers, V x NIT columns each: every operand is read once and every result written once.  T = 64: four
// rows to a workgroup of 256.  Bound by memory: the join at 8192 x 1024 moves 268 MB in 52 us, 5.2 TB/s (a copy of 1 GiB: 5.1); one
// row of 1024 is a launch, 4.5 us.
template <int T, int NIT, int V, bool JOIN>
__global__ __launch_bounds__(T < TPB ? TPB : T) void norm_fwd_kernel(const FwdArgs a, const int policy) {
	constexpr int G = T / 64, ROWS = T < TPB ? TPB / T : 1;
	__shared__ double lds[ROWS * G];
	const int slot = threadIdx.x / T, t = threadIdx.x % T, lane = threadIdx.x & 63, wave = t >> 6;
	const bool live = (long) blockIdx.x * ROWS + slot < a.rows;
	const long row = live ? (long) blockIdx.x * ROWS + slot : a.rows - 1;
	float x_r[NIT][V], x_i[NIT][V], u_r[NIT][V], u_i[NIT][V];
#pragma unroll
	for (int k = 0; k < NIT; ++k) {
		const int c = (k * T + t) * V;
		load_cols<V>(x_r[k], a.x.re + row * a.x.ld, c, a.cols, policy);
		load_cols<V>(x_i[k], a.x.im + row * a.x.ld, c, a.cols, policy);
	}
	if (JOIN) {
#pragma unroll
		for (int k = 0; k < NIT; ++k) {
			const int c = (k * T + t) * V;
			load_cols<V>(u_r[k], a.u.re + row * a.u.ld, c, a.cols, policy);
			load_cols<V>(u_i[k], a.u.im + row * a.u.ld, c, a.cols, policy);
		}
	}
	double sum = 0.0;
#pragma unroll
	for (int k = 0; k < NIT; ++k) {
		const bool in = (k * T + t) * V < a.cols;
#pragma unroll
		for (int q = 0; q < V; ++q) sum = in ? add_power(sum, x_r[k][q], x_i[k][q]) : sum;
	}
	sum = group_reduce<double, G>(sum, SumD(), lds, slot, wave, lane);
	const float s = inv_rms(sum, a.inv_cols, a.eps);
	if (t == 0 && live && a.s) a.s[row] = s;
	double sum2 = 0.0;
#pragma unroll
	for (int k = 0; k < NIT; ++k) {
		const int c = (k * T + t) * V;
		float v_r[V], v_i[V];
		load_cols<V>(v_r, a.v.re + row * a.v.ld, c, a.cols);
		load_cols<V>(v_i, a.v.im + row * a.v.ld, c, a.cols);
#pragma unroll
		for (int q = 0; q < V; ++q) {
			const float n_r = x_r[k][q] * s, n_i = x_i[k][q] * s;
			float y_r = v_r[q] * n_r - v_i[q] * n_i, y_i = v_r[q] * n_i + v_i[q] * n_r;
			if (JOIN) {
				y_r = u_r[k][q] + a.scale * y_r;
				y_i = u_i[k][q] + a.scale * y_i;
				sum2 = c < a.cols ? add_power(sum2, y_r, y_i) : sum2;
			}
			x_r[k][q] = y_r;
			x_i[k][q] = y_i;
		}
		if (live) {
			store_cols<V>((JOIN ? a.h_re + row * a.ldh : a.y_re + row * a.ldy), x_r[k], c, a.cols, 0, policy);
			store_cols<V>((JOIN ? a.h_im + row * a.ldh : a.y_im + row * a.ldy), x_i[k], c, a.cols, 0, policy);
		}
	}
	if (!JOIN || !a.y_re) return;
	sum2 = group_reduce<double, G>(sum2, SumD(), lds, slot, wave, lane);
	const float s2 = inv_rms(sum2, a.inv_cols, a.eps);
	if (!live) return;
	if (t == 0 && a.s2) a.s2[row] = s2;
#pragma unroll
	for (int k = 0; k < NIT; ++k) {
		const int c = (k * T + t) * V;
		float w_r[V], w_i[V], y_r[V], y_i[V];
		load_cols<V>(w_r, a.w.re, c, a.cols);
		load_cols<V>(w_i, a.w.im, c, a.cols);
#pragma unroll
		for (int q = 0; q < V; ++q) {
			const float n_r = x_r[k][q] * s2, n_i = x_i[k][q] * s2;
			y_r[q] = w_r[q] * n_r - w_i[q] * n_i;
			y_i[q] = w_r[q] * n_i + w_i[q] * n_r;
		}
		store_cols<V>(a.y_re + row * a.ldy, y_r, c, a.cols, 0, policy);
		store_cols<V>(a.y_im + row * a.ldy, y_i, c, a.cols, 0, policy);
	}
}

struct Sum3 {
	float a, b, c;
};
struct Sum3Op {
	__device__ Sum3 operator()(Sum3 x, Sum3 y) const { return Sum3{x.a + y.a, x.b + y.b, x.c + y.c}; }
};

// T threads hold one row at a time, V x NIT columns each; R groups of T threads walk the workgroup's rows in turn (group r takes row
// r, r + R, ..) and keep their columns' sums of dv and dw in registers, which meet in LDS in group order at the end.
// One exchange per row: with e = gh + s2 p (p = g w) and z = v n1, t2 = mean Re(p n2) and the mean of Re(dh z), which is
// Re(e z) - s2 t2 Re(conj(n2) z), come from three sums that do not wait for each other.
// SECOND: the next block's norm takes part (the join with a gradient at y).
// KEEP: the weights stay in registers, and the next row's operands are requested before the exchange of this one.
// Bound by memory: the join at 8192 x 1024 moves 403 MB in 81 us, 5.0 TB/s, 5 us of it norm_sum_kernel (one exchange after the other,
// with the rows read twice, took 255 us); 515 x 1001 with a gate per row, 25 MB, 6.5 us.
template <int T, int NIT, int V, bool SECOND, bool KEEP>
__global__ __launch_bounds__(T < TPB ? TPB : T) void norm_bwd_kernel(const BwdArgs a, const int policy) {
	constexpr int G = T / 64, R = T < TPB ? TPB / T : 1, NP = SECOND ? 4 : 2;
	__shared__ Sum3 lds[R * G];
	extern __shared__ __align__(16) float sums[];  // [R - 1][NP][NIT][T][V]
	const int group = threadIdx.x / T, t = threadIdx.x % T, lane = threadIdx.x & 63, wave = t >> 6;
	const int r0 = blockIdx.x * a.rows_per_slab, r1 = min(a.rows, r0 + a.rows_per_slab);
	const bool shared = a.v.ld == 0;
	const float inv_n = 1.0f / (float) a.cols;
	float acc[NP][NIT][V];
#pragma unroll
	for (int p = 0; p < NP; ++p)
#pragma unroll
		for (int k = 0; k < NIT; ++k)
#pragma unroll
			for (int q = 0; q < V; ++q) acc[p][k][q] = 0.f;
	float x_r[NIT][V], x_i[NIT][V], e_r[NIT][V], e_i[NIT][V], h_r[NIT][V], h_i[NIT][V], g_r[NIT][V], g_i[NIT][V];
	float v_r[NIT][V], v_i[NIT][V], w_r[NIT][V], w_i[NIT][V];
	float s, s2;
	auto fetch_gate = [&](long row) {
#pragma unroll
		for (int k = 0; k < NIT; ++k) {
			load_cols<V>(v_r[k], a.v.re + row * a.v.ld, (k * T + t) * V, a.cols);
			load_cols<V>(v_i[k], a.v.im + row * a.v.ld, (k * T + t) * V, a.cols);
		}
	};
	auto fetch = [&](long row) {
		s = a.s[row];
		s2 = SECOND ? a.s2[row] : 0.f;
#pragma unroll
		for (int k = 0; k < NIT; ++k) {
			const int c = (k * T + t) * V;
			load_cols<V>(x_r[k], a.x.re + row * a.x.ld, c, a.cols, policy);
			load_cols<V>(x_i[k], a.x.im + row * a.x.ld, c, a.cols, policy);
			if (a.gh.re) {
				load_cols<V>(e_r[k], a.gh.re + row * a.gh.ld, c, a.cols, policy);
				load_cols<V>(e_i[k], a.gh.im + row * a.gh.ld, c, a.cols, policy);
			} else {
#pragma unroll
				for (int q = 0; q < V; ++q) e_r[k][q] = e_i[k][q] = 0.f;
			}
			if (SECOND) {
				load_cols<V>(h_r[k], a.h.re + row * a.h.ld, c, a.cols, policy);
				load_cols<V>(h_i[k], a.h.im + row * a.h.ld, c, a.cols, policy);
				load_cols<V>(g_r[k], a.g.re + row * a.g.ld, c, a.cols, policy);
				load_cols<V>(g_i[k], a.g.im + row * a.g.ld, c, a.cols, policy);
			}
		}
	};
	auto fetch_weights = [&]() {
#pragma unroll
		for (int k = 0; k < NIT; ++k) {
			load_cols<V>(w_r[k], a.w.re, (k * T + t) * V, a.cols);
			load_cols<V>(w_i[k], a.w.im, (k * T + t) * V, a.cols);
		}
	};
	if (SECOND && KEEP) fetch_weights();
	if (shared && KEEP) fetch_gate(0);
	if (KEEP) fetch(min(r0 + group, r1 - 1));
	// (every group makes the same number of rounds: the exchange is the whole workgroup's; a round beyond the rows stores nothing)
	for (int base = r0; base < r1; base += R) {
		const bool live = base + group < r1;
		const long row = live ? base + group : r1 - 1;
		if (!KEEP) fetch(row);
		if (!shared || !KEEP) fetch_gate(row);
		if (SECOND && !KEEP) fetch_weights();
		Sum3 m = {0.f, 0.f, 0.f};
		// what the row's second half needs, out of the way of the next row's operands: n1, e, n2, g
		float n_r[NIT][V], n_i[NIT][V], f_r[NIT][V], f_i[NIT][V], k_r[NIT][V], k_i[NIT][V], y_r[NIT][V], y_i[NIT][V];
		const float s_row = s;
#pragma unroll
		for (int k = 0; k < NIT; ++k) {
			const bool in = (k * T + t) * V < a.cols;  // (beyond the row n1 and n2 are zero, and with them every sum)
#pragma unroll
			for (int q = 0; q < V; ++q) {
				n_r[k][q] = in ? x_r[k][q] * s : 0.f;
				n_i[k][q] = in ? x_i[k][q] * s : 0.f;
				f_r[k][q] = e_r[k][q];
				f_i[k][q] = e_i[k][q];
				const float z_r = v_r[k][q] * n_r[k][q] - v_i[k][q] * n_i[k][q], z_i = v_r[k][q] * n_i[k][q] + v_i[k][q] * n_r[k][q];
				if (SECOND) {
					y_r[k][q] = g_r[k][q];
					y_i[k][q] = g_i[k][q];
					k_r[k][q] = in ? h_r[k][q] * s2 : 0.f;
					k_i[k][q] = in ? h_i[k][q] * s2 : 0.f;
					const float p_r = y_r[k][q] * w_r[k][q] - y_i[k][q] * w_i[k][q], p_i = y_r[k][q] * w_i[k][q] + y_i[k][q] * w_r[k][q];
					m.b += p_r * k_r[k][q] - p_i * k_i[k][q];
					m.c += k_r[k][q] * z_r + k_i[k][q] * z_i;
					f_r[k][q] += s2 * p_r;
					f_i[k][q] += s2 * p_i;
				}
				m.a += f_r[k][q] * z_r - f_i[k][q] * z_i;
			}
		}
		const float s2_row = s2;
		if (KEEP && base + R < r1) fetch(min(base + R + group, r1 - 1));
		m = group_reduce<Sum3, G>(m, Sum3Op(), lds, group, wave, lane);
		const float t2 = at_clamp(s2_row) ? 0.f : m.b * inv_n * s2_row, t1 = at_clamp(s_row) ? 0.f : a.scale * (m.a - t2 * m.c) * inv_n;
		if (!live) continue;
#pragma unroll
		for (int k = 0; k < NIT; ++k) {
			const int c = (k * T + t) * V;
			float o_r[V], o_i[V], d_r[V], d_i[V];
#pragma unroll
			for (int q = 0; q < V; ++q) {
				d_r[q] = f_r[k][q];
				d_i[q] = f_i[k][q];
				if (SECOND) {
					d_r[q] -= k_r[k][q] * t2;
					d_i[q] += k_i[k][q] * t2;
				}
				f_r[k][q] = a.scale * d_r[q];
				f_i[k][q] = a.scale * d_i[q];
				o_r[q] = s_row * (f_r[k][q] * v_r[k][q] - f_i[k][q] * v_i[k][q] - n_r[k][q] * t1);
				o_i[q] = s_row * (f_r[k][q] * v_i[k][q] + f_i[k][q] * v_r[k][q] + n_i[k][q] * t1);
			}
			if (a.du.re) store_grad<V>(a.du, row, d_r, d_i, c, a.cols, a.accumulate, policy);
			store_grad<V>(a.dx, row, o_r, o_i, c, a.cols, a.accumulate, policy);
#pragma unroll
			for (int q = 0; q < V; ++q) {
				d_r[q] = f_r[k][q] * n_r[k][q] - f_i[k][q] * n_i[k][q];
				d_i[q] = f_r[k][q] * n_i[k][q] + f_i[k][q] * n_r[k][q];
				acc[0][k][q] += d_r[q];
				acc[1][k][q] += d_i[q];
				if (SECOND) {
					acc[2 % NP][k][q] += y_r[k][q] * k_r[k][q] - y_i[k][q] * k_i[k][q];
					acc[3 % NP][k][q] += y_r[k][q] * k_i[k][q] + y_i[k][q] * k_r[k][q];
				}
			}
			if (!shared) store_grad<V>(a.dv, row, d_r, d_i, c, a.cols, a.accumulate_w, policy);
		}
	}
	if (!a.planes) return;
	if (R > 1 && group > 0) {
#pragma unroll
		for (int p = 0; p < NP; ++p)
#pragma unroll
			for (int k = 0; k < NIT; ++k) store_cols<V>(sums + (((group - 1) * NP + p) * NIT + k) * (T * V) + t * V, acc[p][k], 0, V, 0, 0);
	}
	if (R > 1) __syncthreads();
	if (group > 0) return;
	float *part = a.partial + (long) blockIdx.x * a.planes * a.cols;
#pragma unroll
	for (int p = 0; p < NP; ++p) {
		if (p < 2 && !shared) continue;
#pragma unroll
		for (int k = 0; k < NIT; ++k) {
			const int c = (k * T + t) * V;
			for (int r = 1; r < R; ++r) {
				float more[V];
				load_cols<V>(more, sums + (((r - 1) * NP + p) * NIT + k) * (T * V) + t * V, 0, V);
#pragma unroll
				for (int q = 0; q < V; ++q) acc[p][k][q] += more[q];
			}
			float *dst = part + (long) (shared ? p : p - 2) * a.cols;
#pragma unroll
			for (int q = 0; q < V; ++q)
				if (c + q < a.cols) dst[c + q] = acc[p][k][q];
		}
	}
}

// Rows whose operands do not fit in registers, up to T x V x NIT columns: the same sums, then the operands once more (from the caches:
// a row of 8192 columns is half a megabyte), of which a thread keeps only its columns' sums over the rows.  The join at 1024 x 8192:
// 121 us, and 15 for the sum over the slabs; norm_bwd_wide_kernel takes 172 (8191 columns: 172 both, 4999: 73 against 96).
template <int T, int NIT, int V, bool SECOND>
__global__ __launch_bounds__(T) void norm_bwd_twice_kernel(const BwdArgs a) {
	constexpr int G = T / 64, NP = SECOND ? 4 : 2;
	__shared__ Sum3 lds[G];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const int r0 = blockIdx.x * a.rows_per_slab, r1 = min(a.rows, r0 + a.rows_per_slab);
	const bool shared = a.v.ld == 0;
	float acc[NP][NIT][V];
#pragma unroll
	for (int p = 0; p < NP; ++p)
#pragma unroll
		for (int k = 0; k < NIT; ++k)
#pragma unroll
			for (int q = 0; q < V; ++q) acc[p][k][q] = 0.f;
	for (long row = r0; row < r1; ++row) {
		const float s = a.s[row], s2 = SECOND ? a.s2[row] : 0.f;
		float n_r[V], n_i[V], f_r[V], f_i[V], v_r[V], v_i[V], k_r[V], k_i[V], y_r[V], y_i[V], p_r[V], p_i[V];
		// one thread's columns from c on: n1, e without its share of t2, v and, SECOND, n2, g and p
		auto fetch = [&](int c) {
			load_cols<V>(n_r, a.x.re + row * a.x.ld, c, a.cols);
			load_cols<V>(n_i, a.x.im + row * a.x.ld, c, a.cols);
			load_cols<V>(v_r, a.v.re + row * a.v.ld, c, a.cols);
			load_cols<V>(v_i, a.v.im + row * a.v.ld, c, a.cols);
#pragma unroll
			for (int q = 0; q < V; ++q) f_r[q] = f_i[q] = 0.f;
			if (a.gh.re) {
				load_cols<V>(f_r, a.gh.re + row * a.gh.ld, c, a.cols);
				load_cols<V>(f_i, a.gh.im + row * a.gh.ld, c, a.cols);
			}
			if (SECOND) {
				load_cols<V>(k_r, a.h.re + row * a.h.ld, c, a.cols);
				load_cols<V>(k_i, a.h.im + row * a.h.ld, c, a.cols);
				load_cols<V>(y_r, a.g.re + row * a.g.ld, c, a.cols);
				load_cols<V>(y_i, a.g.im + row * a.g.ld, c, a.cols);
				load_cols<V>(p_r, a.w.re, c, a.cols);
				load_cols<V>(p_i, a.w.im, c, a.cols);
			}
#pragma unroll
			for (int q = 0; q < V; ++q) {
				n_r[q] = c < a.cols ? n_r[q] * s : 0.f;
				n_i[q] = c < a.cols ? n_i[q] * s : 0.f;
				if (SECOND) {
					k_r[q] = c < a.cols ? k_r[q] * s2 : 0.f;
					k_i[q] = c < a.cols ? k_i[q] * s2 : 0.f;
					const float w_r = p_r[q], w_i = p_i[q];
					p_r[q] = y_r[q] * w_r - y_i[q] * w_i;
					p_i[q] = y_r[q] * w_i + y_i[q] * w_r;
					f_r[q] += s2 * p_r[q];
					f_i[q] += s2 * p_i[q];
				}
			}
		};
		Sum3 m = {0.f, 0.f, 0.f};
#pragma unroll 1
		for (int k = 0; k < NIT; ++k) {
			if (k * T * V >= a.cols) break;
			fetch((k * T + t) * V);
#pragma unroll
			for (int q = 0; q < V; ++q) {
				const float z_r = v_r[q] * n_r[q] - v_i[q] * n_i[q], z_i = v_r[q] * n_i[q] + v_i[q] * n_r[q];
				if (SECOND) {
					m.b += p_r[q] * k_r[q] - p_i[q] * k_i[q];
					m.c += k_r[q] * z_r + k_i[q] * z_i;
				}
				m.a += f_r[q] * z_r - f_i[q] * z_i;
			}
		}
		m = group_reduce<Sum3, G>(m, Sum3Op(), lds, 0, wave, lane);
		const float inv_n = 1.0f / (float) a.cols, t2 = at_clamp(s2) ? 0.f : m.b * inv_n * s2;
		const float t1 = at_clamp(s) ? 0.f : a.scale * (m.a - t2 * m.c) * inv_n;
#pragma unroll
		for (int k = 0; k < NIT; ++k) {
			if (k * T * V >= a.cols) break;
			const int c = (k * T + t) * V;
			fetch(c);
			float o_r[V], o_i[V], d_r[V], d_i[V];
#pragma unroll
			for (int q = 0; q < V; ++q) {
				d_r[q] = f_r[q];
				d_i[q] = f_i[q];
				if (SECOND) {
					d_r[q] -= k_r[q] * t2;
					d_i[q] += k_i[q] * t2;
					acc[2 % NP][k][q] += y_r[q] * k_r[q] - y_i[q] * k_i[q];
					acc[3 % NP][k][q] += y_r[q] * k_i[q] + y_i[q] * k_r[q];
				}
				f_r[q] = a.scale * d_r[q];
				f_i[q] = a.scale * d_i[q];
				o_r[q] = s * (f_r[q] * v_r[q] - f_i[q] * v_i[q] - n_r[q] * t1);
				o_i[q] = s * (f_r[q] * v_i[q] + f_i[q] * v_r[q] + n_i[q] * t1);
			}
			if (a.du.re) store_grad<V>(a.du, row, d_r, d_i, c, a.cols, a.accumulate, 0);
			store_grad<V>(a.dx, row, o_r, o_i, c, a.cols, a.accumulate, 0);
#pragma unroll
			for (int q = 0; q < V; ++q) {
				d_r[q] = f_r[q] * n_r[q] - f_i[q] * n_i[q];
				d_i[q] = f_r[q] * n_i[q] + f_i[q] * n_r[q];
				acc[0][k][q] += d_r[q];
				acc[1][k][q] += d_i[q];
			}
			if (!shared) store_grad<V>(a.dv, row, d_r, d_i, c, a.cols, a.accumulate_w, 0);
		}
	}
	if (!a.planes) return;
	float *part = a.partial + (long) blockIdx.x * a.planes * a.cols;
#pragma unroll
	for (int p = 0; p < NP; ++p) {
		if (p < 2 && !shared) continue;
#pragma unroll
		for (int k = 0; k < NIT; ++k)
#pragma unroll
			for (int q = 0; q < V; ++q) {
				const int c = (k * T + t) * V + q;
				if (c < a.cols) part[(long) (shared ? p : p - 2) * a.cols + c] = acc[p][k][q];
			}
	}
}

constexpr int WIDE = 1024;  // threads of the two kernels for wide rows

// Rows wider than the kernels above hold in registers: one workgroup per row, which walks it once per stage.  400 x 20000: 60 us,
// 4.3 TB/s (105 with 256 threads).
template <bool JOIN>
__global__ __launch_bounds__(WIDE) void norm_fwd_wide_kernel(const FwdArgs a) {
	__shared__ double lds[WIDE / 64];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const long row = blockIdx.x;
	const float *xr = a.x.re + row * a.x.ld, *xi = a.x.im + row * a.x.ld;
	const float *vr = a.v.re + row * a.v.ld, *vi = a.v.im + row * a.v.ld;
	double sum = 0.0;
	for (int c = t; c < a.cols; c += WIDE) sum = add_power(sum, xr[c], xi[c]);
	sum = group_reduce<double, WIDE / 64>(sum, SumD(), lds, 0, wave, lane);
	const float s = inv_rms(sum, a.inv_cols, a.eps);
	if (t == 0 && a.s) a.s[row] = s;
	if (!JOIN) {
		for (int c = t; c < a.cols; c += WIDE) {
			const float n_r = xr[c] * s, n_i = xi[c] * s;
			a.y_re[row * a.ldy + c] = vr[c] * n_r - vi[c] * n_i;
			a.y_im[row * a.ldy + c] = vr[c] * n_i + vi[c] * n_r;
		}
		return;
	}
	double sum2 = 0.0;
	for (int c = t; c < a.cols; c += WIDE) {
		const float n_r = xr[c] * s, n_i = xi[c] * s;
		const float h_r = a.u.re[row * a.u.ld + c] + a.scale * (vr[c] * n_r - vi[c] * n_i);
		const float h_i = a.u.im[row * a.u.ld + c] + a.scale * (vr[c] * n_i + vi[c] * n_r);
		a.h_re[row * a.ldh + c] = h_r;
		a.h_im[row * a.ldh + c] = h_i;
		sum2 = add_power(sum2, h_r, h_i);
	}
	if (!a.y_re) return;
	sum2 = group_reduce<double, WIDE / 64>(sum2, SumD(), lds, 0, wave, lane);
	const float s2 = inv_rms(sum2, a.inv_cols, a.eps);
	if (t == 0 && a.s2) a.s2[row] = s2;
	const float *wr = a.w.re + row * a.w.ld, *wi = a.w.im + row * a.w.ld;
	for (int c = t; c < a.cols; c += WIDE) {
		const float n_r = a.h_re[row * a.ldh + c] * s2, n_i = a.h_im[row * a.ldh + c] * s2;
		a.y_re[row * a.ldy + c] = wr[c] * n_r - wi[c] * n_i;
		a.y_im[row * a.ldy + c] = wr[c] * n_i + wi[c] * n_r;
	}
}

// The same for rows too wide for registers.  A workgroup takes `rows_per_slab` rows one after the other; its columns' sums of dv and dw
// stay in its own rows of `partial` (each thread always meets the same columns: no atomics, one order), which norm_sum_kernel adds
// in slab order.  512 x 16384: 200 us (552 with 256 threads), and 31 for the sum.
template <bool SECOND>
__global__ __launch_bounds__(WIDE) void norm_bwd_wide_kernel(const BwdArgs a) {
	__shared__ float lds[WIDE / 64];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const int r0 = blockIdx.x * a.rows_per_slab, r1 = min(a.rows, r0 + a.rows_per_slab);
	const bool shared = a.v.ld == 0;
	const float inv_n = 1.0f / (float) a.cols;
	float *part = a.partial + (long) blockIdx.x * a.planes * a.cols;
	for (long row = r0; row < r1; ++row) {
		const float s = a.s[row], s2 = SECOND ? a.s2[row] : 0.f;
		// the gradient that the next norm hands back to h at one column, before its share of t2
		auto next = [&](int c, float &p_r, float &p_i, float &n_r, float &n_i) {
			const float g_r = a.g.re[row * a.g.ld + c], g_i = a.g.im[row * a.g.ld + c];
			const float w_r = a.w.re[row * a.w.ld + c], w_i = a.w.im[row * a.w.ld + c];
			p_r = g_r * w_r - g_i * w_i;
			p_i = g_r * w_i + g_i * w_r;
			n_r = a.h.re[row * a.h.ld + c] * s2;
			n_i = a.h.im[row * a.h.ld + c] * s2;
		};
		float t2 = 0.f;
		if (SECOND) {
			for (int c = t; c < a.cols; c += WIDE) {
				float p_r, p_i, n_r, n_i;
				next(c, p_r, p_i, n_r, n_i);
				t2 += p_r * n_r - p_i * n_i;
			}
			t2 = group_reduce<float, WIDE / 64>(t2, SumF(), lds, 0, wave, lane) * inv_n;
			if (at_clamp(s2)) t2 = 0.f;
		}
		// the gradient at the result of the (first) norm and its weights: scale dh, or g
		auto at = [&](int c, float &d_r, float &d_i) {
			d_r = a.gh.re ? a.gh.re[row * a.gh.ld + c] : 0.f;
			d_i = a.gh.re ? a.gh.im[row * a.gh.ld + c] : 0.f;
			if (SECOND) {
				float p_r, p_i, n_r, n_i;
				next(c, p_r, p_i, n_r, n_i);
				d_r += s2 * (p_r - n_r * t2);
				d_i += s2 * (p_i + n_i * t2);
			}
		};
		const float k = a.scale;
		float t1 = 0.f;
		for (int c = t; c < a.cols; c += WIDE) {
			float d_r, d_i;
			at(c, d_r, d_i);
			d_r *= k;
			d_i *= k;
			const float v_r = a.v.re[row * a.v.ld + c], v_i = a.v.im[row * a.v.ld + c];
			const float n_r = a.x.re[row * a.x.ld + c] * s, n_i = a.x.im[row * a.x.ld + c] * s;
			t1 += (d_r * v_r - d_i * v_i) * n_r - (d_r * v_i + d_i * v_r) * n_i;
		}
		t1 = group_reduce<float, WIDE / 64>(t1, SumF(), lds, 0, wave, lane) * inv_n;
		if (at_clamp(s)) t1 = 0.f;
		for (int c = t; c < a.cols; c += WIDE) {
			float d_r, d_i;
			at(c, d_r, d_i);
			if (a.du.re) {
				const long o = row * a.du.ld + c;
				put(a.du.re + o, d_r, a.accumulate);
				put(a.du.im + o, d_i, a.accumulate);
				if (a.du.sre) {
					put(a.du.sre + o, d_r, a.accumulate);
					put(a.du.sim + o, -d_i, a.accumulate);
				}
			}
			d_r *= k;
			d_i *= k;
			const float v_r = a.v.re[row * a.v.ld + c], v_i = a.v.im[row * a.v.ld + c];
			const float n_r = a.x.re[row * a.x.ld + c] * s, n_i = a.x.im[row * a.x.ld + c] * s;
			const float o_r = s * (d_r * v_r - d_i * v_i - n_r * t1), o_i = s * (d_r * v_i + d_i * v_r + n_i * t1);
			const long o = row * a.dx.ld + c;
			put(a.dx.re + o, o_r, a.accumulate);
			put(a.dx.im + o, o_i, a.accumulate);
			if (a.dx.sre) {
				put(a.dx.sre + o, o_r, a.accumulate);
				put(a.dx.sim + o, -o_i, a.accumulate);
			}
			const float e_r = d_r * n_r - d_i * n_i, e_i = d_r * n_i + d_i * n_r;
			float *pw = part + c;
			if (shared) {
				put(pw, e_r, row > r0);
				put(pw + a.cols, e_i, row > r0);
				pw += 2 * a.cols;
			} else {
				const long ov = row * a.dv.ld + c;
				put(a.dv.re + ov, e_r, a.accumulate_w);
				put(a.dv.im + ov, e_i, a.accumulate_w);
				if (a.dv.sre) {
					put(a.dv.sre + ov, e_r, a.accumulate_w);
					put(a.dv.sim + ov, -e_i, a.accumulate_w);
				}
			}
			if (SECOND) {
				float p_r, p_i, m_r, m_i;
				next(c, p_r, p_i, m_r, m_i);
				const float g_r = a.g.re[row * a.g.ld + c], g_i = a.g.im[row * a.g.ld + c];
				put(pw, g_r * m_r - g_i * m_i, row > r0);
				put(pw + a.cols, g_r * m_i + g_i * m_r, row > r0);
			}
		}
	}
}

// dst[plane][c] (+)= sum over slabs; plane 0, 1: `first`, 2, 3: `second`.  COLS (plane, column) pairs per workgroup x LANES lanes that
// each add one contiguous part of the slabs in order; the lanes' sums are added in lane order.  512 slabs of 4096 sums: 5 us, a launch.
template <int LANES, int COLS>
__global__ __launch_bounds__(LANES * COLS) void norm_sum_kernel(const float *__restrict__ partial, int nslabs, int planes, int cols, Out4 first,
		Out4 second, int accumulate) {
	__shared__ float red[LANES][COLS];
	const int tx = threadIdx.x % COLS, ty = threadIdx.x / COLS;
	const long idx = (long) blockIdx.x * COLS + tx;
	const bool live = idx < (long) planes * cols;
	const int per = (nslabs + LANES - 1) / LANES, k0 = min(nslabs, ty * per), k1 = min(nslabs, k0 + per);
	red[ty][tx] = live ? cnet::ordered_sum(partial + (long) k0 * planes * cols + idx, (long) planes * cols, k1 - k0) : 0.f;
	__syncthreads();
	if (ty || !live) return;
	const int p = (int) (idx / cols), c = (int) (idx - (long) p * cols);
	float sum = red[0][tx];
#pragma unroll 8
	for (int l = 1; l < LANES; ++l) sum += red[l][tx];
	const Out4 &o = p < 2 ? first : second;
	put((p & 1 ? o.im : o.re) + c, sum, accumulate);
	if (o.sre) put((p & 1 ? o.sim : o.sre) + c, p & 1 ? -sum : sum, accumulate);
}

}  // namespace

using namespace cnet;

// (no slabs: the sum over no rows, zero)
static int norm_sum(const float *partial, int nslabs, int planes, int cols, const Out4 &first, const Out4 &second, int accumulate) {
	const long n = (long) planes * cols;
	if (nslabs > 32)
		hipLaunchKernelGGL((norm_sum_kernel<64, 16>), dim3((unsigned) ((n + 15) / 16)), dim3(1024), 0, rt().stream, partial, nslabs, planes, cols, first,
				second, accumulate);
	else
		hipLaunchKernelGGL((norm_sum_kernel<4, 64>), dim3((unsigned) ((n + 63) / 64)), dim3(256), 0, rt().stream, partial, nslabs, planes, cols, first,
				second, accumulate);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

template <int T, int E>
static void launch_fwd(const FwdArgs &a, bool join, bool vec, int policy) {
	constexpr int ROWS = T < TPB ? TPB / T : 1;
	const dim3 grid((unsigned) ((a.rows + ROWS - 1) / ROWS)), block(T < TPB ? TPB : T);
	if (join && vec) hipLaunchKernelGGL((norm_fwd_kernel<T, E / 4, 4, true>), grid, block, 0, rt().stream, a, policy);
	else if (join) hipLaunchKernelGGL((norm_fwd_kernel<T, E, 1, true>), grid, block, 0, rt().stream, a, policy);
	else if (vec) hipLaunchKernelGGL((norm_fwd_kernel<T, E / 4, 4, false>), grid, block, 0, rt().stream, a, policy);
	else hipLaunchKernelGGL((norm_fwd_kernel<T, E, 1, false>), grid, block, 0, rt().stream, a, policy);
}

// 128-bit accesses: every row of every plane starts on 16 bytes
static bool vec_ok(const Planes &p) { return p.ld % 4 == 0 && aligned16(p.re) && aligned16(p.im); }
static bool vec_ok(const Out4 &o) { return o.ld % 4 == 0 && aligned16(o.re) && aligned16(o.im) && aligned16(o.sre) && aligned16(o.sim); }

static int norm_fwd(FwdArgs &a, bool join) {
	a.inv_cols = 1.0 / a.cols;
	const bool vec = a.cols % 4 == 0 && vec_ok(a.x) && vec_ok(a.v) && vec_ok(a.u) && vec_ok(a.w) && vec_ok(Planes{a.y_re, a.y_im, a.ldy}) &&
			vec_ok(Planes{a.h_re, a.h_im, a.ldh});
	const int policy = stream_policy(ST_STORES, join ? 8 : 4, (long) a.rows * a.cols);
	if (a.cols <= 256) launch_fwd<64, 4>(a, join, vec, policy);
	else if (a.cols <= 512) launch_fwd<64, 8>(a, join, vec, policy);
	else if (a.cols <= 1024) launch_fwd<64, 16>(a, join, vec, policy);
	else if (a.cols <= 2048) launch_fwd<256, 8>(a, join, vec, policy);
	else if (a.cols <= 4096) launch_fwd<256, 16>(a, join, vec, policy);
	else if (a.cols <= 8192) launch_fwd<1024, 8>(a, join, vec, policy);
	else if (a.cols <= 16384) launch_fwd<1024, 16>(a, join, vec, policy);
	else if (join) hipLaunchKernelGGL(norm_fwd_wide_kernel<true>, dim3((unsigned) a.rows), dim3(WIDE), 0, rt().stream, a);
	else hipLaunchKernelGGL(norm_fwd_wide_kernel<false>, dim3((unsigned) a.rows), dim3(WIDE), 0, rt().stream, a);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

template <int T, int E>
static void launch_bwd(const BwdArgs &a, bool second, bool vec, int nslabs, int policy) {
	constexpr int R = T < TPB ? TPB / T : 1;
	const dim3 grid((unsigned) nslabs), block(T < TPB ? TPB : T);
	const size_t lds = (size_t) (R - 1) * (second ? 4 : 2) * T * E * sizeof(float);
	if (second && vec) hipLaunchKernelGGL((norm_bwd_kernel<T, E / 4, 4, true, true>), grid, block, lds, rt().stream, a, policy);
	else if (second) hipLaunchKernelGGL((norm_bwd_kernel<T, E, 1, true, true>), grid, block, lds, rt().stream, a, policy);
	else if (vec) hipLaunchKernelGGL((norm_bwd_kernel<T, E / 4, 4, false, true>), grid, block, lds, rt().stream, a, policy);
	else hipLaunchKernelGGL((norm_bwd_kernel<T, E, 1, false, true>), grid, block, lds, rt().stream, a, policy);
}

static void launch_bwd_twice(const BwdArgs &a, bool second, bool vec, int nslabs) {
	const dim3 grid((unsigned) nslabs), block(512);
	if (second && vec) hipLaunchKernelGGL((norm_bwd_twice_kernel<512, 4, 4, true>), grid, block, 0, rt().stream, a);
	else if (second) hipLaunchKernelGGL((norm_bwd_twice_kernel<512, 16, 1, true>), grid, block, 0, rt().stream, a);
	else if (vec) hipLaunchKernelGGL((norm_bwd_twice_kernel<512, 4, 4, false>), grid, block, 0, rt().stream, a);
	else hipLaunchKernelGGL((norm_bwd_twice_kernel<512, 16, 1, false>), grid, block, 0, rt().stream, a);
}

// The gate alone is the join without a second norm, without a residual path to hand its gradient to, and with scale 1: its gradient
// at y arrives in a.gh then.
static int norm_bwd(BwdArgs &a, const Out4 &dv, const Out4 &dw) {
	const bool shared = a.v.ld == 0, second = a.g.re != nullptr;
	a.planes = (shared ? 2 : 0) + (second ? 2 : 0);
	const bool vec = a.cols % 4 == 0 && vec_ok(a.x) && vec_ok(a.v) && vec_ok(a.h) && vec_ok(a.w) && vec_ok(a.g) && vec_ok(a.gh) && vec_ok(a.du) && vec_ok(a.dx) && vec_ok(a.dv);
	// Two workgroups to a compute unit, one of the wide ones, all with as many rows: a workgroup's sums are written and read again, which more of them
	// would do more often (8192 x 1024: 81 us with 512 workgroups, 89 with 768, 93 with 1024; 1024 x 8192: 139 with 256, 154 with 512).
	const int groups = a.cols <= 256 ? 4 : a.cols <= 512 ? 2 : 1;  // rows that a workgroup works on at a time
	// Without such sums (a gate per row) four to a unit: 515 x 1001 6.4 against 8.3 us, 3000 x 130 5.7 against 7.4, 8192 x 1024 the same;
	// the wide ones stay at one (1000 x 4000: 35 against 37).
	const int per_unit = a.cols > 1024 ? 1 : a.planes ? 2 : 4;
	const int want = std::max(1, std::min((a.rows + groups - 1) / groups, per_unit * rt().prop.multiProcessorCount));
	a.rows_per_slab = (a.rows + want - 1) / want;
	const int nslabs = (a.rows + a.rows_per_slab - 1) / a.rows_per_slab;
	if (a.planes) {
		a.partial = (float *) workspace((size_t) nslabs * a.planes * a.cols * sizeof(float));
		if (!a.partial) return rt().capturing ? CNET_ERR_UNSUPPORTED : CNET_ERR_OUT_OF_MEMORY;
	}
	const int policy = stream_policy(ST_LOADS, second ? 12 : 6, (long) a.rows * a.cols);
	if (a.cols <= 256) launch_bwd<64, 4>(a, second, vec, nslabs, policy);
	else if (a.cols <= 512) launch_bwd<128, 4>(a, second, vec, nslabs, policy);
	else if (a.cols <= 1024) launch_bwd<256, 4>(a, second, vec, nslabs, policy);
	else if (a.cols <= 2048) launch_bwd<512, 4>(a, second, vec, nslabs, policy);
	else if (a.cols <= 4096 && vec && second) hipLaunchKernelGGL((norm_bwd_kernel<512, 2, 4, true, false>), dim3((unsigned) nslabs), dim3(512), 0, rt().stream, a, policy);
	else if (a.cols <= 4096 && vec) hipLaunchKernelGGL((norm_bwd_kernel<512, 2, 4, false, false>), dim3((unsigned) nslabs), dim3(512), 0, rt().stream, a, policy);
	else if (a.cols <= 8192) launch_bwd_twice(a, second, vec, nslabs);
	else if (second) hipLaunchKernelGGL(norm_bwd_wide_kernel<true>, dim3((unsigned) nslabs), dim3(WIDE), 0, rt().stream, a);
	else hipLaunchKernelGGL(norm_bwd_wide_kernel<false>, dim3((unsigned) nslabs), dim3(WIDE), 0, rt().stream, a);
	CNET_LAUNCH_CHECK();
	return a.planes ? norm_sum(a.partial, nslabs, a.planes, a.cols, shared ? dv : dw, dw, a.accumulate_w) : CNET_OK;
}

static int norm_no_rows(int planes, int cols, const Out4 &first, const Out4 &second) { return norm_sum(nullptr, 0, planes, cols, first, second, 0); }

extern "C" {

int cnet_norm_gate_fwd(const float *x_re, const float *x_im, int64_t ldx, const float *v_re, const float *v_im, int64_t ldv, float *y_re,
		float *y_im, int64_t ldy, float *s, int rows, int cols, float eps) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 22) && cols > 0 && cols < (1 << 30));
	CNET_CHECK_ARG(eps >= 0.0f && std::isfinite(eps));
	if (!rows) return CNET_OK;
	CNET_CHECK_ARG(x_re && x_im && v_re && v_im && y_re && y_im);
	CNET_CHECK_ARG(ldx >= cols && (ldv == 0 || ldv >= cols) && ldy >= cols);
	FwdArgs a = {};
	a.x = Planes{x_re, x_im, (long) ldx};
	a.v = Planes{v_re, v_im, (long) ldv};
	a.y_re = y_re;
	a.y_im = y_im;
	a.ldy = ldy;
	a.s = s;
	a.eps = eps;
	a.rows = rows;
	a.cols = cols;
	return norm_fwd(a, false);
}

int cnet_norm_gate_bwd_sym(const float *x_re, const float *x_im, int64_t ldx, const float *s, const float *v_re, const float *v_im, int64_t ldv,
		const float *g_dz_re, const float *g_dz_im, int64_t ldg, float *dx_dz_re, float *dx_dz_im, float *dx_dzs_re, float *dx_dzs_im,
		int64_t lddx, float *dv_dz_re, float *dv_dz_im, float *dv_dzs_re, float *dv_dzs_im, int64_t lddv, int rows, int cols, int accumulate,
		int accumulate_w) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 22) && cols > 0 && cols < (1 << 30));
	if (!rows && (ldv || accumulate_w)) return CNET_OK;
	CNET_CHECK_ARG(dv_dz_re && dv_dz_im && ((dv_dzs_re == nullptr) == (dv_dzs_im == nullptr)) && lddv >= cols);
	const Out4 dv = {dv_dz_re, dv_dz_im, dv_dzs_re, dv_dzs_im, (long) lddv};
	BwdArgs a = {};
	a.rows = rows;
	a.cols = cols;
	if (!rows) return norm_no_rows(2, cols, dv, dv);
	CNET_CHECK_ARG(x_re && x_im && s && v_re && v_im && g_dz_re && g_dz_im && dx_dz_re && dx_dz_im);
	CNET_CHECK_ARG((dx_dzs_re == nullptr) == (dx_dzs_im == nullptr));
	CNET_CHECK_ARG(ldx >= cols && (ldv == 0 || ldv >= cols) && ldg >= cols && lddx >= cols);
	a.x = Planes{x_re, x_im, (long) ldx};
	a.v = Planes{v_re, v_im, (long) ldv};
	a.gh = Planes{g_dz_re, g_dz_im, (long) ldg};
	a.s = s;
	a.dx = Out4{dx_dz_re, dx_dz_im, dx_dzs_re, dx_dzs_im, (long) lddx};
	a.dv = dv;
	a.scale = 1.0f;
	a.accumulate = accumulate;
	a.accumulate_w = accumulate_w;
	return norm_bwd(a, dv, dv);
}

int cnet_norm_join_fwd(const float *u_re, const float *u_im, int64_t ldu, const float *f_re, const float *f_im, int64_t ldf, const float *v_re,
		const float *v_im, int64_t ldv, float scale, float *h_re, float *h_im, int64_t ldh, float *s, const float *w_re, const float *w_im,
		float *y_re, float *y_im, int64_t ldy, float *s2, int rows, int cols, float eps) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 22) && cols > 0 && cols < (1 << 30));
	CNET_CHECK_ARG(eps >= 0.0f && std::isfinite(eps));
	if (!rows) return CNET_OK;
	CNET_CHECK_ARG(u_re && u_im && f_re && f_im && v_re && v_im && h_re && h_im);
	CNET_CHECK_ARG(ldu >= cols && ldf >= cols && (ldv == 0 || ldv >= cols) && ldh >= cols);
	CNET_CHECK_ARG((w_re == nullptr) == (w_im == nullptr) && (y_re == nullptr) == (y_im == nullptr) && (w_re == nullptr) == (y_re == nullptr));
	CNET_CHECK_ARG(y_re == nullptr || ldy >= cols);
	FwdArgs a = {};
	a.x = Planes{f_re, f_im, (long) ldf};
	a.v = Planes{v_re, v_im, (long) ldv};
	a.u = Planes{u_re, u_im, (long) ldu};
	a.w = Planes{w_re, w_im, 0};
	a.y_re = y_re;
	a.y_im = y_im;
	a.ldy = ldy;
	a.h_re = h_re;
	a.h_im = h_im;
	a.ldh = ldh;
	a.s = s;
	a.s2 = s2;
	a.scale = scale;
	a.eps = eps;
	a.rows = rows;
	a.cols = cols;
	return norm_fwd(a, true);
}

int cnet_norm_join_bwd_sym(const float *f_re, const float *f_im, int64_t ldf, const float *s, const float *v_re, const float *v_im, int64_t ldv,
		float scale, const float *h_re, const float *h_im, int64_t ldh, const float *s2, const float *w_re, const float *w_im,
		const float *gh_dz_re, const float *gh_dz_im, int64_t ldgh, const float *gy_dz_re, const float *gy_dz_im, int64_t ldgy, float *du_dz_re,
		float *du_dz_im, float *du_dzs_re, float *du_dzs_im, int64_t lddu, float *df_dz_re, float *df_dz_im, float *df_dzs_re, float *df_dzs_im,
		int64_t lddf, float *dv_dz_re, float *dv_dz_im, float *dv_dzs_re, float *dv_dzs_im, int64_t lddv, float *dw_dz_re, float *dw_dz_im,
		float *dw_dzs_re, float *dw_dzs_im, int rows, int cols, int accumulate, int accumulate_w) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 22) && cols > 0 && cols < (1 << 30));
	CNET_CHECK_ARG((gh_dz_re == nullptr) == (gh_dz_im == nullptr) && (gy_dz_re == nullptr) == (gy_dz_im == nullptr));
	const bool second = gy_dz_re != nullptr || (!rows && dw_dz_re != nullptr);
	if (!rows && accumulate_w) return CNET_OK;
	CNET_CHECK_ARG(dv_dz_re && dv_dz_im && ((dv_dzs_re == nullptr) == (dv_dzs_im == nullptr)) && lddv >= cols);
	CNET_CHECK_ARG(!second || (dw_dz_re && dw_dz_im && ((dw_dzs_re == nullptr) == (dw_dzs_im == nullptr))));
	const Out4 dv = {dv_dz_re, dv_dz_im, dv_dzs_re, dv_dzs_im, (long) lddv}, dw = {dw_dz_re, dw_dz_im, dw_dzs_re, dw_dzs_im, 0};
	if (!rows) {
		if (ldv) return second ? norm_no_rows(2, cols, dw, dw) : CNET_OK;
		return norm_no_rows(second ? 4 : 2, cols, dv, dw);
	}
	CNET_CHECK_ARG(f_re && f_im && s && v_re && v_im && (gh_dz_re || gy_dz_re));
	CNET_CHECK_ARG(!second || (h_re && h_im && s2 && w_re && w_im && ldh >= cols && ldgy >= cols));
	CNET_CHECK_ARG(gh_dz_re == nullptr || ldgh >= cols);
	CNET_CHECK_ARG(du_dz_re && du_dz_im && ((du_dzs_re == nullptr) == (du_dzs_im == nullptr)) && lddu >= cols);
	CNET_CHECK_ARG(df_dz_re && df_dz_im && ((df_dzs_re == nullptr) == (df_dzs_im == nullptr)) && lddf >= cols);
	CNET_CHECK_ARG(ldf >= cols && (ldv == 0 || ldv >= cols));
	BwdArgs a = {};
	a.x = Planes{f_re, f_im, (long) ldf};
	a.v = Planes{v_re, v_im, (long) ldv};
	a.h = Planes{h_re, h_im, (long) ldh};
	a.w = Planes{w_re, w_im, 0};
	a.g = Planes{gy_dz_re, gy_dz_im, (long) ldgy};
	a.gh = Planes{gh_dz_re, gh_dz_im, (long) ldgh};
	a.s = s;
	a.s2 = s2;
	a.du = Out4{du_dz_re, du_dz_im, du_dzs_re, du_dzs_im, (long) lddu};
	a.dx = Out4{df_dz_re, df_dz_im, df_dzs_re, df_dzs_im, (long) lddf};
	a.dv = dv;
	a.scale = scale;
	a.rows = rows;
	a.cols = cols;
	a.accumulate = accumulate;
	a.accumulate_w = accumulate_w;
	return norm_bwd(a, dv, dw);
}

}  // extern "C"
