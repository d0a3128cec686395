// Norms around a block of layers, with the weights, the residual path and the scale that go with them.
//
//   in front of a block   y = v .* n,            n = x s,   s = 1 / max(sqrt(mean |x|^2 + eps), 1e-15)   (one s per row)
//   behind it             h = u + scale v .* (f s1)         f: what the block computed, u: the residual path
//   and for the next one  y = w .* (h s2)
//
// Backward, for a conjugate gradient pair, all as dL/dz: with g = dL/dy and p = g v (= dL/dn),
//   dx = s (p - conj(n) t),  t = mean Re(p n),     dv = g n  (summed over the rows when they share v);
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
	int rows, cols;
};

struct BwdArgs {
	Planes x, v, h, w, g, gh;  // x the operand of the (first) norm; h, w, gh belong to the join; g = dL/dy
	const float *s, *s2;
	Out4 du, dx, dv;   // dv: only with a gate of its own for every row (the shared one goes through `partial`)
	float *partial;    // [slab][planes][cols]: dv re, im (unless every row has a gate of its own), dw re, im
	int planes, rows_per_slab;
	float scale;
	int rows, cols, accumulate, accumulate_w;
};

// (the clamp lets a NaN through, which fmaxf would not: the whole row is then NaN)
__device__ __forceinline__ float inv_rms(float sum, int cols, float eps) {
	const float rms = sqrtf(sum / (float) cols + eps);
	return 1.0f / (rms <= 1.0e-15f ? 1.0e-15f : rms);
}

__device__ __forceinline__ void put(float *p, float v, int accumulate) { *p = accumulate ? *p + v : v; }

// One workgroup per row, any width: the row is walked once per stage.
template <bool JOIN>
__global__ __launch_bounds__(TPB) void norm_fwd_kernel(const FwdArgs a) {
	__shared__ float lds[TPB / 64];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const long row = blockIdx.x;
	const float *xr = a.x.re + row * a.x.ld, *xi = a.x.im + row * a.x.ld;
	const float *vr = a.v.re + row * a.v.ld, *vi = a.v.im + row * a.v.ld;
	float sum = 0.f;
	for (int c = t; c < a.cols; c += TPB) sum += xr[c] * xr[c] + xi[c] * xi[c];
	sum = group_reduce<float, TPB / 64>(sum, SumF(), lds, 0, wave, lane);
	const float s = inv_rms(sum, a.cols, a.eps);
	if (t == 0 && a.s) a.s[row] = s;
	if (!JOIN) {
		for (int c = t; c < a.cols; c += TPB) {
			const float n_r = xr[c] * s, n_i = xi[c] * s;
			a.y_re[row * a.ldy + c] = vr[c] * n_r - vi[c] * n_i;
			a.y_im[row * a.ldy + c] = vr[c] * n_i + vi[c] * n_r;
		}
		return;
	}
	float sum2 = 0.f;
	for (int c = t; c < a.cols; c += TPB) {
		const float n_r = xr[c] * s, n_i = xi[c] * s;
		const float h_r = a.u.re[row * a.u.ld + c] + a.scale * (vr[c] * n_r - vi[c] * n_i);
		const float h_i = a.u.im[row * a.u.ld + c] + a.scale * (vr[c] * n_i + vi[c] * n_r);
		a.h_re[row * a.ldh + c] = h_r;
		a.h_im[row * a.ldh + c] = h_i;
		sum2 += h_r * h_r + h_i * h_i;
	}
	if (!a.y_re) return;
	sum2 = group_reduce<float, TPB / 64>(sum2, SumF(), lds, 0, wave, lane);
	const float s2 = inv_rms(sum2, a.cols, a.eps);
	if (t == 0 && a.s2) a.s2[row] = s2;
	const float *wr = a.w.re + row * a.w.ld, *wi = a.w.im + row * a.w.ld;
	for (int c = t; c < a.cols; c += TPB) {
		const float n_r = a.h_re[row * a.ldh + c] * s2, n_i = a.h_im[row * a.ldh + c] * s2;
		a.y_re[row * a.ldy + c] = wr[c] * n_r - wi[c] * n_i;
		a.y_im[row * a.ldy + c] = wr[c] * n_i + wi[c] * n_r;
	}
}

// A workgroup takes `rows_per_slab` rows one after the other; its columns' sums of dv and dw stay in its own rows of `partial`
// (each thread always meets the same columns: no atomics, one order), which norm_sum_kernel adds in slab order.
template <bool JOIN>
__global__ __launch_bounds__(TPB) void norm_bwd_kernel(const BwdArgs a) {
	__shared__ float lds[TPB / 64];
	const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
	const int r0 = blockIdx.x * a.rows_per_slab, r1 = min(a.rows, r0 + a.rows_per_slab);
	const bool shared = a.v.ld == 0;
	const float inv_n = 1.0f / (float) a.cols;
	float *part = a.partial + (long) blockIdx.x * a.planes * a.cols;
	for (long row = r0; row < r1; ++row) {
		const float s = a.s[row], s2 = JOIN && a.g.re ? a.s2[row] : 0.f;
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
		if (JOIN && a.g.re) {
			for (int c = t; c < a.cols; c += TPB) {
				float p_r, p_i, n_r, n_i;
				next(c, p_r, p_i, n_r, n_i);
				t2 += p_r * n_r - p_i * n_i;
			}
			t2 = group_reduce<float, TPB / 64>(t2, SumF(), lds, 0, wave, lane) * inv_n;
		}
		// the gradient at the result of the (first) norm and its weights: scale dh, or g
		auto at = [&](int c, float &d_r, float &d_i) {
			if (!JOIN) {
				d_r = a.g.re[row * a.g.ld + c];
				d_i = a.g.im[row * a.g.ld + c];
				return;
			}
			d_r = a.gh.re ? a.gh.re[row * a.gh.ld + c] : 0.f;
			d_i = a.gh.re ? a.gh.im[row * a.gh.ld + c] : 0.f;
			if (a.g.re) {
				float p_r, p_i, n_r, n_i;
				next(c, p_r, p_i, n_r, n_i);
				d_r += s2 * (p_r - n_r * t2);
				d_i += s2 * (p_i + n_i * t2);
			}
		};
		const float k = JOIN ? a.scale : 1.0f;
		float t1 = 0.f;
		for (int c = t; c < a.cols; c += TPB) {
			float d_r, d_i;
			at(c, d_r, d_i);
			d_r *= k;
			d_i *= k;
			const float v_r = a.v.re[row * a.v.ld + c], v_i = a.v.im[row * a.v.ld + c];
			const float n_r = a.x.re[row * a.x.ld + c] * s, n_i = a.x.im[row * a.x.ld + c] * s;
			t1 += (d_r * v_r - d_i * v_i) * n_r - (d_r * v_i + d_i * v_r) * n_i;
		}
		t1 = group_reduce<float, TPB / 64>(t1, SumF(), lds, 0, wave, lane) * inv_n;
		for (int c = t; c < a.cols; c += TPB) {
			float d_r, d_i;
			at(c, d_r, d_i);
			if (JOIN) {
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
			if (JOIN && a.g.re) {
				float p_r, p_i, m_r, m_i;
				next(c, p_r, p_i, m_r, m_i);
				const float g_r = a.g.re[row * a.g.ld + c], g_i = a.g.im[row * a.g.ld + c];
				put(pw, g_r * m_r - g_i * m_i, row > r0);
				put(pw + a.cols, g_r * m_i + g_i * m_r, row > r0);
			}
		}
	}
}

// dst[plane][c] (+)= sum over slabs, in slab order; plane 0, 1: `first`, 2, 3: `second`
__global__ __launch_bounds__(TPB) void norm_sum_kernel(const float *__restrict__ partial, int nslabs, int planes, int cols, Out4 first, Out4 second,
		int accumulate) {
	const long idx = (long) blockIdx.x * TPB + threadIdx.x;
	if (idx >= (long) planes * cols) return;
	const int p = (int) (idx / cols), c = (int) (idx - (long) p * cols);
	const float sum = cnet::ordered_sum(partial + idx, (long) planes * cols, nslabs);
	const Out4 &o = p < 2 ? first : second;
	put((p & 1 ? o.im : o.re) + c, sum, accumulate);
	if (o.sre) put((p & 1 ? o.sim : o.sre) + c, p & 1 ? -sum : sum, accumulate);
}

}  // namespace

using namespace cnet;

static int norm_fwd(const FwdArgs &a, bool join) {
	dim3 grid((unsigned) a.rows);
	if (join) hipLaunchKernelGGL(norm_fwd_kernel<true>, grid, dim3(TPB), 0, rt().stream, a);
	else hipLaunchKernelGGL(norm_fwd_kernel<false>, grid, dim3(TPB), 0, rt().stream, a);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

static int norm_bwd(BwdArgs &a, bool join, const Out4 &dv, const Out4 &dw) {
	const bool shared = a.v.ld == 0, second = join && a.g.re;
	a.planes = (shared ? 2 : 0) + (second ? 2 : 0);
	const int want = std::min(a.rows, 4 * rt().prop.multiProcessorCount);
	a.rows_per_slab = (a.rows + want - 1) / want;
	const int nslabs = (a.rows + a.rows_per_slab - 1) / a.rows_per_slab;
	if (a.planes) {
		a.partial = (float *) workspace((size_t) nslabs * a.planes * a.cols * sizeof(float));
		if (!a.partial) return rt().capturing ? CNET_ERR_UNSUPPORTED : CNET_ERR_OUT_OF_MEMORY;
	}
	if (join) hipLaunchKernelGGL(norm_bwd_kernel<true>, dim3((unsigned) nslabs), dim3(TPB), 0, rt().stream, a);
	else hipLaunchKernelGGL(norm_bwd_kernel<false>, dim3((unsigned) nslabs), dim3(TPB), 0, rt().stream, a);
	CNET_LAUNCH_CHECK();
	if (a.planes) {
		const long n = (long) a.planes * a.cols;
		hipLaunchKernelGGL(norm_sum_kernel, dim3((unsigned) ((n + TPB - 1) / TPB)), dim3(TPB), 0, rt().stream, a.partial, nslabs, a.planes, a.cols,
				shared ? dv : dw, dw, a.accumulate_w);
		CNET_LAUNCH_CHECK();
	}
	return CNET_OK;
}

// no rows: the sum over them is zero
static int norm_no_rows(int planes, int cols, const Out4 &first, const Out4 &second) {
	const long n = (long) planes * cols;
	hipLaunchKernelGGL(norm_sum_kernel, dim3((unsigned) ((n + TPB - 1) / TPB)), dim3(TPB), 0, rt().stream, nullptr, 0, planes, cols, first, second, 0);
	CNET_LAUNCH_CHECK();
	return CNET_OK;
}

extern "C" {

int cnet_norm_gate_fwd(const float *x_re, const float *x_im, int64_t ldx, const float *v_re, const float *v_im, int64_t ldv, float *y_re,
		float *y_im, int64_t ldy, float *s, int rows, int cols, float eps) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 24) && cols > 0);
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
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 24) && cols > 0);
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
	a.g = Planes{g_dz_re, g_dz_im, (long) ldg};
	a.s = s;
	a.dx = Out4{dx_dz_re, dx_dz_im, dx_dzs_re, dx_dzs_im, (long) lddx};
	a.dv = dv;
	a.scale = 1.0f;
	a.accumulate = accumulate;
	a.accumulate_w = accumulate_w;
	return norm_bwd(a, false, dv, dv);
}

int cnet_norm_join_fwd(const float *u_re, const float *u_im, int64_t ldu, const float *f_re, const float *f_im, int64_t ldf, const float *v_re,
		const float *v_im, int64_t ldv, float scale, float *h_re, float *h_im, int64_t ldh, float *s, const float *w_re, const float *w_im,
		float *y_re, float *y_im, int64_t ldy, float *s2, int rows, int cols, float eps) {
	CNET_REQUIRE_INIT();
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 24) && cols > 0);
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
	CNET_CHECK_ARG(rows >= 0 && rows < (1 << 24) && cols > 0);
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
	return norm_bwd(a, true, dv, dw);
}

}  // extern "C"
