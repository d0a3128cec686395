// Gram matrices in double and products with them (gram.hip), as the vocabulary head uses them.
#ifndef CNET_CSRC_GRAM_HPP_
#define CNET_CSRC_GRAM_HPP_

namespace cnet {

constexpr int GRAM_TILE = 64, GRAM_CHUNK = 16;  // edge of a block of the result, and of what it is summed over

// planes re and im [K][ld] of a K x K matrix, one behind the other
struct Gram64 {
	double *re;
	long ld;
};

// Where conj(A) G goes: fp32 planes (all NULL: nowhere), the conjugate's (NULL: not wanted), added or not; part [M][blocks of columns]
// (or NULL): Re sum_j C_ij A_ij over each block's columns.
struct GramOut {
	float *re, *im, *sre, *sim;
	long ld;
	int accumulate;
	double *part;
};

// C = A^H diag(weight) A for L > 0 rows of K columns.  weight NULL: all 1; a row of weight 0 is left out whatever it holds.
// The order of the sums depends on K and L alone.
int gram64(int K, int L, const float *a_re, const float *a_im, long lda, const double *weight, const Gram64 &c);
// C = conj(A) G for M > 0 rows
int times_gram(int M, int K, const float *a_re, const float *a_im, long lda, const Gram64 &g, const GramOut &out);
// what the two take, in microseconds, from the work of their matrix instructions
double gram64_us(int K, int L);
double times_gram_us(int M, int K);

}  // namespace cnet

#endif
