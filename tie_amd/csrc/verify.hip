// verify.hip -- which drafted tokens of a tree the target accepts, and the
// token that follows, from given random numbers.
//
// p = softmax(logits / temperature) of a node, q its draft distribution.  Its
// children are tried in order, with c = 0 and M = 1 at first: child x is taken
// when u q(x) M < max(0, p(x) - c q(x)); else c += M and M = sum max(0, p - c
// q).  (That is rejection sampling with the residual max(0, p' - q) / sum of
// it after each rejection, written for p' = max(0, p - c q) / M.)  Without a
// draft distribution q is one at x: u M < p(x), and a refused x leaves p.
// Where no child is taken the next token is the first whose running sum of the
// residual exceeds u M.  Tokens follow the target's distribution whatever the
// draft was.
//
// Each node's outcome depends on its own rows and random numbers alone, so all
// nodes are worked on at once and the path is read off at the end.  Sums are
// in 64 bits: the running sum crosses u M at the same token whatever the
// order of the sum.
#include "kv.h"

namespace tie {

constexpr int V_CHUNK = 4096; // logits of a workgroup
constexpr int V_KIDS = VERIFY_KIDS;

struct VerifyWork {
	int chunks;
	double *s;     // [n_tokens][chunks] sum of exp((l - m) / temperature)
	float *m;      // [n_tokens][chunks] largest logit
	int32_t *arg;  // [n_tokens][chunks] its lowest index
	double *res;   // [max_children][n_tokens][chunks] sums of max(0, p - c q) after each refusal
	int32_t *take; // [n_tokens] the child taken (a token row), -1: none
	int32_t *own;  // [n_tokens] the next token where none is taken
	int32_t *leaf; // [n_tokens] the next token where the children do not count
};

static size_t carve_verify(const VerifyArgs &a, bool with_draft, uint8_t *base, VerifyWork *w)
{
	size_t off = WORK_COUNTERS * sizeof(int);
	auto take = [&](size_t bytes) {
		const size_t o = off;
		off += (bytes + 255) & ~(size_t)255;
		return base + o;
	};
	const size_t N = a.n_tokens, C = (a.vocab + V_CHUNK - 1) / V_CHUNK;
	VerifyWork v;
	v.chunks = (int)C;
	v.s = (double *)take(N * C * 8);
	v.res = (double *)take(with_draft ? (size_t)a.max_children * N * C * 8 : 0);
	v.m = (float *)take(N * C * 4);
	v.arg = (int32_t *)take(N * C * 4);
	v.take = (int32_t *)take(N * 4);
	v.own = (int32_t *)take(N * 4);
	v.leaf = (int32_t *)take(N * 4);
	if (w)
		*w = v;
	return off;
}

size_t verify_work_bytes(const VerifyArgs &a, bool with_draft)
{
	return carve_verify(a, with_draft, nullptr, nullptr);
}

template <typename T>
__device__ __forceinline__ T wave_total(T x)
{
#pragma unroll
	for (int m = 1; m < 64; m <<= 1)
		x += __shfl_xor(x, m);
	return x;
}

// the sum over a workgroup of 256, in every thread
__device__ __forceinline__ double block_total(double x, double *tmp)
{
	x = wave_total(x);
	__syncthreads();
	if ((threadIdx.x & 63) == 0)
		tmp[threadIdx.x >> 6] = x;
	__syncthreads();
	return (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
}

__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a, VerifyWork w)
{
	__shared__ float tm[4];
	__shared__ int ti[4];
	__shared__ double ts[4];
	const int t = blockIdx.y, chunk = blockIdx.x, base = chunk * V_CHUNK;
	const float *l = a.logits + (size_t)t * a.l_stride;
	constexpr int E = V_CHUNK / 256;
	float x[E];
	float m = -__builtin_inff();
	int at = 0x7fffffff;
#pragma unroll
	for (int e = 0; e < E; e++) {
		const int i = base + e * 256 + threadIdx.x;
		x[e] = i < a.vocab ? l[i] : -__builtin_inff();
		if (x[e] > m) {
			m = x[e];
			at = i;
		}
	}
#pragma unroll
	for (int q = 1; q < 64; q <<= 1) {
		const float om = __shfl_xor(m, q);
		const int oi = __shfl_xor(at, q);
		if (om > m || (om == m && oi < at)) {
			m = om;
			at = oi;
		}
	}
	if ((threadIdx.x & 63) == 0) {
		tm[threadIdx.x >> 6] = m;
		ti[threadIdx.x >> 6] = at;
	}
	__syncthreads();
#pragma unroll
	for (int q = 0; q < 4; q++)
		if (tm[q] > m || (tm[q] == m && ti[q] < at)) {
			m = tm[q];
			at = ti[q];
		}
	double s = 0.0;
	if (a.temperature > 0.0f && m > -__builtin_inff()) {
		const double inv = 1.0 / (double)a.temperature;
#pragma unroll
		for (int e = 0; e < E; e++)
			if (x[e] > -__builtin_inff())
				s += exp(((double)x[e] - (double)m) * inv);
		s = block_total(s, ts);
	}
	if (threadIdx.x == 0) {
		const size_t o = (size_t)t * w.chunks + chunk;
		w.m[o] = m;
		w.s[o] = s;
		w.arg[o] = at < a.vocab ? at : 0;
	}
}

// A node as every thread of a workgroup sees it.
struct Node {
	float m;             // largest logit
	double inv, scale;   // p(i) = exp((l - m) inv) * scale
	int best;            // greedy: its index
	int kids[V_KIDS], n; // children tried (token rows), in order
	int taken;           // the child taken, -1: none (so far)
	int refused;         // children refused
	double c, M;
	int more;            // the residual sum that is still to be formed (-1: none)
	int gone[V_KIDS], n_gone; // no draft: refused tokens
};

__device__ __forceinline__ double prob(const Node &d, float l)
{
	return exp(((double)l - (double)d.m) * d.inv) * d.scale;
}

// The node's state after `passes` residual sums: thread-uniform, all threads.
__device__ void node_state(const VerifyArgs &a, const VerifyWork &w, int t, int passes, Node &d, int *lds)
{
	// the largest logit and the sum
	const float *m = w.m + (size_t)t * w.chunks;
	d.m = -__builtin_inff();
	d.best = 0;
	for (int c = 0; c < w.chunks; c++)
		if (m[c] > d.m) {
			d.m = m[c];
			d.best = w.arg[(size_t)t * w.chunks + c];
		}
	d.inv = a.temperature > 0.0f ? 1.0 / (double)a.temperature : 0.0;
	double z = 0.0;
	if (a.temperature > 0.0f)
		for (int c = 0; c < w.chunks; c++)
			if (m[c] > -__builtin_inff())
				z += w.s[(size_t)t * w.chunks + c] * exp(((double)m[c] - (double)d.m) * d.inv);
	d.scale = 1.0 / z;
	// the children: later nodes of the same sequence whose parent this is
	int lo = 0, hi = a.n_seqs;
	if (a.first) {
		while (lo < hi) {
			const int mid = (lo + hi) >> 1;
			if (a.first[mid + 1] <= t)
				lo = mid + 1;
			else
				hi = mid;
		}
	} else {
		lo = t;
	}
	int t0 = t, t1 = t + 1;
	if (a.first) {
		t0 = lo < a.n_seqs ? max(0, a.first[lo]) : t;
		t1 = lo < a.n_seqs ? min(a.n_tokens, a.first[lo + 1]) : t;
	}
	__syncthreads();
	if (threadIdx.x < 64) {
		int n = 0;
		for (int b = t + 1; b < t1 && n < a.max_children; b += 64) {
			const int j = b + (int)threadIdx.x;
			const bool is = j < t1 && a.parent[j] == t - t0;
			const unsigned long long set = __ballot(is);
			const int place = n + __builtin_popcountll(set & ((1ull << threadIdx.x) - 1));
			if (is && place < a.max_children)
				lds[1 + place] = j;
			n += __builtin_popcountll(set);
		}
		if (threadIdx.x == 0)
			lds[0] = min(n, a.max_children);
	}
	__syncthreads();
	d.n = lds[0];
	for (int i = 0; i < d.n; i++)
		d.kids[i] = lds[1 + i];
	d.taken = -1;
	d.refused = d.n_gone = 0;
	d.more = -1;
	d.c = 0.0;
	d.M = 1.0;
	const float *l = a.logits + (size_t)t * a.l_stride;
	for (int i = 0; i < d.n; i++) {
		const int x = a.tokens[d.kids[i]];
		if (x < 0 || x >= a.vocab)
			continue; // no token: not tried
		if (a.temperature == 0.0f) {
			if (x == d.best) {
				d.taken = d.kids[i];
				return;
			}
			continue;
		}
		const double p = prob(d, l[x]), u = (double)a.u_accept[d.kids[i]];
		if (a.draft) {
			const double q = (double)a.draft[(size_t)t * a.d_stride + x];
			const double r = p - d.c * q;
			if (u * d.M * q < (r > 0.0 ? r : 0.0)) {
				d.taken = d.kids[i];
				return;
			}
			d.c += d.M;
			if (d.refused >= passes) {
				d.more = d.refused;
				return;
			}
			const double *s = w.res + ((size_t)d.refused * a.n_tokens + t) * w.chunks;
			double M = 0.0;
			for (int c = 0; c < w.chunks; c++)
				M += s[c];
			d.M = M;
			d.refused++;
		} else {
			bool again = false;
			for (int k = 0; k < d.n_gone; k++)
				again = again || d.gone[k] == x;
			if (!again && u * d.M < p) {
				d.taken = d.kids[i];
				return;
			}
			if (!again) {
				d.gone[d.n_gone++] = x;
				d.M -= p;
			}
		}
	}
}

// One more residual sum for the nodes that need it.
__global__ __launch_bounds__(256) void verify_residual_kernel(VerifyArgs a, VerifyWork w, int pass)
{
	__shared__ int lds[1 + V_KIDS];
	__shared__ double ts[4];
	const int t = blockIdx.y, base = blockIdx.x * V_CHUNK;
	Node d;
	node_state(a, w, t, pass, d, lds);
	if (d.more != pass)
		return;
	const float *l = a.logits + (size_t)t * a.l_stride, *q = a.draft + (size_t)t * a.d_stride;
	double s = 0.0;
	for (int e = 0; e < V_CHUNK / 256; e++) {
		const int i = base + e * 256 + threadIdx.x;
		if (i < a.vocab) {
			const double r = prob(d, l[i]) - d.c * (double)q[i];
			s += r > 0.0 ? r : 0.0;
		}
	}
	s = block_total(s, ts);
	if (threadIdx.x == 0)
		w.res[((size_t)pass * a.n_tokens + t) * w.chunks + blockIdx.x] = s;
}

// The first index whose running weight exceeds u times the whole: over the
// chunks' sums, then inside the chunk.  weight(i) >= 0; sum(c): of chunk c.
template <typename W, typename S>
__device__ int locate(const VerifyArgs &a, int chunks, double u, W weight, S sum, double *tmp, int *ti)
{
	double all = 0.0;
	for (int c = 0; c < chunks; c++)
		all += sum(c);
	const double want = u * all;
	double before = 0.0;
	int at = -1, last = 0;
	for (int c = 0; c < chunks; c++) {
		const double s = sum(c);
		if (s > 0.0)
			last = c;
		if (at < 0 && before + s > want)
			at = c;
		if (at < 0)
			before += s;
	}
	if (at < 0) { // (u of one, or a rounding at the end: the last weight there is)
		at = last;
		before -= sum(last);
	}
	// thread i has 16 weights in a row
	constexpr int E = V_CHUNK / 256;
	const int base = at * V_CHUNK + threadIdx.x * E;
	double mine = 0.0;
	for (int e = 0; e < E; e++)
		mine += base + e < a.vocab ? weight(base + e) : 0.0;
	double incl = mine;
#pragma unroll
	for (int m = 1; m < 64; m <<= 1) {
		const double o = __shfl_up(incl, m);
		if ((int)(threadIdx.x & 63) >= m)
			incl += o;
	}
	__syncthreads();
	if ((threadIdx.x & 63) == 63)
		tmp[threadIdx.x >> 6] = incl;
	if (threadIdx.x == 0)
		ti[0] = 0x7fffffff, ti[1] = 0;
	__syncthreads();
	double run = before + incl - mine;
	for (int q = 0; q < (int)(threadIdx.x >> 6); q++)
		run += tmp[q];
	for (int e = 0; e < E; e++) {
		const int i = base + e;
		const double x = i < a.vocab ? weight(i) : 0.0;
		run += x;
		if (x > 0.0) {
			atomicMax(&ti[1], i);
			if (run > want) {
				atomicMin(&ti[0], i);
				break;
			}
		}
	}
	__syncthreads();
	const int got = ti[0] < a.vocab ? ti[0] : ti[1];
	__syncthreads();
	return got;
}

// A node's outcome: the child taken, or the next token.
__global__ __launch_bounds__(256) void verify_node_kernel(VerifyArgs a, VerifyWork w)
{
	__shared__ int lds[1 + V_KIDS], ti[2];
	__shared__ double tmp[4];
	const int t = blockIdx.x;
	Node d;
	node_state(a, w, t, a.max_children, d, lds);
	int own = d.best, leaf = d.best;
	if (a.temperature > 0.0f) {
		const float *l = a.logits + (size_t)t * a.l_stride, *q = a.draft ? a.draft + (size_t)t * a.d_stride : nullptr;
		const float *m = w.m + (size_t)t * w.chunks;
		const double *s = w.s + (size_t)t * w.chunks;
		const double u = (double)a.u_sample[t];
		auto p_sum = [&](int c) { return m[c] > -__builtin_inff() ? s[c] * exp(((double)m[c] - (double)d.m) * d.inv) * d.scale : 0.0; };
		auto p_at = [&](int i) { return prob(d, l[i]); };
		leaf = own = locate(a, w.chunks, u, p_at, p_sum, tmp, ti);
		if (d.taken < 0 && a.draft && d.refused && d.M > 0.0) {
			const double *r = w.res + ((size_t)(d.refused - 1) * a.n_tokens + t) * w.chunks;
			// (c before the last M was added to it: d.c holds the sum that r was formed with)
			own = locate(a, w.chunks, u, [&](int i) {
				const double x = prob(d, l[i]) - d.c * (double)q[i];
				return x > 0.0 ? x : 0.0;
			}, [&](int c) { return r[c]; }, tmp, ti);
		} else if (d.taken < 0 && d.n_gone && d.M > 0.0) {
			auto left = [&](int i) {
				for (int k = 0; k < d.n_gone; k++)
					if (d.gone[k] == i)
						return 0.0;
				return prob(d, l[i]);
			};
			own = locate(a, w.chunks, u, left, [&](int c) {
				double x = p_sum(c);
				for (int k = 0; k < d.n_gone; k++)
					if (d.gone[k] / V_CHUNK == c)
						x -= prob(d, l[d.gone[k]]);
				return x > 0.0 ? x : 0.0;
			}, tmp, ti);
		}
	}
	if (threadIdx.x == 0) {
		w.take[t] = d.taken;
		w.own[t] = own;
		w.leaf[t] = leaf;
	}
}

// The path of each sequence: a thread each.
__global__ __launch_bounds__(64) void verify_path_kernel(VerifyArgs a, VerifyWork w)
{
	const int b = blockIdx.x * 64 + threadIdx.x;
	if (b >= a.n_seqs)
		return;
	int t0 = b, t1 = b + 1;
	if (a.first) {
		t0 = a.first[b];
		t1 = a.first[b + 1];
	}
	int32_t *path = a.path + (size_t)b * a.max_path;
	int n = 0, next = 0;
	if (t0 >= 0 && t0 < t1 && t1 <= a.n_tokens) {
		int t = t0;
		for (;;) {
			path[n++] = t - t0;
			if (n >= a.max_path) {
				next = w.leaf[t]; // (its children were never to be tried)
				break;
			}
			const int kid = w.take[t];
			if (kid < 0) {
				next = w.own[t];
				break;
			}
			t = kid; // (a later row of the same sequence)
		}
	}
	for (int i = n; i < a.max_path; i++)
		path[i] = -1;
	a.n_keep[b] = n;
	a.next[b] = n ? next : -1;
}

hipError_t launch_verify(const VerifyArgs &a, void *work, hipStream_t st)
{
	VerifyWork w;
	carve_verify(a, a.draft != nullptr, (uint8_t *)work, &w);
	if (a.n_tokens == 0) {
		tie_launch(verify_path_kernel, dim3((a.n_seqs + 63) / 64), dim3(64), 0, st, a, w);
		return hipGetLastError();
	}
	tie_launch(verify_stats_kernel, dim3(w.chunks, a.n_tokens), dim3(256), 0, st, a, w);
	if (a.draft && a.temperature > 0.0f)
		for (int p = 0; p < a.max_children; p++)
			tie_launch(verify_residual_kernel, dim3(w.chunks, a.n_tokens), dim3(256), 0, st, a, w, p);
	tie_launch(verify_node_kernel, dim3(a.n_tokens), dim3(256), 0, st, a, w);
	tie_launch(verify_path_kernel, dim3((a.n_seqs + 63) / 64), dim3(64), 0, st, a, w);
	return hipGetLastError();
}

} // namespace tie
