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
// nodes are worked on at once, a workgroup to V_CHUNK logits, and the path is
// read off at the end.  The last workgroup of a row forms the row's outcome, the
// last row of a sequence its path: one launch, and one more for each residual
// sum that some row may need (rows that do not leave it at once).  Sums are in 64
// bits: the running sum crosses u M at the same token whatever the order of the
// sum.
#include "kv.h"

namespace tie {

constexpr int V_CHUNK = 4096; // logits of a workgroup
constexpr int V_THREADS = 256, V_E = V_CHUNK / V_THREADS;
constexpr int V_KIDS = VERIFY_KIDS;
constexpr int V_PATH_LDS = 1024; // nodes of a sequence whose outcomes the path's reader keeps in LDS

// A row between its passes.
struct VRow {
	double scale, c, M; // p(i) = exp((l - m) / temperature) scale; the residual's c and M
	float m;
	int best;    // the lowest index of the largest logit
	int kid;     // the next child to try
	int waits;   // the residual sum it waits for (-1: none)
};

struct VerifyWork {
	int chunks;
	int join;      // 1: rows and sequences are finished by the last to arrive (counters)
	double *s;     // [n_tokens][chunks] sums of exp((l - m) / temperature), then of the residual
	uint64_t *top; // [n_tokens][chunks] largest logit, and its lowest index above it
	VRow *row;     // [n_tokens]
	int32_t *take; // [n_tokens] the child taken (a token row), -1: none
	int32_t *own;  // [n_tokens] the next token where none is taken
	int32_t *leaf; // [n_tokens] the next token where the children do not count
	double *res;   // [n_tokens][chunks] the residual's sums
	int *count;    // [n_tokens] rows, [n_seqs] sequences
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
	v.join = N + a.n_seqs <= (size_t)WORK_COUNTERS;
	v.count = (int *)base;
	v.s = (double *)take(N * C * 8);
	v.res = (double *)take(with_draft ? N * C * 8 : 0);
	v.top = (uint64_t *)take(N * C * 8);
	v.row = (VRow *)take(N * sizeof(VRow));
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

// exp(x) for x <= 0, to about 1e-15: 2^k times the series of exp(r), |r| <= ln 2
// / 2 (0.3466^13 / 13! < 1e-15)
__device__ __forceinline__ double exp_below(double x)
{
	const double k = __builtin_rint(x * 1.4426950408889634);
	// ln 2 in two parts: its first 32 bits, and the rest
	double r = __builtin_fma(k, -2977044471.0 / 4294967296.0, x);
	r = __builtin_fma(k, -1.90821492927058770e-10, r);
	double y = 1.0 / 479001600.0;
	y = __builtin_fma(y, r, 1.0 / 39916800.0);
	y = __builtin_fma(y, r, 1.0 / 3628800.0);
	y = __builtin_fma(y, r, 1.0 / 362880.0);
	y = __builtin_fma(y, r, 1.0 / 40320.0);
	y = __builtin_fma(y, r, 1.0 / 5040.0);
	y = __builtin_fma(y, r, 1.0 / 720.0);
	y = __builtin_fma(y, r, 1.0 / 120.0);
	y = __builtin_fma(y, r, 1.0 / 24.0);
	y = __builtin_fma(y, r, 1.0 / 6.0);
	y = __builtin_fma(y, r, 0.5);
	y = __builtin_fma(y, r, 1.0);
	y = __builtin_fma(y, r, 1.0);
	return x > -745.0 ? __builtin_amdgcn_ldexp(y, (int)k) : x != x ? x : 0.0;
}

template <typename T> __device__ __forceinline__ T wave_total(T x)
{
#pragma unroll
	for (int m = 1; m < 64; m <<= 1)
		x += __shfl_xor(x, m);
	return x;
}

// x of a lane (the same in all lanes), whether it is active here or not
__device__ __forceinline__ double of_lane(double x, int lane)
{
	const uint64_t v = (uint64_t)__double_as_longlong(x);
	const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
	return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// what one workgroup writes for another of the same launch goes past the
// dies' caches
template <typename T> __device__ __forceinline__ void give(T *p, T x)
{
	__hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T> __device__ __forceinline__ T have(const T *p)
{
	return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void give(double *p, double x)
{
	give(reinterpret_cast<uint64_t *>(p), (uint64_t)__double_as_longlong(x));
}
__device__ __forceinline__ double have(const double *p)
{
	return __longlong_as_double((long long)have(reinterpret_cast<const uint64_t *>(p)));
}

// Whether this workgroup is the last of n to arrive at a counter (which it
// leaves at 0), after all that its waves have written.
__device__ __forceinline__ bool last_of(int *count, int n, int *lds)
{
	asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
	__syncthreads();
	if (threadIdx.x == 0) {
		const int got = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
		*lds = got == n - 1;
		if (got == n - 1)
			give(count, 0);
	}
	__syncthreads();
	const bool last = *lds;
	__syncthreads();
	return last;
}

struct Shared {
	double d[4];
	float f[4];
	int i[4];
	int flag;
	int32_t path[V_PATH_LDS];
};

// the sum over the workgroup, in every thread
__device__ __forceinline__ double block_total(double x, Shared &sh)
{
	x = wave_total(x);
	__syncthreads();
	if ((threadIdx.x & 63) == 0)
		sh.d[threadIdx.x >> 6] = x;
	__syncthreads();
	return (sh.d[0] + sh.d[1]) + (sh.d[2] + sh.d[3]);
}

// The token rows [t0, t1) of row t's sequence; its number, or -1: none holds it.
__device__ __forceinline__ int seq_of_row(const VerifyArgs &a, int t, int &t0, int &t1)
{
	t0 = t;
	t1 = t + 1;
	if (!a.first)
		return t;
	int lo = 0, hi = a.n_seqs;
	while (lo < hi) {
		const int mid = (lo + hi) >> 1;
		if (a.first[mid + 1] <= t)
			lo = mid + 1;
		else
			hi = mid;
	}
	if (lo >= a.n_seqs)
		return -1;
	t0 = a.first[lo];
	t1 = a.first[lo + 1];
	return t0 >= 0 && t0 <= t && t < t1 && t1 <= a.n_tokens ? lo : -1;
}

// Whether the sequences' ranges ascend within the rows (the whole workgroup).
__device__ __forceinline__ bool ranges_good(const VerifyArgs &a)
{
	int bad = 0;
	if (a.first)
		for (int b = threadIdx.x; b < a.n_seqs; b += blockDim.x)
			bad |= a.first[b] < 0 || a.first[b] > a.first[b + 1] || a.first[b + 1] > a.n_tokens;
	return !__syncthreads_or(bad);
}

// The path of sequence b, rows [t0, t1): a workgroup; the outcomes through LDS.
__device__ void write_path(const VerifyArgs &a, const VerifyWork &w, int b, int t0, int t1, Shared &sh)
{
	int32_t *path = a.path + (size_t)b * a.max_path;
	const int n = t1 - t0;
	for (int i = threadIdx.x; i < n && i < V_PATH_LDS; i += blockDim.x)
		sh.path[i] = have(w.take + t0 + i);
	__syncthreads();
	if (threadIdx.x == 0) {
		int t = t0, k = 0, next = -1;
		while (n > 0) {
			path[k++] = t - t0;
			if (k >= a.max_path) {
				next = have(w.leaf + t); // (its children were never to be tried)
				break;
			}
			const int kid = t - t0 < V_PATH_LDS ? sh.path[t - t0] : have(w.take + t);
			if (kid < 0) {
				next = have(w.own + t);
				break;
			}
			t = kid; // (a later row of the same sequence)
		}
		a.n_keep[b] = k;
		a.next[b] = next;
		sh.flag = k;
	}
	__syncthreads();
	for (int i = sh.flag + threadIdx.x; i < a.max_path; i += blockDim.x)
		path[i] = -1;
}

// The first index whose running weight exceeds u times the whole: over the
// chunks' sums (sum(c): of chunk c), then inside the chunk (weight(i) >= 0).
template <typename W, typename S>
__device__ __forceinline__ int locate(const VerifyArgs &a, int chunks, double u, W weight, S sum, Shared &sh)
{
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	// (every wave for itself: a lane a chunk)
	double all = 0.0;
	int last = 0;
	for (int c0 = 0; c0 < chunks; c0 += 64) {
		const double x = c0 + lane < chunks ? sum(c0 + lane) : 0.0;
		const unsigned long long some = __ballot(x > 0.0);
		if (some)
			last = c0 + 63 - __builtin_clzll(some);
		all += wave_total(x);
	}
	const double want = u * all;
	double before = 0.0, upto = 0.0;
	int at = -1;
	for (int c0 = 0; c0 < chunks && at < 0; c0 += 64) {
		const double x = c0 + lane < chunks ? sum(c0 + lane) : 0.0;
		double incl = x;
#pragma unroll
		for (int m = 1; m < 64; m <<= 1) {
			const double o = __shfl_up(incl, m);
			if (lane >= m)
				incl += o;
		}
		const unsigned long long over = __ballot(upto + incl > want && c0 + lane < chunks);
		const int l = over ? __builtin_ctzll(over) : last - c0; // (for the fallback: the last chunk of any weight)
		if (over || (last >= c0 && last < c0 + 64)) {
			before = upto + __shfl(incl - x, l & 63);
			if (over)
				at = c0 + l;
		}
		upto += __shfl(incl, 63);
	}
	if (at < 0)
		at = last; // (u of one, or a rounding at the end)
	// thread i has V_E weights in a row
	const int base = at * V_CHUNK + threadIdx.x * V_E;
	double x[V_E], mine = 0.0;
#pragma unroll
	for (int e = 0; e < V_E; e++) {
		x[e] = base + e < a.vocab ? weight(base + e) : 0.0;
		mine += x[e];
	}
	double incl = mine;
#pragma unroll
	for (int m = 1; m < 64; m <<= 1) {
		const double o = __shfl_up(incl, m);
		if (lane >= m)
			incl += o;
	}
	__syncthreads();
	if (lane == 63)
		sh.d[wave] = incl;
	if (threadIdx.x == 0)
		sh.i[0] = 0x7fffffff, sh.i[1] = 0;
	__syncthreads();
	double run = before + incl - mine;
	for (int q = 0; q < wave; q++)
		run += sh.d[q];
	int first = 0x7fffffff, some = -1;
#pragma unroll
	for (int e = 0; e < V_E; e++) {
		run += x[e];
		if (x[e] > 0.0) {
			some = base + e;
			if (run > want && first == 0x7fffffff)
				first = base + e;
		}
	}
	if (first != 0x7fffffff)
		atomicMin(&sh.i[0], first);
	if (some >= 0)
		atomicMax(&sh.i[1], some);
	__syncthreads();
	const int got = sh.i[0] < a.vocab ? sh.i[0] : sh.i[1];
	__syncthreads();
	return got;
}

// Row t's outcome as far as the sums so far carry it: the largest logit and the
// whole (pass 0), its children in turn, the next token; and, of the sequence's
// last row, the path.  The whole workgroup, all of it uniform.
__device__ void row_step(const VerifyArgs &a, const VerifyWork &w, int t, int pass, Shared &sh)
{
	const int lane = threadIdx.x & 63;
	int t0, t1;
	const int b = seq_of_row(a, t, t0, t1);
	if (b < 0)
		return;
	const double inv = a.temperature > 0.0f ? 1.0 / (double)a.temperature : 0.0;
	const double *s = w.s + (size_t)t * w.chunks, *res = w.res + (size_t)t * w.chunks;
	const uint64_t *top = w.top + (size_t)t * w.chunks;
	VRow r;
	if (pass == 0) {
		r.m = -__builtin_inff();
		r.best = 0x7fffffff;
		for (int c0 = 0; c0 < w.chunks; c0 += 64) {
			if (c0 + lane < w.chunks) {
				const uint64_t v = have(top + c0 + lane);
				const float m = __uint_as_float((uint32_t)v);
				if (m > r.m) {
					r.m = m;
					r.best = (int)(v >> 32);
				}
			}
		}
#pragma unroll
		for (int q = 1; q < 64; q <<= 1) {
			const float om = __shfl_xor(r.m, q);
			const int oi = __shfl_xor(r.best, q);
			if (om > r.m || (om == r.m && oi < r.best)) {
				r.m = om;
				r.best = oi;
			}
		}
		if (r.best >= a.vocab)
			r.best = 0;
		double z = 0.0;
		if (a.temperature > 0.0f)
			for (int c = lane; c < w.chunks; c += 64) {
				const float m = __uint_as_float((uint32_t)have(top + c));
				if (m > -__builtin_inff())
					z += have(s + c) * exp_below(((double)m - (double)r.m) * inv);
			}
		r.scale = 1.0 / wave_total(z);
		r.c = 0.0;
		r.M = 1.0;
		r.kid = 0;
		r.waits = -1;
	} else {
		r = w.row[t];
		double M = 0.0;
		for (int c = lane; c < w.chunks; c += 64)
			M += have(res + c);
		r.M = wave_total(M);
		r.waits = -1;
	}
	const float *l = a.logits + (size_t)t * a.l_stride, *q = a.draft ? a.draft + (size_t)t * a.d_stride : nullptr;
	auto p_of = [&](float x) { return exp_below(((double)x - (double)r.m) * inv) * r.scale; };

	// the children: later rows of the sequence whose parent this is; lane i has
	// the i-th
	int n = 0, kid = -1;
	for (int j0 = t + 1; j0 < t1 && n < a.max_children; j0 += 64) {
		const int j = j0 + lane;
		unsigned long long set = __ballot(j < t1 && a.parent[j < t1 ? j : t] == t - t0);
		while (set && n < a.max_children) {
			if (lane == n)
				kid = j0 + __builtin_ctzll(set);
			set &= set - 1;
			n++;
		}
	}
	int x = -1;
	double px = 0.0, qx = 1.0, u = 0.0;
	if (kid >= 0) {
		x = a.tokens[kid];
		u = (double)a.u_accept[kid];
		if (x >= 0 && x < a.vocab && a.temperature > 0.0f) {
			px = p_of(l[x]);
			if (q)
				qx = (double)q[x];
		}
	}
	int taken = -1;
	unsigned long long gone = 0; // no draft rows: refused children
	for (int i = r.kid; i < n; i++) {
		const int xi = __builtin_amdgcn_readlane(x, i);
		if (xi < 0 || xi >= a.vocab)
			continue; // no token: not tried
		if (a.temperature == 0.0f) {
			if (xi == r.best) {
				taken = __builtin_amdgcn_readlane(kid, i);
				break;
			}
			continue;
		}
		const double pi = of_lane(px, i), qi = of_lane(qx, i), ui = of_lane(u, i);
		if (q) {
			const double left = pi - r.c * qi;
			if (ui * r.M * qi < (left > 0.0 ? left : 0.0)) {
				taken = __builtin_amdgcn_readlane(kid, i);
				break;
			}
			r.c += r.M;
			r.kid = i + 1;
			r.waits = pass;
			break;
		}
		if (__ballot(x == xi) & gone)
			continue; // (left p with an earlier child)
		if (ui * r.M < pi) {
			taken = __builtin_amdgcn_readlane(kid, i);
			break;
		}
		gone |= 1ull << i;
		r.M -= pi;
	}
	if (r.waits >= 0) {
		if (threadIdx.x == 0)
			w.row[t] = r; // (for the next launch)
		return;
	}
	if (pass == 0 && threadIdx.x == 0)
		w.row[t].waits = -1;

	int own = r.best, leaf = r.best;
	if (a.temperature > 0.0f) {
		auto p_sum = [&](int c) {
			const float m = __uint_as_float((uint32_t)have(top + c));
			return m > -__builtin_inff() ? have(s + c) * exp_below(((double)m - (double)r.m) * inv) * r.scale : 0.0;
		};
		auto p_at = [&](int i) { return p_of(l[i]); };
		const double us = (double)a.u_sample[t];
		const bool cut = a.max_path < t1 - t0; // a path may end at any node
		const bool plain = (r.c == 0.0 && !gone) || !(r.M > 0.0);
		if ((taken < 0 && plain) || (cut && n > 0))
			own = leaf = locate(a, w.chunks, us, p_at, p_sum, sh);
		if (taken < 0 && !plain && q)
			own = locate(
				a, w.chunks, us,
				[&](int i) {
					const double y = p_of(l[i]) - r.c * (double)q[i];
					return y > 0.0 ? y : 0.0;
				},
				[&](int c) { return have(res + c); }, sh);
		else if (taken < 0 && !plain)
			own = locate(
				a, w.chunks, us,
				[&](int i) {
					double y = p_of(l[i]);
					for (unsigned long long g = gone; g; g &= g - 1)
						if (__builtin_amdgcn_readlane(x, __builtin_ctzll(g)) == i)
							y = 0.0;
					return y;
				},
				[&](int c) {
					double y = c < w.chunks ? p_sum(c) : 0.0;
					for (unsigned long long g = gone; g; g &= g - 1) {
						const int k = __builtin_ctzll(g);
						if (__builtin_amdgcn_readlane(x, k) / V_CHUNK == c)
							y -= of_lane(px, k);
					}
					return y > 0.0 ? y : 0.0;
				},
				sh);
		if (n == 0)
			leaf = own;
	}
	if (threadIdx.x == 0) {
		give(w.take + t, taken);
		give(w.own + t, own);
		give(w.leaf + t, leaf);
	}
	if (!w.join || !ranges_good(a))
		return;
	if (last_of(w.count + a.n_tokens + b, t1 - t0, &sh.flag))
		write_path(a, w, b, t0, t1, sh);
}

// The first launch: largest logit and sum of each chunk.
__global__ __launch_bounds__(V_THREADS) void verify_stats_kernel(VerifyArgs a, VerifyWork w)
{
	__shared__ Shared sh;
	const int t = blockIdx.y, chunk = blockIdx.x, base = chunk * V_CHUNK;
	const float *l = a.logits + (size_t)t * a.l_stride;
	float x[V_E];
	if (base + V_CHUNK <= a.vocab && ((uintptr_t)(l + base) & 15) == 0) {
#pragma unroll
		for (int e = 0; e < V_E; e += 4) {
			const float4 v = reinterpret_cast<const float4 *>(l + base)[e / 4 * V_THREADS + threadIdx.x];
			x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
		}
	} else {
#pragma unroll
		for (int e = 0; e < V_E; e++) {
			const int i = base + (e / 4 * V_THREADS + threadIdx.x) * 4 + e % 4;
			x[e] = i < a.vocab ? l[i] : -__builtin_inff();
		}
	}
	float m = -__builtin_inff();
	int at = 0x7fffffff;
#pragma unroll
	for (int e = 0; e < V_E; e++)
		if (x[e] > m) {
			m = x[e];
			at = base + (e / 4 * V_THREADS + threadIdx.x) * 4 + e % 4;
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
		sh.f[threadIdx.x >> 6] = m;
		sh.i[threadIdx.x >> 6] = at;
	}
	__syncthreads();
#pragma unroll
	for (int q = 0; q < 4; q++)
		if (sh.f[q] > m || (sh.f[q] == m && sh.i[q] < at)) {
			m = sh.f[q];
			at = sh.i[q];
		}
	double s = 0.0;
	if (a.temperature > 0.0f && m > -__builtin_inff()) {
		const double inv = 1.0 / (double)a.temperature;
#pragma unroll
		for (int e = 0; e < V_E; e++)
			s += exp_below(((double)x[e] - (double)m) * inv);
		s = block_total(s, sh);
	}
	if (threadIdx.x == 0) {
		const size_t o = (size_t)t * w.chunks + chunk;
		give(w.top + o, (uint64_t)__float_as_uint(m) | (uint64_t)(uint32_t)at << 32);
		give(w.s + o, s);
	}
	if (w.join) {
		// sequences of no rows have nobody to arrive; ranges that do not ascend
		// have no paths
		if (t == 0 && chunk == 0) {
			const bool good = ranges_good(a);
			for (int b = threadIdx.x; b < a.n_seqs; b += V_THREADS)
				if (!good || (a.first && a.first[b] == a.first[b + 1])) {
					for (int i = 0; i < a.max_path; i++)
						a.path[(size_t)b * a.max_path + i] = -1;
					a.n_keep[b] = 0;
					a.next[b] = -1;
				}
		}
		if (last_of(w.count + t, w.chunks, &sh.flag))
			row_step(a, w, t, 0, sh);
	}
}

// One more residual sum for the rows that wait for it.
__global__ __launch_bounds__(V_THREADS) void verify_residual_kernel(VerifyArgs a, VerifyWork w, int pass)
{
	__shared__ Shared sh;
	const int t = blockIdx.y, base = blockIdx.x * V_CHUNK;
	if (w.row[t].waits != pass)
		return;
	const VRow r = w.row[t];
	const double inv = 1.0 / (double)a.temperature;
	const float *l = a.logits + (size_t)t * a.l_stride, *q = a.draft + (size_t)t * a.d_stride;
	double s = 0.0;
#pragma unroll
	for (int e = 0; e < V_E; e++) {
		const int i = base + e * V_THREADS + threadIdx.x;
		const bool in = i < a.vocab;
		const float li = in ? l[i] : -__builtin_inff(), qi = in ? q[i] : 0.0f;
		const double y = exp_below(((double)li - (double)r.m) * inv) * r.scale - r.c * (double)qi;
		s += y > 0.0 ? y : 0.0;
	}
	s = block_total(s, sh);
	if (threadIdx.x == 0)
		give(w.res + (size_t)t * w.chunks + blockIdx.x, s);
	if (w.join && last_of(w.count + t, w.chunks, &sh.flag))
		row_step(a, w, t, pass + 1, sh);
}

// More rows and sequences than there are counters: the steps as launches.
__global__ __launch_bounds__(V_THREADS) void verify_row_kernel(VerifyArgs a, VerifyWork w, int pass)
{
	__shared__ Shared sh;
	if (pass && w.row[blockIdx.x].waits != pass - 1)
		return;
	row_step(a, w, blockIdx.x, pass, sh);
}

__global__ __launch_bounds__(V_THREADS) void verify_path_kernel(VerifyArgs a, VerifyWork w)
{
	__shared__ Shared sh;
	const bool good = ranges_good(a);
	const int b = blockIdx.x, t0 = a.first ? a.first[b] : b, t1 = a.first ? a.first[b + 1] : b + 1;
	write_path(a, w, b, good ? t0 : 0, good ? t1 : 0, sh);
}

hipError_t launch_verify(const VerifyArgs &a, void *work, hipStream_t st)
{
	VerifyWork w;
	carve_verify(a, a.draft != nullptr, (uint8_t *)work, &w);
	const dim3 grid(w.chunks, a.n_tokens), block(V_THREADS);
	const int passes = a.draft && a.temperature > 0.0f ? a.max_children : 0;
	if (a.n_tokens > 0) {
		tie_launch(verify_stats_kernel, grid, block, 0, st, a, w);
		if (!w.join)
			tie_launch(verify_row_kernel, dim3(a.n_tokens), block, 0, st, a, w, 0);
		for (int p = 0; p < passes; p++) {
			tie_launch(verify_residual_kernel, grid, block, 0, st, a, w, p);
			if (!w.join)
				tie_launch(verify_row_kernel, dim3(a.n_tokens), block, 0, st, a, w, p + 1);
		}
	}
	if (!w.join || a.n_tokens == 0)
		tie_launch(verify_path_kernel, dim3(a.n_seqs), block, 0, st, a, w);
	return hipGetLastError();
}

} // namespace tie
