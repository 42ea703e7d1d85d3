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
// nodes are worked on at once, a workgroup to one or two V_CHUNK logits, and the
// path is read off at the end.  The last workgroup of a row forms the row's outcome, the
// last row of a sequence its path: one launch, and one more for each residual
// sum that some row may need, for the rows that the path can still reach.  Sums are in 64
// bits: the running sum crosses u M at the same token whatever the order of the
// sum.
#include "kv.h"

namespace tie {

constexpr int V_CHUNK = 4096; // logits of a workgroup
constexpr int V_THREADS = 256, V_E = V_CHUNK / V_THREADS;
constexpr size_t V_AT_ONCE = 1024; // workgroups that run together: 4 on a CU
constexpr int V_PATH_LDS = 512; // nodes of a sequence whose outcomes the path's reader keeps in LDS

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
	int32_t *act;  // [n_tokens] draft rows: the residual sum that the row takes part in
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
	v.act = (int32_t *)take(with_draft ? N * 4 : 0);
	if (w)
		*w = v;
	return off;
}

size_t verify_work_bytes(const VerifyArgs &a, bool with_draft)
{
	return carve_verify(a, with_draft, nullptr, nullptr);
}

// 2^(j / 16), which every workgroup copies to LDS (16 entries: a wave's lanes
// read them without bank conflicts)
__constant__ const double POW16[16] = {
	1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
	1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
	1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
	1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

// exp(x inv) = 2^(t / 16) with t = x EXP16 inv, x <= 0: 2^k of the table's
// entry and the series of 2^(r / 16), |r| <= 1 / 2 (0.0217^7 / 7! = 5e-16).  A
// series alone takes twice the steps.
constexpr double EXP16 = 16.0 * 1.4426950408889634;
__device__ __forceinline__ double pow16(double t, const double *tab)
{
	constexpr double L = 0.69314718055994531 / 16.0;
	const double s = t + 6755399441055744.0; // 1.5 2^52: the nearest integer, in the low bits
	const int n = (int)(uint32_t)(uint64_t)__double_as_longlong(s);
	const double r = t - (s - 6755399441055744.0);
	double y = L * L * L * L * L * L / 720.0;
	y = __builtin_fma(y, r, L * L * L * L * L / 120.0);
	y = __builtin_fma(y, r, L * L * L * L / 24.0);
	y = __builtin_fma(y, r, L * L * L / 6.0);
	y = __builtin_fma(y, r, L * L / 2.0);
	y = __builtin_fma(y, r, L);
	y = __builtin_fma(y, r, 1.0);
	y = __builtin_amdgcn_ldexp(y * tab[n & 15], n >> 4);
	return t < -17400.0 ? 0.0 : y; // (NaN stays NaN)
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
	int i[4], j[4];
	int flag;
	double pow[16];
	int32_t path[V_PATH_LDS], own[V_PATH_LDS], leaf[V_PATH_LDS], parent[V_PATH_LDS];

	__device__ __forceinline__ void fill() // (a barrier before its use)
	{
		if (threadIdx.x < 16)
			pow[threadIdx.x] = POW16[threadIdx.x];
	}
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
// A wave: the sequences' ends a lane each, after bisection down to 64 of them.
// good: whether all ranges ascend within the rows, as far as the wave has seen
// (all of them up to 64; else ranges_good has to look).
__device__ __forceinline__ int seq_of_row(const VerifyArgs &a, int t, int &t0, int &t1, bool &good)
{
	t0 = t;
	t1 = t + 1;
	good = true;
	if (!a.first)
		return t;
	int lo = 0, hi = a.n_seqs;
	while (hi - lo > 64) {
		const int mid = (lo + hi) >> 1;
		if (a.first[mid] <= t)
			lo = mid;
		else
			hi = mid;
	}
	// the last b in [lo, hi) with first[b] <= t (of equal ones the last: the others hold nothing)
	const int lane = threadIdx.x & 63, b = lo + lane;
	const int from = b < hi ? a.first[b] : 0x7fffffff, to = b < hi ? a.first[b + 1] : 0;
	good = !__ballot(b < hi && (from < 0 || from > to || to > a.n_tokens));
	const unsigned long long below = __ballot(from <= t);
	if (!below)
		return -1;
	const int l = 63 - __builtin_clzll(below);
	t0 = __builtin_amdgcn_readlane(from, l);
	t1 = __builtin_amdgcn_readlane(to, l);
	return t0 >= 0 && t < t1 && t1 <= a.n_tokens ? lo + l : -1;
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

// The outcomes of rows [t0, t1) into LDS, as many as it holds (a workgroup).
__device__ void get_outcomes(const VerifyArgs &a, const VerifyWork &w, int t0, int t1, Shared &sh)
{
	for (int i = threadIdx.x; i < t1 - t0 && i < V_PATH_LDS; i += blockDim.x) {
		sh.path[i] = have(w.take + t0 + i);
		sh.own[i] = have(w.own + t0 + i);
		sh.leaf[i] = have(w.leaf + t0 + i);
		sh.parent[i] = a.parent[t0 + i];
	}
	__syncthreads();
}

// The path of sequence b, rows [t0, t1): a workgroup.
__device__ void write_path(const VerifyArgs &a, const VerifyWork &w, int b, int t0, int t1, Shared &sh)
{
	int32_t *path = a.path + (size_t)b * a.max_path;
	const int n = t1 - t0;
	if (threadIdx.x == 0) {
		int t = t0, k = 0, next = -1;
		while (n > 0) {
			const int i = t - t0;
			path[k++] = i;
			if (k >= a.max_path) {
				// (its children were never to be tried)
				next = i < V_PATH_LDS ? sh.leaf[i] : have(w.leaf + t);
				break;
			}
			const int kid = i < V_PATH_LDS ? sh.path[i] : have(w.take + t);
			if (kid < 0) {
				next = i < V_PATH_LDS ? sh.own[i] : have(w.own + t);
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

// All rows of sequence b have arrived with an outcome, or with the child they
// refused last (take = -2 - its row) and a residual sum to wait for: the path, or
// which of the waiting rows the next launch works on.  A row that the path
// cannot reach any more is left: an ancestor took another child, none, or
// refused the one on the way here.
__device__ void settle(const VerifyArgs &a, const VerifyWork &w, int b, int t0, int t1, int pass, Shared &sh)
{
	const int n = t1 - t0;
	get_outcomes(a, w, t0, t1, sh);
	int waiting = 0;
	for (int i0 = 0; i0 < n; i0 += V_THREADS) {
		const int i = i0 + threadIdx.x;
		const int take = i >= n ? -1 : i < V_PATH_LDS ? sh.path[i] : have(w.take + t0 + i);
		bool act = take <= -2;
		if (n <= V_PATH_LDS)
			for (int j = i; act && j > 0;) {
				const int up = sh.parent[j];
				act = up >= 0 && up < j;
				if (act) {
					const int of_up = sh.path[up];
					act = of_up >= -1 ? of_up == t0 + j : t0 + j > -2 - of_up;
					j = up;
				}
			}
		if (a.draft && i < n)
			give(w.act + t0 + i, act ? pass : -1);
		waiting += __syncthreads_count(act);
	}
	if (waiting == 0)
		write_path(a, w, b, t0, t1, sh);
	else if (threadIdx.x == 0)
		give(w.count + a.n_tokens + b, n - waiting); // (the others are there already)
}

// The first index whose running weight exceeds u times the whole: over the
// chunks' sums (lane_sum: of the first 64, a lane each; sum(c) of the others),
// then inside the chunk: weights(i0, w) gives the V_E weights from i0 on (>= 0).
// A workgroup, once for a row: what bounds it is the chain of its steps.
template <typename W, typename S>
__device__ __forceinline__ int locate(const VerifyArgs &a, int chunks, double u, double lane_sum, W weights, S sum, Shared &sh)
{
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	double all = wave_total(lane_sum);
	const unsigned long long some0 = __ballot(lane_sum > 0.0);
	int last = some0 ? 63 - __builtin_clzll(some0) : 0;
	for (int c0 = 64; c0 < chunks; c0 += 64) {
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
		const double x = c0 == 0 ? lane_sum : c0 + lane < chunks ? sum(c0 + lane) : 0.0;
		const double incl = running_of<64>(x);
		const unsigned long long over = __ballot(upto + incl > want && c0 + lane < chunks);
		const int l = over ? __builtin_ctzll(over) : last - c0; // (for the fallback: the last chunk of any weight)
		if (over || (last >= c0 && last < c0 + 64)) {
			before = upto + of_lane(incl - x, l & 63);
			if (over)
				at = c0 + l;
		}
		upto += of_lane(incl, 63);
	}
	if (at < 0)
		at = last; // (u of one, or a rounding at the end)
	const int i0 = at * V_CHUNK + threadIdx.x * V_E;
	double w[V_E], mine = 0.0;
	weights(i0, w);
	int some = 0; // the last of the thread's indexes with a weight, + 1
#pragma unroll
	for (int e = 0; e < V_E; e++) {
		mine += w[e];
		some = w[e] > 0.0 ? e + 1 : some;
	}
	const double incl = running_of<64>(mine);
	__syncthreads();
	if (lane == 63)
		sh.d[wave] = incl;
	__syncthreads();
	for (int q = 0; q < wave; q++)
		before += sh.d[q];
	// the first thread whose weights pass `want`; where none does, the last
	// that has any
	const unsigned long long over = __ballot(before + incl > want), any = __ballot(some > 0);
	if (lane == 0) {
		sh.i[wave] = over ? wave * 64 + __builtin_ctzll(over) : V_THREADS;
		sh.j[wave] = any ? wave * 64 + 63 - __builtin_clzll(any) : 0;
	}
	__syncthreads();
	int owner = V_THREADS, end = 0;
#pragma unroll
	for (int q = 0; q < V_THREADS / 64; q++) {
		owner = min(owner, sh.i[q]);
		end = max(end, sh.j[q]);
	}
	owner = owner < V_THREADS ? owner : end;
	if ((int)threadIdx.x == owner) {
		double run = before + incl - mine;
		int e0 = some > 0 ? some - 1 : 0; // (a rounding between the two sums: its last weight)
#pragma unroll
		for (int e = 0; e < V_E; e++) {
			run += w[e];
			e0 = run > want && w[e] > 0.0 && e < e0 ? e : e0;
		}
		sh.flag = i0 + e0;
	}
	__syncthreads();
	const int got = sh.flag;
	__syncthreads();
	return got < a.vocab ? got : 0;
}

// V_E values of a row from i0 on, `none` behind its end
__device__ __forceinline__ void get_run(const float *row, int i0, int n, float none, float (&x)[V_E])
{
	if (i0 + V_E <= n && ((uintptr_t)row & 15) == 0) {
#pragma unroll
		for (int e = 0; e < V_E; e += 4) {
			const float4 v = reinterpret_cast<const float4 *>(row + i0)[e / 4];
			x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
		}
	} else {
#pragma unroll
		for (int e = 0; e < V_E; e++)
			x[e] = i0 + e < n ? row[i0 + e] : none;
	}
}

// Row t's outcome as far as the sums so far carry it: the largest logit and the
// whole (pass 0), its children in turn, the next token; and, of the sequence's
// last row, the path.  The whole workgroup, all of it uniform.
__device__ void row_step(const VerifyArgs &a, const VerifyWork &w, int t, int pass, Shared &sh)
{
	const int lane = threadIdx.x & 63;
	int t0, t1;
	bool good;
	const int b = seq_of_row(a, t, t0, t1, good);
	if (b < 0)
		return;
	// (no row of such a call has what a later pass would read)
	if (w.join && (!good || (a.n_seqs > 64 && !ranges_good(a))))
		return;
	const double rate = a.temperature > 0.0f ? EXP16 / (double)a.temperature : 0.0;
	const double *s = w.s + (size_t)t * w.chunks, *res = w.res + (size_t)t * w.chunks;
	const uint64_t *top = w.top + (size_t)t * w.chunks;
	const float *l = a.logits + (size_t)t * a.l_stride, *q = a.draft ? a.draft + (size_t)t * a.d_stride : nullptr;
	// all that the first steps need is requested at once: the first 64 chunks'
	// sums, the 64 rows behind this one (its children are among them, mostly)
	const float us = a.u_sample[t];
	uint64_t top0 = 0;
	double s0 = 0.0, r0 = 0.0;
	if (lane < w.chunks) {
		top0 = have(top + lane);
		s0 = have(s + lane);
		if (pass)
			r0 = have(res + lane);
	}
	const int j1 = min(t + 1 + lane, a.n_tokens - 1);
	const int parent1 = a.parent[j1], token1 = a.tokens[j1];
	const float u1 = a.u_accept[j1];

	// the children: later rows of the sequence whose parent this is; lane i has
	// the i-th
	int n = 0, kid = -1, x = -1;
	float uf = 0.0f;
	for (int j0 = t + 1; j0 < t1 && n < a.max_children; j0 += 64) {
		const int j = j0 + lane;
		const bool near = j0 == t + 1;
		unsigned long long set = __ballot(j < t1 && (near ? parent1 : a.parent[j < t1 ? j : t]) == t - t0);
		while (set && n < a.max_children) {
			const int from = __builtin_ctzll(set);
			const int xi = near ? __builtin_amdgcn_readlane(token1, from) : a.tokens[j0 + from];
			const float ui = near ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, u1), from)) : a.u_accept[j0 + from];
			if (lane == n) {
				kid = j0 + from;
				x = xi;
				uf = ui;
			}
			set &= set - 1;
			n++;
		}
	}
	// (their logits and draft probabilities, on the way while the sums are joined)
	const bool is_token = kid >= 0 && x >= 0 && x < a.vocab;
	const float lx = is_token ? l[x] : 0.0f;
	const double qx = is_token && q ? (double)q[x] : 1.0, u = (double)uf;

	VRow r;
	double z0 = 0.0; // lane c: the whole of chunk c, times exp(largest of all)
	if (pass == 0) {
		r.m = lane < w.chunks ? __uint_as_float((uint32_t)top0) : -__builtin_inff();
		r.best = lane < w.chunks ? (int)(top0 >> 32) : 0x7fffffff;
		for (int c = 64 + lane; c < w.chunks; c += 64) {
			const uint64_t v = have(top + c);
			const float m = __uint_as_float((uint32_t)v);
			if (m > r.m) {
				r.m = m;
				r.best = (int)(v >> 32);
			}
		}
		const float most = wave_max(r.m);
		if (a.temperature == 0.0f) {
			r.best = r.m == most ? r.best : 0x7fffffff;
#pragma unroll
			for (int k = 1; k < 64; k <<= 1)
				r.best = min(r.best, __shfl_xor(r.best, k));
		}
		r.m = most;
		if (r.best < 0 || r.best >= a.vocab)
			r.best = 0;
	} else {
		r = w.row[t];
	}
	auto whole_of = [&](uint64_t v, double sum) {
		const float m = __uint_as_float((uint32_t)v);
		return m > -__builtin_inff() ? sum * pow16(((double)m - (double)r.m) * rate, sh.pow) : 0.0;
	};
	if (a.temperature > 0.0f && lane < w.chunks)
		z0 = whole_of(top0, s0);
	if (pass == 0) {
		double z = z0;
		if (a.temperature > 0.0f)
			for (int c = 64 + lane; c < w.chunks; c += 64)
				z += whole_of(have(top + c), have(s + c));
		r.scale = 1.0 / wave_total(z);
		r.c = 0.0;
		r.M = 1.0;
		r.kid = 0;
	} else {
		double M = r0;
		for (int c = 64 + lane; c < w.chunks; c += 64)
			M += have(res + c);
		r.M = wave_total(M);
	}
	r.waits = -1;
	auto p_of = [&](float y) { return pow16(((double)y - (double)r.m) * rate, sh.pow) * r.scale; };
	const double px = is_token && a.temperature > 0.0f ? p_of(lx) : 0.0;

	int taken = -1, refused = 0;
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
			refused = __builtin_amdgcn_readlane(kid, i);
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
	if (threadIdx.x == 0) {
		if (r.waits >= 0)
			w.row[t] = r; // (for the next launch)
		else if (!w.join)
			w.row[t].waits = -1;
	}

	int own = r.best, leaf = r.best;
	if (a.temperature > 0.0f && r.waits < 0) {
		auto p_sum = [&](int c) { return whole_of(have(top + c), have(s + c)) * r.scale; };
		const bool cut = a.max_path < t1 - t0; // a path may end at any node
		const bool plain = (r.c == 0.0 && !gone) || !(r.M > 0.0);
		auto without = [&](int c, double y) { // of chunk c: less what left p
			for (unsigned long long g = gone; g; g &= g - 1) {
				const int k = __builtin_ctzll(g);
				if (__builtin_amdgcn_readlane(x, k) / V_CHUNK == c)
					y -= of_lane(px, k);
			}
			return y > 0.0 ? y : 0.0;
		};
#pragma unroll 1
		for (int what = 0; what < 2; what++) {
			if (what == 0 ? taken >= 0 : !(cut && n > 0))
				continue;
			const bool of_p = what == 1 || plain;
			const double c_q = of_p || !q ? 0.0 : r.c;
			const unsigned long long out = of_p ? 0 : gone;
			const int got = locate(
				a, w.chunks, (double)us, c_q > 0.0 ? r0 : out ? without(lane, z0 * r.scale) : z0 * r.scale,
				[&](int i0, double (&y)[V_E]) {
					float li[V_E], qi[V_E];
					get_run(l, i0, a.vocab, -__builtin_inff(), li);
					if (c_q > 0.0)
						get_run(q, i0, a.vocab, 0.0f, qi);
#pragma unroll
					for (int e = 0; e < V_E; e++)
						y[e] = p_of(li[e]);
					if (c_q > 0.0)
#pragma unroll
						for (int e = 0; e < V_E; e++)
							y[e] -= c_q * (double)qi[e];
					for (unsigned long long g = out; g; g &= g - 1) {
						const int away = __builtin_amdgcn_readlane(x, __builtin_ctzll(g)) - i0;
#pragma unroll
						for (int e = 0; e < V_E; e++)
							y[e] = away == e ? 0.0 : y[e];
					}
#pragma unroll
					for (int e = 0; e < V_E; e++)
						y[e] = y[e] > 0.0 ? y[e] : 0.0;
				},
				[&](int c) { return c_q > 0.0 ? have(res + c) : out ? without(c, p_sum(c)) : p_sum(c); }, sh);
			if (what == 0)
				own = got;
			else
				leaf = got;
		}
		if (n == 0)
			leaf = own;
	}
	if (threadIdx.x == 0) {
		give(w.take + t, r.waits >= 0 ? -2 - refused : taken);
		give(w.own + t, own);
		give(w.leaf + t, leaf);
	}
	if (!w.join)
		return;
	if (last_of(w.count + a.n_tokens + b, t1 - t0, &sh.flag))
		settle(a, w, b, t0, t1, pass, sh);
}

// A workgroup's logits (or draft probabilities): four at a time to a thread
__device__ __forceinline__ void get_chunk(const float *row, int base, int n, float none, float (&x)[V_E])
{
	if (base + V_CHUNK <= n && ((uintptr_t)(row + base) & 15) == 0) {
#pragma unroll
		for (int e = 0; e < V_E; e += 4) {
			const float4 v = reinterpret_cast<const float4 *>(row + base)[e / 4 * V_THREADS + threadIdx.x];
			x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
		}
	} else {
#pragma unroll
		for (int e = 0; e < V_E; e++) {
			const int i = base + (e / 4 * V_THREADS + threadIdx.x) * 4 + e % 4;
			x[e] = i < n ? row[i] : none;
		}
	}
}

// The first launch: largest logit and sum of each chunk; a workgroup PER chunks,
// whose logits are under way together.  57 rows of 151936 logits (35 MB): 23 us, of
// which the sums are 15 (bound by the 64-bit exponentials and the loads in turn)
// and the last rows' steps 8; one chunk each 30.6.  5 rows of 32000: 12 us, 4.5 to
// the sums and then the chain of a row's steps (children, the next token's search,
// the sequence's count, the path).
template <int PER>
__global__ __launch_bounds__(V_THREADS, 4) void verify_stats_kernel(VerifyArgs a, VerifyWork w)
{
	__shared__ Shared sh;
	__shared__ float fs[PER][4];
	__shared__ double ds[PER][4];
	__shared__ int is[PER][4];
	const int t = blockIdx.y, chunk = blockIdx.x * PER, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
	const float *l = a.logits + (size_t)t * a.l_stride;
	float x[PER][V_E], m[PER];
	sh.fill();
#pragma unroll
	for (int q = 0; q < PER; q++)
		get_chunk(l, (chunk + q) * V_CHUNK, a.vocab, -__builtin_inff(), x[q]);
#pragma unroll
	for (int q = 0; q < PER; q++) {
		m[q] = x[q][0];
#pragma unroll
		for (int e = 1; e < V_E; e++)
			m[q] = __builtin_fmaxf(m[q], x[q][e]);
		m[q] = wave_max(m[q]);
		if (lane == 0)
			fs[q][wave] = m[q];
	}
	__syncthreads();
#pragma unroll
	for (int q = 0; q < PER; q++)
		m[q] = __builtin_fmaxf(__builtin_fmaxf(fs[q][0], fs[q][1]), __builtin_fmaxf(fs[q][2], fs[q][3]));
	if (a.temperature == 0.0f) { // its lowest index
#pragma unroll
		for (int q = 0; q < PER; q++) {
			int at = 0x7fffffff;
#pragma unroll
			for (int e = V_E - 1; e >= 0; e--)
				at = x[q][e] == m[q] ? (chunk + q) * V_CHUNK + (e / 4 * V_THREADS + (int)threadIdx.x) * 4 + e % 4 : at;
#pragma unroll
			for (int k = 1; k < 64; k <<= 1)
				at = min(at, __shfl_xor(at, k));
			if (lane == 0)
				is[q][wave] = at;
		}
	} else {
		const double rate = EXP16 / (double)a.temperature;
#pragma unroll
		for (int q = 0; q < PER; q++) {
			double s = 0.0;
			if (m[q] > -__builtin_inff())
#pragma unroll
				for (int e = 0; e < V_E; e++)
					s += pow16(((double)x[q][e] - (double)m[q]) * rate, sh.pow);
			s = wave_total(s);
			if (lane == 0)
				ds[q][wave] = s;
		}
	}
	__syncthreads();
	if (threadIdx.x < PER && chunk + (int)threadIdx.x < w.chunks) {
		const int q = threadIdx.x;
		const size_t o = (size_t)t * w.chunks + chunk + q;
		const bool greedy = a.temperature == 0.0f;
		const int at = greedy ? min(min(is[q][0], is[q][1]), min(is[q][2], is[q][3])) : 0;
		const float most = __builtin_fmaxf(__builtin_fmaxf(fs[q][0], fs[q][1]), __builtin_fmaxf(fs[q][2], fs[q][3]));
		give(w.top + o, (uint64_t)__float_as_uint(most) | (uint64_t)(uint32_t)at << 32);
		give(w.s + o, greedy ? 0.0 : (ds[q][0] + ds[q][1]) + (ds[q][2] + ds[q][3]));
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
		if (last_of(w.count + t, gridDim.x, &sh.flag))
			row_step(a, w, t, 0, sh);
	}
}

// One more residual sum for the rows that wait for it.  (Eight trees with draft
// rows of 151936: 11 to 13 us, nearly all of it a row's chain of steps.)
__global__ __launch_bounds__(V_THREADS, 4) void verify_residual_kernel(VerifyArgs a, VerifyWork w, int pass)
{
	__shared__ Shared sh;
	const int t = blockIdx.y, base = blockIdx.x * V_CHUNK;
	const VRow r = w.row[t];
	if ((w.join ? w.act[t] : r.waits) != pass)
		return;
	sh.fill();
	float li[V_E], qi[V_E];
	get_chunk(a.logits + (size_t)t * a.l_stride, base, a.vocab, -__builtin_inff(), li);
	get_chunk(a.draft + (size_t)t * a.d_stride, base, a.vocab, 0.0f, qi);
	const double rate = EXP16 / (double)a.temperature;
	double s = 0.0;
	__syncthreads();
#pragma unroll
	for (int e = 0; e < V_E; e++) {
		const double y = pow16(((double)li[e] - (double)r.m) * rate, sh.pow) * r.scale - r.c * (double)qi[e];
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
	sh.fill();
	__syncthreads();
	row_step(a, w, blockIdx.x, pass, sh);
}

__global__ __launch_bounds__(V_THREADS) void verify_path_kernel(VerifyArgs a, VerifyWork w)
{
	__shared__ Shared sh;
	const bool good = ranges_good(a);
	const int b = blockIdx.x, t0 = a.first ? a.first[b] : b, t1 = a.first ? a.first[b + 1] : b + 1;
	get_outcomes(a, w, good ? t0 : 0, good ? t1 : 0, sh);
	write_path(a, w, b, good ? t0 : 0, good ? t1 : 0, sh);
}

hipError_t launch_verify(const VerifyArgs &a, void *work, hipStream_t st)
{
	VerifyWork w;
	carve_verify(a, a.draft != nullptr, (uint8_t *)work, &w);
	const dim3 grid(w.chunks, a.n_tokens), block(V_THREADS);
	const int passes = a.draft && a.temperature > 0.0f ? a.max_children : 0;
	if (a.n_tokens > 0) {
		// (as many workgroups as run at once: two chunks each where there are more)
		if ((size_t)w.chunks * a.n_tokens <= V_AT_ONCE)
			tie_launch(verify_stats_kernel<1>, grid, block, 0, st, a, w);
		else
			tie_launch(verify_stats_kernel<2>, dim3((w.chunks + 1) / 2, a.n_tokens), block, 0, st, a, w);
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
