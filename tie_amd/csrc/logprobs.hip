// logprobs.hip -- log-probabilities of given tokens, with their rank, the
// distribution's entropy and the likeliest alternatives, from one read of the logits.
//
// With x_i = l_i - m, m the largest logit, and T the temperature
//   Z = sum exp(x_i / T),  log p(i) = x_i / T - log Z,
//   entropy = -sum p log p = log Z - sum x_i exp(x_i / T) / (T Z).
// Each lane keeps its own running m with its two sums in 64 bits; they are
// brought to one m when lanes are joined.  Exponentials are F32 (an ulp each, so that
// the sums are good to 1e-7 of themselves whatever their length).
//
// The n likeliest: a wave keeps the 64 largest so far sorted over its lanes, as
// 64-bit keys (the logit's order, then the lower index first).  A logit is a
// candidate if it reaches the n-th of them; candidates gather in LDS and are sorted and
// merged 64 at a time.  The first bound is the n-th largest of the lanes' own
// maxima, which n logits reach for certain: then few others do.
//
// A workgroup has a row, or a part of one where there are few rows; the last
// of a row's parts to finish joins them.
#include "kv.h"

namespace tie {

constexpr int LP_THREADS = 256, LP_WAVES = LP_THREADS / 64, LP_E = 16, LP_CHUNK = LP_THREADS * LP_E;
constexpr float NONE = -3.402823466e38f; // the lowest finite value

// One part's result.
struct LpPart {
	double s, t;
	float m;
	int above; // logits before the token in order
};

struct LpWork {
	LpPart *part;  // [rows][parts]
	uint64_t *top; // [rows][parts][n]
	int *count;    // [rows]
};

static int lp_parts(int vocab, int rows)
{
	// as many workgroups as run at once (four on a CU)
	const int chunks = (vocab + LP_CHUNK - 1) / LP_CHUNK, want = (1024 + rows - 1) / rows;
	return rows > WORK_COUNTERS || want < 2 ? 1 : want < chunks ? want : chunks;
}

static size_t carve_logprobs(int rows, int parts, int n, uint8_t *base, LpWork *w)
{
	size_t off = WORK_COUNTERS * sizeof(int);
	auto take = [&](size_t bytes) {
		const size_t o = off;
		off += (bytes + 255) & ~(size_t)255;
		return base + o;
	};
	LpWork v;
	v.part = (LpPart *)take((size_t)rows * parts * sizeof(LpPart));
	v.top = (uint64_t *)take((size_t)rows * parts * n * 8);
	v.count = (int *)base;
	if (w)
		*w = v;
	return off;
}

// Enough for every call of no more logits, rows and alternatives: rows * parts is at most
// 1024 + rows, where there are parts.
size_t logprobs_work_bytes(int vocab, int rows, int n)
{
	const int chunks = (vocab + LP_CHUNK - 1) / LP_CHUNK, r = rows < 1024 ? rows : 1024;
	const size_t most = (size_t)r * chunks < 2047 ? (size_t)r * chunks : 2047;
	return carve_logprobs(1, (int)most, n, nullptr, nullptr);
}

// what one workgroup writes for another of the same launch goes past the dies' caches
__device__ __forceinline__ void put64(void *p, uint64_t x)
{
	__hip_atomic_store((uint64_t *)p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t get64(const void *p)
{
	return __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ uint64_t key_of(float l, int i)
{
	const uint32_t b = __float_as_uint(l + 0.0f); // (-0 as 0)
	const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
	return (uint64_t)up << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float logit_of(uint64_t key)
{
	const uint32_t up = (uint32_t)(key >> 32);
	return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int lane)
{
	return (uint64_t)(uint32_t)__shfl((int)(x >> 32), lane) << 32 | (uint32_t)__shfl((int)(uint32_t)x, lane);
}

// The larger (or the smaller) of x and the key of lane ^ k.
__device__ __forceinline__ uint64_t swap64(uint64_t x, int k, bool larger)
{
	const uint64_t y = shfl64(x, (int)(threadIdx.x & 63) ^ k);
	return (x > y) == larger ? x : y;
}

// Keys sorted over the wave, the largest in lane 0.
__device__ __forceinline__ uint64_t sort64(uint64_t x)
{
	const int lane = threadIdx.x & 63;
#pragma unroll
	for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
		for (int k = size / 2; k > 0; k >>= 1)
			x = swap64(x, k, ((lane & size) == 0) == ((lane & k) == 0));
	return x;
}

// The 64 largest of two sorted lots.
__device__ __forceinline__ uint64_t merge64(uint64_t a, uint64_t b)
{
	const int lane = threadIdx.x & 63;
	const uint64_t r = shfl64(b, 63 - lane);
	uint64_t x = a > r ? a : r;
#pragma unroll
	for (int k = 32; k > 0; k >>= 1)
		x = swap64(x, k, (lane & k) == 0);
	return x;
}

// the same of floats: sorted, the largest in lane 0
__device__ __forceinline__ float sort_floats(float x)
{
	const int lane = threadIdx.x & 63;
#pragma unroll
	for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
		for (int k = size / 2; k > 0; k >>= 1) {
			const float y = __shfl_xor(x, k);
			x = ((lane & size) == 0) == ((lane & k) == 0) ? __builtin_fmaxf(x, y) : __builtin_fminf(x, y);
		}
	return x;
}

// A wave's n largest so far.
struct Best {
	uint64_t key = 0;    // the lane's, sorted; 0: none
	uint64_t bound = 0;  // the n-th: candidates are above it
	float least = NONE;  // its logit
	int n = 0, held = 0; // candidates that wait in `wait`
	uint64_t *wait = nullptr; // [128]

	__device__ __forceinline__ void merge()
	{
		const int lane = threadIdx.x & 63;
		uint64_t x = lane < held ? wait[lane] : 0;
		const uint64_t rest = 64 + lane < held ? wait[64 + lane] : 0;
		if (held > 64)
			wait[lane] = rest;
		held = held > 64 ? held - 64 : 0;
		key = merge64(key, sort64(x));
		const uint64_t last = shfl64(key, n - 1);
		if (last > bound) {
			bound = last;
			least = __builtin_fmaxf(least, logit_of(last));
		}
	}
	// the wave's logits x[0 .. E) of indexes i[e]
	template <typename I> __device__ __forceinline__ void offer(const float (&x)[LP_E], float most, I index)
	{
		if (!__any(most >= least))
			return;
		// (n lanes have a logit that reaches the n-th of their maxima)
		if (bound == 0)
			least = __builtin_fmaxf(least, __shfl(sort_floats(most), n - 1));
		const int lane = threadIdx.x & 63;
#pragma unroll
		for (int e = 0; e < LP_E; e++) {
			const uint64_t k = key_of(x[e], index(e));
			const bool in = x[e] >= least && k > bound;
			const unsigned long long set = __ballot(in);
			if (!set)
				continue;
			if (in)
				wait[held + __popcll(set & ((1ull << lane) - 1))] = k;
			held += __popcll(set);
			__builtin_amdgcn_wave_barrier();
			if (held >= 64)
				merge();
		}
	}
};

// A running distribution: the largest logit, and sums of exp((l - m) / T) and of
// (l - m) exp(...).
struct Sums {
	double s = 0.0, t = 0.0;
	float m = -__builtin_inff();
};

// b's sums added to a's (rate: log2 e / T)
__device__ __forceinline__ void add(Sums &a, double s, double t, float m, double rate)
{
	const float most = __builtin_fmaxf(a.m, m);
	if (most == -__builtin_inff()) {
		a.s += s; // (0, or NaN)
		return;
	}
	const double da = a.m == -__builtin_inff() ? 0.0 : (double)a.m - most, db = m == -__builtin_inff() ? 0.0 : (double)m - most;
	const double fa = exp2(da * rate), fb = exp2(db * rate);
	const double s0 = a.s * fa, s1 = s * fb;
	a.t = a.t * fa + da * s0 + t * fb + db * s1;
	a.s = s0 + s1;
	a.m = most;
}

// over the wave
__device__ __forceinline__ void join_lanes(Sums &a, double rate)
{
	const float most = wave_max(a.m);
	if (most == -__builtin_inff()) {
		a.s = wave_total(a.s);
		a.t = 0.0;
		return;
	}
	const double d = a.m == -__builtin_inff() ? 0.0 : (double)a.m - most, f = exp2(d * rate), s = a.s * f;
	a.t = wave_total(a.t * f + d * s);
	a.s = wave_total(s);
	a.m = most;
}

struct LpShared {
	uint64_t wait[LP_WAVES][128];
	uint64_t top[LP_WAVES][64];
	double s[LP_WAVES], t[LP_WAVES];
	float m[LP_WAVES];
	int above[LP_WAVES], flag;
};

// The waves' results joined, in the first wave.
__device__ __forceinline__ void join_waves(LpShared &sh, Sums &a, int &above, Best &best, double rate)
{
	const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
	join_lanes(a, rate);
	above = (int)wave_total((double)above);
	if (lane == 0) {
		sh.s[wave] = a.s;
		sh.t[wave] = a.t;
		sh.m[wave] = a.m;
		sh.above[wave] = above;
	}
	sh.top[wave][lane] = best.key;
	__syncthreads();
	if (wave)
		return;
	for (int w = 1; w < LP_WAVES; w++) {
		add(a, sh.s[w], sh.t[w], sh.m[w], rate);
		above += sh.above[w];
		if (best.n)
			best.key = merge64(best.key, sh.top[w][lane]);
	}
}

// The row's outputs (a wave).
__device__ __forceinline__ void write_row(const LogprobArgs &a, int row, const Sums &d, int above, uint64_t key)
{
	const int lane = threadIdx.x & 63;
	const bool good = d.m > -__builtin_inff() && d.m < __builtin_inff() && d.s < (double)__builtin_inff(); // (no NaN among them)
	const double inv = 1.0 / (double)a.temperature, logz = log(d.s);
	if (lane == 0) {
		if (a.tokens) {
			const int token = a.tokens[row];
			const bool is = good && token >= 0 && token < a.vocab;
			const float l = is ? a.logits[(size_t)row * a.stride + token] : 0.0f;
			if (a.logprob)
				a.logprob[row] = is ? (float)(((double)l - d.m) * inv - logz) : __builtin_nanf("");
			if (a.rank)
				a.rank[row] = is ? above : -1;
		}
		if (a.entropy)
			a.entropy[row] = good ? (float)(logz - d.t * inv / d.s) : __builtin_nanf("");
	}
	if (lane < a.n_top) {
		const size_t o = (size_t)row * a.n_top + lane;
		const bool is = good && key != 0;
		a.top_tokens[o] = is ? (int)~(uint32_t)key : -1;
		a.top_logprobs[o] = !good ? __builtin_nanf("") : is ? (float)(((double)logit_of(key) - d.m) * inv - logz) : -__builtin_inff();
	}
}

__global__ __launch_bounds__(LP_THREADS, 4) void logprobs_kernel(LogprobArgs a, LpWork w, int parts)
{
	__shared__ LpShared sh;
	const int row = (uint32_t)blockIdx.x / (uint32_t)parts, part = (uint32_t)blockIdx.x % (uint32_t)parts, tid = threadIdx.x, lane = tid & 63;
	const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const float *l = a.logits + (size_t)row * a.stride;
	const int chunks = (a.vocab + LP_CHUNK - 1) / LP_CHUNK;
	const int c0 = (int)((long long)chunks * part / parts), c1 = (int)((long long)chunks * (part + 1) / parts);
	const int token = a.tokens ? a.tokens[row] : -1;
	const bool is_token = token >= 0 && token < a.vocab;
	const float mine = is_token ? l[token] : __builtin_inff();
	const bool vec = ((uintptr_t)l & 15) == 0;
	const double rate = 1.4426950408889634 / (double)a.temperature;
	const float rate_hi = (float)rate, rate_lo = (float)(rate - (double)rate_hi);
	const float far = -200.0f / rate_hi; // from there on exp() is 0
	Sums d;
	Best best;
	best.n = a.n_top;
	best.wait = sh.wait[wave];
	int above = 0;
	for (int c = c0; c < c1; c++) {
		const int base = c * LP_CHUNK;
		float x[LP_E];
		auto index = [&](int e) { return base + (e / 4 * LP_THREADS + tid) * 4 + e % 4; };
		if (vec && base + LP_CHUNK <= a.vocab) {
#pragma unroll
			for (int e = 0; e < LP_E; e += 4) {
				const float4 v = reinterpret_cast<const float4 *>(l + base)[e / 4 * LP_THREADS + tid];
				x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
			}
		} else {
#pragma unroll
			for (int e = 0; e < LP_E; e++)
				x[e] = index(e) < a.vocab ? l[index(e)] : -__builtin_inff();
		}
		float most = x[0];
#pragma unroll
		for (int e = 1; e < LP_E; e++)
			most = __builtin_fmaxf(most, x[e]);
		if (a.n_top)
			best.offer(x, most, index);
#pragma unroll
		for (int e = 0; e < LP_E; e++)
			above += x[e] > mine || (x[e] == mine && index(e) < token);
		if (__any(most > d.m)) {
			const float m = __builtin_fmaxf(d.m, most);
			if (d.m > -__builtin_inff() && m > d.m) {
				const double by = (double)d.m - m, f = exp2(by * rate);
				d.s *= f;
				d.t = d.t * f + by * d.s;
			}
			d.m = m;
		}
		const float base_m = d.m == -__builtin_inff() ? 0.0f : d.m;
#pragma unroll
		for (int e = 0; e < LP_E; e++) {
			float y = x[e] - base_m;
			y = y < far ? far : y; // (NaN stays)
			const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(y, rate_lo, y * rate_hi));
			d.s += (double)p;
			d.t = __builtin_fma((double)y, (double)p, d.t);
		}
	}
	while (best.held > 0)
		best.merge();
	join_waves(sh, d, above, best, rate);
	if (parts == 1) {
		if (wave == 0)
			write_row(a, row, d, above, best.key);
		return;
	}
	LpPart *to = w.part + (size_t)row * parts;
	uint64_t *tops = w.top + (size_t)row * parts * a.n_top;
	if (wave == 0) {
		if (lane == 0) {
			put64(&to[part].s, (uint64_t)__double_as_longlong(d.s));
			put64(&to[part].t, (uint64_t)__double_as_longlong(d.t));
			put64(&to[part].m, (uint64_t)__float_as_uint(d.m) | (uint64_t)(uint32_t)above << 32);
		}
		if (lane < a.n_top)
			put64(tops + (size_t)part * a.n_top + lane, best.key);
		// the last of the row's parts joins them: what the parts wrote is there once the
		// writer's stores are done, which it waits for before it counts
		asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
		if (lane == 0) {
			const int got = __hip_atomic_fetch_add(w.count + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
			sh.flag = got == parts - 1;
			if (got == parts - 1)
				__hip_atomic_store(w.count + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
		}
	}
	__syncthreads();
	if (!sh.flag)
		return;
	// a lane a part
	Sums all;
	int sum = 0;
	for (int q = tid; q < parts; q += LP_THREADS) {
		const double s = __longlong_as_double((long long)get64(&to[q].s)), t = __longlong_as_double((long long)get64(&to[q].t));
		const uint64_t v = get64(&to[q].m);
		add(all, s, t, __uint_as_float((uint32_t)v), rate);
		sum += (int)(v >> 32);
	}
	best.key = 0;
	if (a.n_top)
		for (int q = wave; q < parts; q += LP_WAVES)
			best.key = merge64(best.key, lane < a.n_top ? get64(tops + (size_t)q * a.n_top + lane) : 0);
	join_waves(sh, all, sum, best, rate);
	if (wave == 0)
		write_row(a, row, all, sum, best.key);
}

hipError_t launch_logprobs(const LogprobArgs &a, void *work, hipStream_t st)
{
	const int parts = lp_parts(a.vocab, a.n_rows);
	LpWork w;
	carve_logprobs(a.n_rows, parts, a.n_top, (uint8_t *)work, &w);
	tie_launch(logprobs_kernel, dim3((uint32_t)a.n_rows * parts), dim3(LP_THREADS), 0, st, a, w, parts);
	return hipGetLastError();
}

} // namespace tie
