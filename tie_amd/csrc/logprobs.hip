// logprobs.hip -- log-probabilities of given tokens, with their rank, the
// distribution's entropy and the likeliest alternatives, from one read of the logits.
//
// With x_i = l_i - m, m the largest logit, and T the temperature
//   Z = sum exp(x_i / T),  log p(i) = x_i / T - log Z,
//   entropy = -sum p log p = log Z - sum x_i exp(x_i / T) / (T Z).
// Each wave keeps a running m (which moves a few times in a row) and each lane its two
// sums in 64 bits; they are brought to one m when waves are joined.  Exponentials are
// F32, of arguments x / T in 64 bits whose rest beside a whole power of two is rounded to
// 23 bits: each is off by at most 1.4 2^-23 of itself however far x is (2^-24 log 2 of the
// rest, an ulp of v_exp_f32), and so are the sums whatever their length.  (An argument rounded
// to F32 is off by half a unit in its last place, which equal and near logits have in common:
// 1.2e-6 of exponentials at x = -20, and no sum averages it out.)  The largest
// logit's is exactly 1, so that a sure token's small logarithm keeps its digits.
//
// The n likeliest: each thread keeps the largest of its logits.  n threads have one
// that reaches the n-th largest of those maxima, so no logit below it is among the n
// largest, and few threads have more than one that reaches it (n threads of 256 hold the
// n + n^2 / 512 largest, as a mean): only the chunk that a maximum came from is read
// again, and all chunks of a thread whose second best chunk reaches it too.  What
// reaches the bound is sorted, 64 at a time where equal logits bring more.
//
// A workgroup has a row, or a part of one where there are few rows; the last
// of a row's parts to finish joins them.  Many rows: bound by memory and the 64-bit arithmetic
// at once (2047 of 151936 202 to 210 us from card to card, 6.0 TB/s; with exponentials of F32
// arguments 201 to 204); few: by the row's chain of steps (one of 32000 8.9 us, 61 of 151936 22.4, of which the logits 6.4).
#include "kv.h"

namespace tie {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int LP_THREADS = 256, LP_WAVES = LP_THREADS / 64, LP_E = 16, LP_CHUNK = LP_THREADS * LP_E;
constexpr int LP_AT_ONCE = 384, LP_PARTS = 1024; // workgroups where rows are few, parts of a call at most
constexpr int LP_LIST = 1024; // (chunk, thread) whose logits are read again, at most: else all of the threads'
constexpr float LOWEST = -3.402823466e38f;

// One part's result.
struct LpPart {
	double s, t;
	float m;
	int above; // logits before the token in order
};

struct LpWork {
	LpPart *part; // [rows][parts]
	float *most;  // [rows][parts][LP_THREADS] the threads' largest logits
	int *count;   // [rows]
};

// A row's parts.  Fewer than 64 rows: enough workgroups for a CU and a half each, a chunk or more
// to each, and more than 16 only where each has eight chunks (a hand-over costs 5 us and the last
// part's chain 6: 61 rows of 151936 by seven 22.4 us, by five 25.2; 32 by twelve 19.8, by 16 20.8;
// 8 by 16 15.8, by eight 17.7; one 13.7).  64 to 170: just under two workgroups to a CU (100 rows
// by five 26.7, by four 30; 128 by four 29.8, by three 34).  To 341: three parts (200 rows 41, by
// two 44; 300 52, by two 55; by one 39 and 54, but rows that are not 16-byte aligned, of 128257, 46
// against 37).  Then two (383 58, by one 55, unaligned 54 and 63), and whole rows where those fill
// the card (384 by one 55, by three 65).
static int lp_parts(int vocab, int rows)
{
	const int chunks = (vocab + LP_CHUNK - 1) / LP_CHUNK, most = chunks < 16 ? chunks : chunks / 8 < 16 ? 16 : chunks / 8;
	const int want = rows >= 64 && rows <= 170 ? 512 / rows : rows > 170 && rows <= 341 ? 3 : (LP_AT_ONCE + rows - 1) / rows;
	return want < most ? want : most;
}

static size_t carve_logprobs(size_t parts, int n, uint8_t *base, LpWork *w)
{
	size_t off = WORK_COUNTERS * sizeof(int);
	auto take = [&](size_t bytes) {
		const size_t o = off;
		off += (bytes + 255) & ~(size_t)255;
		return base + o;
	};
	LpWork v;
	v.part = (LpPart *)take(parts * sizeof(LpPart));
	v.most = (float *)take(n ? parts * LP_THREADS * sizeof(float) : 0);
	v.count = (int *)base;
	if (w)
		*w = v;
	return off;
}

// Enough for every call of no more logits, rows and alternatives.
size_t logprobs_work_bytes(int vocab, int rows, int n)
{
	const size_t chunks = ((size_t)vocab + LP_CHUNK - 1) / LP_CHUNK, all = rows * chunks;
	return carve_logprobs(all < LP_PARTS ? all : LP_PARTS, n, nullptr, nullptr);
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

__device__ __forceinline__ void put32(float *p, float x)
{
	__hip_atomic_store((uint32_t *)p, __float_as_uint(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get32(const float *p)
{
	return __uint_as_float(__hip_atomic_load((const uint32_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
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
#pragma unroll 1
	for (int size = 2; size <= 64; size <<= 1)
#pragma unroll 1
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
#pragma unroll 1
	for (int k = 32; k > 0; k >>= 1)
		x = swap64(x, k, (lane & k) == 0);
	return x;
}

// A wave's n largest so far.
struct Best {
	uint64_t key = 0;   // the lane's, sorted; 0: none
	uint64_t bound = 0; // candidates are above it: the n-th, or one that n others reach
	int n = 0, held = 0;      // candidates that wait in `wait`
	uint64_t *wait = nullptr; // [128]

	__device__ __forceinline__ void merge()
	{
		const int lane = threadIdx.x & 63;
		const uint64_t x = lane < held ? wait[lane] : 0, rest = 64 + lane < held ? wait[64 + lane] : 0;
		if (held > 64)
			wait[lane] = rest;
		held = held > 64 ? held - 64 : 0;
		key = merge64(key, sort64(x));
		const uint64_t last = shfl64(key, n - 1);
		bound = last > bound ? last : bound;
	}
	// the keys of the lanes that `in` says
	__device__ __forceinline__ void offer(bool in, uint64_t k)
	{
		const unsigned long long set = __ballot(in && k > bound);
		if (!set)
			return;
		if (set >> (threadIdx.x & 63) & 1)
			wait[held + __popcll(set & ((1ull << (threadIdx.x & 63)) - 1))] = k;
		held += __popcll(set);
		__builtin_amdgcn_wave_barrier();
		if (held >= 64)
			merge();
	}
};

// A running distribution: the largest logit, and sums of exp((l - m) / T) and of
// (l - m) exp(...).
struct Sums {
	double s = 0.0, t = 0.0;
	float m = -__builtin_inff();
	// to another m, not below its own (rate: log2 e / T)
	__device__ __forceinline__ void move(float to, double rate)
	{
		if (m > -__builtin_inff() && m < to) {
			const double by = (double)m - to, f = exp2(by * rate);
			s *= f;
			t = t * f + by * s;
		}
		m = to;
	}
};

struct LpShared {
	uint64_t wait[LP_WAVES][128];
	uint64_t top[LP_WAVES][64];
	double s[LP_WAVES], t[LP_WAVES];
	float m[LP_WAVES], most[LP_THREADS];
	int above, held[LP_WAVES], list[LP_LIST], listed, flag;
};

// The threads' sums joined, in all of them.
__device__ __forceinline__ void join_threads(LpShared &sh, Sums &d, double rate)
{
	const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
	const float m = wave_max(d.m);
	if (lane == 0)
		sh.m[wave] = m;
	__syncthreads();
	d.move(__builtin_fmaxf(__builtin_fmaxf(sh.m[0], sh.m[1]), __builtin_fmaxf(sh.m[2], sh.m[3])), rate);
	d.s = wave_total(d.s);
	d.t = wave_total(d.t);
	if (lane == 0) {
		sh.s[wave] = d.s;
		sh.t[wave] = d.t;
	}
	__syncthreads();
	d.s = (sh.s[0] + sh.s[1]) + (sh.s[2] + sh.s[3]);
	d.t = (sh.t[0] + sh.t[1]) + (sh.t[2] + sh.t[3]);
}

// The logarithm of a sum that is 1 or more, with the digits of what it has above 1: of 2^k
// f, f from 2/3 to 4/3, k log 2 + 2 artanh((f - 1) / (f + 1)), by its series up to the 17th power
// (0.2^19 / 19 = 3e-15).
__device__ __forceinline__ double log_of(double s)
{
	int k = (int)(__double_as_longlong(s) >> 52) - 1023;
	double f = __builtin_amdgcn_ldexp(s, -k); // [1, 2)
	if (f > 4.0 / 3.0) {
		f *= 0.5;
		k++;
	}
	const double over = f + 1.0;
	double inv = __builtin_amdgcn_rcp(over); // (2^-26)
	inv = __builtin_fma(__builtin_fma(-over, inv, 1.0), inv, inv);
	const double r = (f - 1.0) * inv, r2 = r * r;
	double y = 2.0 / 17.0;
#pragma unroll
	for (int i = 15; i > 0; i -= 2)
		y = __builtin_fma(y, r2, 2.0 / i);
	return __builtin_fma((double)k, 0.69314718055994531, y * r);
}

// A row's distribution, for its outputs.
struct Row {
	bool good; // there is one
	double m, inv, logz;
	__device__ __forceinline__ float log_p(float l) const
	{
		return (float)(((double)l - m) * inv - logz);
	}
};

// The place-th of a row's alternatives: a key, or 0 for none.
__device__ __forceinline__ void write_top(const LogprobArgs &a, int row, const Row &r, int place, uint64_t key)
{
	const size_t o = (size_t)row * a.n_top + place;
	const bool is = r.good && key != 0;
	a.top_tokens[o] = is ? (int)~(uint32_t)key : -1;
	a.top_logprobs[o] = !r.good ? __builtin_nanf("") : is ? r.log_p(logit_of(key)) : -__builtin_inff();
}

// The first chunk of a part (of 2^24 logits there are 2^12).
__device__ __forceinline__ int chunk_from(int chunks, int part, int parts)
{
	return (int)((uint32_t)chunks * (uint32_t)part / (uint32_t)parts);
}

// What n of the threads' maxima sh.most reach and hardly more (a wave, each for itself), as
// the upper half of a key, to its sign, exponent and 11 bits: bit by bit from the top,
// counted in the wave's masks.  Up to 32 of them: by the lanes' maxima of four
// threads (64 lanes' hold the n + n^2 / 128 largest, as a mean).
__device__ __forceinline__ uint32_t nth_most(const LpShared &sh, int n)
{
	const int lane = threadIdx.x & 63;
	uint32_t v[LP_WAVES], t = 0, top = 0;
#pragma unroll
	for (int i = 0; i < LP_WAVES; i++) {
		v[i] = (uint32_t)(key_of(sh.most[i * 64 + lane], 0) >> 32);
		top = max(top, v[i]);
	}
	if (n <= 32) {
#pragma unroll 4
		for (int bit = 31; bit >= 12; bit--) {
			const uint32_t c = t | 1u << bit;
			t = __popcll(__ballot(top >= c)) >= n ? c : t;
		}
		return t;
	}
#pragma unroll 1
	for (int bit = 31; bit >= 12; bit--) {
		const uint32_t c = t | 1u << bit;
		int count = 0;
#pragma unroll
		for (int i = 0; i < LP_WAVES; i++)
			count += __popcll(__ballot(v[i] >= c));
		t = count >= n ? c : t;
	}
	return t;
}

// A thread's largest logit so far, the chunk (or part) that it is of, and the largest of
// its others.
struct Mosts {
	float most = -__builtin_inff(), second = most;
	int at = 0;
	__device__ __forceinline__ void add(float x, int where)
	{
		second = __builtin_fmaxf(second, __builtin_fminf(most, x));
		at = x > most ? where : at;
		most = __builtin_fmaxf(most, x);
	}
};

// The n likeliest of a row whose threads' maxima are known (where there are parts: of
// all of them, by part).
__device__ __forceinline__ void likeliest(const LogprobArgs &a, LpShared &sh, int row, const Row &r, const float *l, int parts,
					  const Mosts &t, bool vec)
{
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const int chunks = (a.vocab + LP_CHUNK - 1) / LP_CHUNK;
	sh.most[tid] = t.most;
	__syncthreads();
	// (none at -infinity)
	uint32_t nth = nth_most(sh, a.n_top);
	const uint32_t lowest = (uint32_t)(key_of(LOWEST, 0) >> 32);
	nth = nth > lowest ? nth : lowest;
	auto reaches = [&](float x) { return x > -__builtin_inff() && (uint32_t)(key_of(x, 0) >> 32) >= nth; };
	Best best;
	best.n = a.n_top;
	best.wait = sh.wait[wave];
	best.bound = (uint64_t)nth << 32; // (no key's lower half is 0)
	if (reaches(t.most)) {
		// (the chunks of one place: a chunk, or a part)
		const bool all = reaches(t.second);
		const int from = all ? 0 : parts == 1 ? t.at : chunk_from(chunks, t.at, parts);
		const int to = all ? chunks : parts == 1 ? t.at + 1 : chunk_from(chunks, t.at + 1, parts);
		int i = atomicAdd(&sh.listed, to - from);
		for (int c = from; c < to && i < LP_LIST; c++, i++)
			sh.list[i] = c * LP_THREADS + tid;
	}
	__syncthreads();
	// the logits of the listed pairs of chunk and thread again, 16 of a pair, four to a
	// lane (equal logits may bring more pairs than the list holds: then those of all
	// threads that have one, chunk by chunk).  One place that sorts, in a loop: a copy for
	// each of the logits is 100 KB of code
	const bool all = sh.listed > LP_LIST;
	const int pairs = all ? LP_THREADS : sh.listed;
#pragma unroll 1
	for (int q = 0; q < (all ? chunks : 1); q++)
#pragma unroll 1
		for (int p0 = wave * 64; p0 < pairs * 4; p0 += LP_THREADS) {
			const int p = p0 + lane;
			int at = a.vocab;
			if (p < pairs * 4) {
				const int pair = all ? q * LP_THREADS + p / 4 : sh.list[p / 4], thread = pair % LP_THREADS;
				if (!all || reaches(sh.most[thread]))
					at = pair / LP_THREADS * LP_CHUNK + (p % 4 * LP_THREADS + thread) * 4;
			}
			float x[4];
			if (vec && at + 4 <= a.vocab) {
				const float4 v = *reinterpret_cast<const float4 *>(l + at);
				x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
			} else {
#pragma unroll
				for (int e = 0; e < 4; e++)
					x[e] = at + e < a.vocab ? l[at + e] : -__builtin_inff();
			}
#pragma unroll 1
			for (int e = 0; e < 4; e++) {
				best.offer(reaches(x[0]), key_of(x[0], at + e));
				x[0] = x[1], x[1] = x[2], x[2] = x[3];
			}
		}
	// where all candidates wait still and are one wave's lot, they are sorted once
	const bool merged = best.key != 0; // (in lane 0 if in any)
	if (lane == 0)
		sh.held[wave] = merged ? 1000 : best.held;
	__syncthreads();
	int total = 0, from = 0, w0 = 0;
	for (int w = 0; w < LP_WAVES; w++) {
		if (lane >= total) {
			w0 = w;
			from = total;
		}
		total += sh.held[w];
	}
	if (total <= 64) {
		// (each candidate's place: how many are larger)
		const uint64_t key = lane < total ? sh.wait[w0][lane - from] : 0;
		int place = 0;
		for (int i = 0; i < total; i++) {
			const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), i) << 32 |
					       (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)key, i);
			place += other > key;
		}
		if (wave == 0 && (lane < total ? place : lane) < a.n_top)
			write_top(a, row, r, lane < total ? place : lane, key);
		return;
	}
	while (best.held > 0)
		best.merge();
	sh.top[wave][lane] = best.key;
	__syncthreads();
	if (wave == 0)
#pragma unroll 1
		for (int w = 1; w < LP_WAVES; w++)
			best.key = merge64(best.key, sh.top[w][lane]);
	if (wave == 0 && lane < a.n_top)
		write_top(a, row, r, lane, best.key);
}

__global__ __launch_bounds__(LP_THREADS, 4) void logprobs_kernel(LogprobArgs a, LpWork w, int parts)
{
	__shared__ LpShared sh;
	const int row = (uint32_t)blockIdx.x / (uint32_t)parts, part = (uint32_t)blockIdx.x % (uint32_t)parts, tid = threadIdx.x;
	const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const float *l = a.logits + (size_t)row * a.stride;
	const int chunks = (a.vocab + LP_CHUNK - 1) / LP_CHUNK;
	const int c0 = chunk_from(chunks, part, parts), c1 = chunk_from(chunks, part + 1, parts);
	const bool vec = ((uintptr_t)l & 15) == 0;
	auto index = [&](int c, int e) { return c * LP_CHUNK + (e / 4 * LP_THREADS + tid) * 4 + e % 4; };
	// (past the caches: nothing is read twice soon; 2047 rows of 151936 233 us without)
	auto get = [&](int c, float (&x)[LP_E]) {
		if (vec && (c + 1) * LP_CHUNK <= a.vocab) {
#pragma unroll
			for (int e = 0; e < LP_E; e += 4) {
				const f4 v = __builtin_nontemporal_load(reinterpret_cast<const f4 *>(l + (size_t)c * LP_CHUNK) + e / 4 * LP_THREADS + tid);
				x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
			}
		} else {
#pragma unroll
			for (int e = 0; e < LP_E; e++)
				x[e] = index(c, e) < a.vocab ? l[index(c, e)] : -__builtin_inff();
		}
	};
	float next[LP_E];
	get(c0, next);
	const int token = a.tokens ? a.tokens[row] : -1;
	const bool is_token = token >= 0 && token < a.vocab;
	const float mine = is_token ? l[token] : __builtin_inff();
	const double rate = a.rate, far = -127.0 / rate;
	const double grid = 0x1.8p29 - 1.0; // added to z, it leaves z - 1 in units of 2^-23 in the lower half
	// x > mine, and x < mine, are the signs of differences (of zeros +0), where mine is above -infinity
	const bool signs = mine > -__builtin_inff();
	const float mine_up = mine + 0.0f, mine_down = mine == 0.0f ? -0.0f : mine;
	Sums d;
	Mosts t;
	int above = 0;
	bool nan = false;
	for (int c = c0; c < c1; c++) {
		float x[LP_E];
#pragma unroll
		for (int e = 0; e < LP_E; e++)
			x[e] = next[e];
		if (c + 1 < c1)
			get(c + 1, next);
		float most = x[0];
#pragma unroll
		for (int e = 1; e < LP_E; e++)
			most = __builtin_elementwise_maximum(most, x[e]); // (NaN if any is)
		nan = nan || most != most;
		// (equal logits count where they come before the token: not in chunks behind its own.
		// By signs: 400 rows of 151936 55 us, by comparisons whose masks are counted 59.  A
		// likely token has few chunks with a logit before it)
		if (a.rank && __any(most >= mine)) {
			if (signs && (c + 1) * LP_CHUNK <= token) {
				above += LP_E;
#pragma unroll
				for (int e = 0; e < LP_E; e++)
					above -= (int)(__float_as_uint(x[e] - mine_down) >> 31);
			} else if (signs && c * LP_CHUNK > token) {
#pragma unroll
				for (int e = 0; e < LP_E; e++)
					above += (int)(__float_as_uint(mine_up - x[e]) >> 31);
			} else {
#pragma unroll
				for (int e = 0; e < LP_E; e++)
					above += (int)(x[e] > mine) | ((int)(x[e] == mine) & (int)(index(c, e) < token));
			}
		}
		t.add(most, c);
		if (__any(most > d.m))
			d.move(wave_max(t.most), rate);
		const double m = d.m == -__builtin_inff() ? 0.0 : (double)d.m;
#pragma unroll
		for (int e = 0; e < LP_E; e++) {
			// 2^z = 2^n 2^f: w holds n - 1 in its upper 9 bits and f in the lower 23, which are 1 + f's
			// mantissa; the exponential of that, from 2 on, gets n - 1 added to its exponent.  (Whole
			// numbers at twice the 64-bit rate: 2047 rows of 151936 207 us where whole and rest of z by
			// 64-bit sums take 218; 203 without the clamp.  z of -127, -infinity and NaN give 0, z above
			// that and below -126 less than 2^-126)
			const double y = __builtin_fmax((double)x[e] - m, far);
			const uint32_t w = (uint32_t)__double_as_longlong(__builtin_fma(y, rate, grid));
			const float e2 = __builtin_amdgcn_exp2f(__uint_as_float((w & 0x7fffffu) | 0x3f800000u));
			const double p = (double)__uint_as_float(__float_as_uint(e2) + (w & 0xff800000u));
			d.s += p;
			d.t = __builtin_fma(y, p, d.t);
		}
	}
	if (nan)
		d.s = __builtin_nan("");
	if (a.rank)
		above = (int)wave_total((double)above);
	// the threads joined; then, where there are parts, the parts by the last of them to
	// finish, by the same code
	if (tid == 0) {
		sh.above = 0;
		sh.listed = 0;
	}
	float *mosts = w.most + (size_t)row * parts * LP_THREADS;
	LpPart *to = w.part + (size_t)row * parts;
#pragma unroll 1
	for (bool whole = parts == 1;; whole = true) {
		join_threads(sh, d, rate);
		if (whole)
			break;
		if (lane == 0)
			atomicAdd(&sh.above, above);
		if (a.n_top)
			put32(mosts + (size_t)part * LP_THREADS + tid, t.most);
		if (tid == 0) {
			put64(&to[part].s, (uint64_t)__double_as_longlong(d.s));
			put64(&to[part].t, (uint64_t)__double_as_longlong(d.t));
		}
		__syncthreads();
		if (tid == 0)
			put64(&to[part].m, (uint64_t)__float_as_uint(d.m) | (uint64_t)(uint32_t)sh.above << 32);
		// what the parts wrote is there once the writers' stores are done, which each waits
		// for before its workgroup counts
		asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
		__syncthreads();
		if (tid == 0) {
			const int got = __hip_atomic_fetch_add(w.count + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
			sh.flag = got == parts - 1;
			sh.above = 0;
			if (got == parts - 1)
				__hip_atomic_store(w.count + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
		}
		__syncthreads();
		if (!sh.flag)
			return;
		// a thread a part, and a column of the maxima
		d = Sums();
		above = 0;
		for (int q = tid; q < parts; q += LP_THREADS) {
			const double ps = __longlong_as_double((long long)get64(&to[q].s)), pt = __longlong_as_double((long long)get64(&to[q].t));
			const uint64_t v = get64(&to[q].m);
			const float m = __uint_as_float((uint32_t)v), most = __builtin_fmaxf(d.m, m);
			Sums b;
			b.s = ps, b.t = pt, b.m = m;
			above += (int)(v >> 32);
			if (q >= LP_THREADS) { // (a thread's second part)
				d.move(most, rate);
				b.move(most, rate);
			}
			d.s += b.s, d.t += b.t, d.m = most;
		}
		t = Mosts();
		for (int q0 = 0; a.n_top && q0 < parts; q0 += 16) {
			float x[16];
#pragma unroll
			for (int i = 0; i < 16; i++)
				x[i] = get32(mosts + (size_t)min(q0 + i, parts - 1) * LP_THREADS + tid);
#pragma unroll
			for (int i = 0; i < 16; i++)
				if (q0 + i < parts)
					t.add(x[i], q0 + i);
		}
	}
	// (of parts a thread's own, else a wave's)
	if (parts > 1 ? above != 0 : lane == 0)
		atomicAdd(&sh.above, above);
	Row r;
	r.good = d.m > -__builtin_inff() && d.m < __builtin_inff() && d.s < (double)__builtin_inff(); // (no NaN among them)
	r.m = d.m;
	r.inv = a.inv;
	r.logz = log_of(d.s);
	if (a.n_top)
		likeliest(a, sh, row, r, l, parts, t, vec);
	else
		__syncthreads();
	// (behind all barriers, which wait for stores; by the last wave: the first has written the alternatives)
	if (tid == LP_THREADS - 64) {
		if (a.logprob)
			a.logprob[row] = r.good && is_token ? r.log_p(mine) : __builtin_nanf("");
		if (a.rank)
			a.rank[row] = r.good && is_token ? sh.above : -1;
		if (a.entropy) {
			double inv = __builtin_amdgcn_rcp(d.s); // (2^-26)
			inv = __builtin_fma(__builtin_fma(-d.s, inv, 1.0), inv, inv);
			a.entropy[row] = r.good ? (float)(r.logz - d.t * r.inv * inv) : __builtin_nanf("");
		}
	}
}

hipError_t launch_logprobs(const LogprobArgs &a, void *work, hipStream_t st)
{
	const int parts = lp_parts(a.vocab, a.n_rows);
	LpWork w;
	carve_logprobs(parts > 1 ? (size_t)a.n_rows * parts : 0, a.n_top, (uint8_t *)work, &w);
	tie_launch(logprobs_kernel, dim3((uint32_t)a.n_rows * parts), dim3(LP_THREADS), 0, st, a, w, parts);
	return hipGetLastError();
}

} // namespace tie
