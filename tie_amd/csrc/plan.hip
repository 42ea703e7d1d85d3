// plan.hip -- the pages of a step: which rows of the activations each request's
// tokens have, the pages that they are written to, and the pages that come free.
//
// Request b has len[b] rows and asks for n_new[b] more.  It needs the pages of
// its new rows that its row of the table does not name yet,
//   need(b) = #{ c : ceil(len / 64) <= c < ceil((len + n_new) / 64), pages[b][c] is none },
// and requests are served in order while their running sums of need and of n_new stay
// within the free pages and the token rows: the first that does not fit ends it, so
// what is served is a prefix, and running sums over all requests are those over the
// served ones.  Pages that go back (of requests that ended, and behind the window)
// are numbered by a running sum too.  No atomics: two equal calls give equal arrays.
//
// Free pages lie in a ring: taken from its head, put behind its tail.  What a call
// takes and what it puts never share a place, so the call can be made again from the
// same state.
//
// A wave has a request, its lanes 64 columns of the page table at a time.  Many
// requests: one launch counts (and copies the table), one sums the counts of the
// blocks before its own and writes.  Few: both in one workgroup.  Bound by the
// chain of loads (length, table, sums, ring) and the launches, not by bytes: 5 requests
// 4.3 us, 257 of 512 columns 11.6, 1024 prompts of 300 10.0.
#include "kv.h"

namespace tie {

constexpr int PLAN_BLOCK = 16; // requests of a workgroup, one to a wave
constexpr int PLAN_THREADS = 64 * PLAN_BLOCK;
constexpr int PLAN_SMALL = 64; // requests that one workgroup takes alone

struct PlanCounts {
	int need, want, away; // pages to take, token rows, pages to give back
	int held;             // pages of its new rows that the table names already
	int away0;            // the first column whose page goes back
	int len;
};

struct PlanWork {
	PlanCounts *counts; // [n_seqs]
	uint32_t *sums;     // [blocks][3] of need, want and away
	int *state;         // the ring's, as the call found it (it may be updated in place)
};

static size_t carve_plan(int n_seqs, uint8_t *base, PlanWork *w)
{
	size_t off = WORK_COUNTERS * sizeof(int);
	auto take = [&](size_t bytes) {
		const size_t o = off;
		off += (bytes + 255) & ~(size_t)255;
		return base + o;
	};
	PlanWork v;
	v.counts = (PlanCounts *)take((size_t)n_seqs * sizeof(PlanCounts));
	v.sums = (uint32_t *)take(((size_t)n_seqs + PLAN_BLOCK - 1) / PLAN_BLOCK * 3 * sizeof(uint32_t));
	v.state = (int *)take(2 * sizeof(int));
	if (w)
		*w = v;
	return off;
}

size_t plan_work_bytes(int n_seqs)
{
	return carve_plan(n_seqs, nullptr, nullptr);
}

// Sums that stay at 2^32 - 1 when they pass it.  A limit is below 2^31, and so is one request's
// count: a sum that fits is exact, and so is the one that first does not, less that request.
// A block's sum may have stayed at 2^32 - 1 itself: it says that the block does not fit, and
// nothing is taken off it or off a sum that holds it.
__device__ __forceinline__ uint32_t plus(uint32_t x, uint32_t y)
{
	return __builtin_elementwise_add_sat(x, y);
}

template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t plus_dpp(uint32_t x)
{
	return plus(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false));
}

// the running sum over the wave, as running_of() makes it
__device__ __forceinline__ uint32_t running_sum(uint32_t x)
{
	x = plus_dpp<0x111, 0xf>(x);
	x = plus_dpp<0x112, 0xf>(x);
	x = plus_dpp<0x114, 0xf>(x);
	x = plus_dpp<0x118, 0xf>(x);
	x = plus_dpp<0x142, 0xa>(x);
	return plus_dpp<0x143, 0xc>(x);
}

__device__ __forceinline__ uint32_t sum_at(uint32_t x, int lane)
{
	return (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// The columns of a request's new rows: from c0 on, of which all but the first may be
// taken from the ring, those from `fresh` on.
struct Columns {
	int c0, c1, fresh;
	__device__ __forceinline__ Columns(int len, int want)
	{
		c0 = want ? len / PAGE : 0;
		c1 = want ? (len + want - 1) / PAGE + 1 : 0;
		fresh = want ? c0 + (len % PAGE != 0) : 0;
	}
};

__device__ __forceinline__ bool is_page(const PlanArgs &a, int id)
{
	return id >= 0 && id < a.n_pages;
}

// A wave: the counts of request b, and its row of the table copied.  Columns are loaded
// PLAN_AHEAD times 64 at a time.
constexpr int PLAN_AHEAD = 8;
__device__ __forceinline__ PlanCounts count_request(const PlanArgs &a, int b)
{
	const int32_t *row = a.pages + (size_t)b * a.max_pages;
	int32_t *out = a.pages_out + (size_t)b * a.max_pages;
	const int lane = threadIdx.x & 63, len = a.len[b], more = a.n_new[b];
	const bool copy = out != row, good = len >= 0 && more >= 0 && (long long)len + more <= (long long)a.max_pages * PAGE;
	PlanCounts n = {0, good ? more : 0, 0, 0, 0, len};
	const Columns c(len, n.want);
	// the columns whose pages go back: all of one that ended; else those whose last row is
	// below the window of the next token, at row len
	int r0 = 0, r1 = more < 0 ? a.max_pages : 0;
	if (a.window && more >= 0) {
		const long long low = (long long)len - a.window + 1;
		r0 = a.sinks / PAGE + (a.sinks % PAGE != 0);
		r1 = low > 0 ? min((int)(low / PAGE), a.max_pages) : 0;
	}
	// (in place: the two ranges, which do not meet, and what lies between them)
	const int from = copy ? 0 : r0 < r1 ? r0 : c.fresh, to = copy ? a.max_pages : c.c1 > c.fresh ? c.c1 : r1;
#pragma unroll 1
	for (int c0 = from; c0 < to; c0 += 64 * PLAN_AHEAD) {
		int id[PLAN_AHEAD];
#pragma unroll
		for (int i = 0; i < PLAN_AHEAD; i++) {
			const int x = c0 + i * 64 + lane;
			id[i] = x < to ? row[x] : -1;
		}
#pragma unroll
		for (int i = 0; i < PLAN_AHEAD; i++) {
			const int x = c0 + i * 64 + lane;
			if (c0 + i * 64 >= to)
				break;
			if (copy && x < to)
				out[x] = id[i];
			const bool page = is_page(a, id[i]);
			n.held += __popcll(__ballot(page && x >= c.fresh && x < c.c1));
			const unsigned long long away = __ballot(page && x >= r0 && x < r1);
			if (away && n.away == 0)
				n.away0 = c0 + i * 64 + __builtin_ctzll(away);
			n.away += __popcll(away);
		}
	}
	n.need = c.c1 - c.fresh - n.held;
	return n;
}

// The ring as the call found it; one that is none has no pages and takes none.
struct Ring {
	int head, free, room;
};

__device__ __forceinline__ Ring ring_of(const PlanArgs &a, const int *state)
{
	Ring r = {state[0], state[1], 0};
	if (r.head < 0 || r.head >= a.n_pages || r.free < 0 || r.free > a.n_pages)
		r.head = r.free = 0;
	else
		r.room = a.n_pages - r.free;
	return r;
}

__device__ __forceinline__ int ring_at(const PlanArgs &a, const Ring &r, int i)
{
	const long long at = (long long)r.head + i;
	return (int)(at < a.n_pages ? at : at - a.n_pages < a.n_pages ? at - a.n_pages : at - 2 * (long long)a.n_pages);
}

// The table's entries of a request's columns that may be named already, from `at` on: a
// lane each.
__device__ __forceinline__ int named(const PlanArgs &a, int b, const PlanCounts &n, const Columns &c, int at)
{
	const int col = at + (int)(threadIdx.x & 63);
	return col < (n.held ? c.c1 : c.fresh) ? a.pages[(size_t)b * a.max_pages + col] : -1;
}

// A wave: what request b gets, its columns' chunks y, y + ny, ... of 64, the first of which
// has the entries id (see named()).  need0, want0, away0: the sums over the requests before it.
__device__ __forceinline__ void fill_request(const PlanArgs &a, int b, const PlanCounts &n, const Ring &ring, uint32_t need0,
					     uint32_t want0, uint32_t away0, int y, int ny, int id)
{
	const int32_t *row = a.pages + (size_t)b * a.max_pages;
	int32_t *out = a.pages_out + (size_t)b * a.max_pages;
	const int lane = threadIdx.x & 63;
	if (n.want && plus(need0, n.need) <= (uint32_t)ring.free && plus(want0, n.want) <= (uint32_t)a.n_tokens) {
		const Columns k(n.len, n.want);
		const int t0 = (int)want0 - n.len, end = n.len + n.want; // (token row of cache row 0)
		// (where the table names some of the pages, the ones before are counted in turn)
		const bool all_fresh = n.held == 0;
		int taken = 0;
		for (int c = k.c0 + (all_fresh ? y * 64 : 0); c < k.c1 && (all_fresh || y == 0);) {
			const int col = c + lane;
			const bool fresh = col >= k.fresh && col < k.c1 && !is_page(a, id);
			const unsigned long long set = __ballot(fresh);
			const int rank = all_fresh ? col - k.fresh : taken + __popcll(set & ((1ull << lane) - 1));
			if (fresh) {
				id = a.ring[ring_at(a, ring, (int)need0 + rank)];
				out[col] = id;
			}
			taken += __popcll(set);
			const int from = max(n.len, c * PAGE), to = (int)min((long long)end, ((long long)c + 64) * PAGE);
			if (a.pos || a.slot)
				for (int x0 = from; x0 < to; x0 += 64) {
					const int x = x0 + lane, page = __shfl(id, x / PAGE - c);
					if (x < to) {
						if (a.pos)
							a.pos[t0 + x] = x;
						if (a.slot)
							a.slot[t0 + x] = is_page(a, page) ? page * PAGE + x % PAGE : -1;
					}
				}
			c += all_fresh ? ny * 64 : 64;
			id = named(a, b, n, k, c);
		}
	}
	if (y)
		return;
	// (the first n.away pages from the first of them on)
	int gone = 0;
	for (int c = n.away0; gone < n.away && c < a.max_pages; c += 64) {
		const int col = c + lane, page = col < a.max_pages ? row[col] : -1;
		const bool away = is_page(a, page);
		const unsigned long long set = __ballot(away);
		const int at = gone + __popcll(set & ((1ull << lane) - 1));
		if (away && at < n.away && plus(away0, at) < (uint32_t)ring.room) {
			a.ring[ring_at(a, ring, ring.free + (int)away0 + at)] = page;
			out[col] = -1;
		}
		gone += __popcll(set);
	}
}

// What is known when all requests are summed: the last range's end, the token rows
// behind it and the ring's new state.
__device__ __forceinline__ void finish_plan(const PlanArgs &a, const Ring &ring, const int *state, uint32_t need, uint32_t want,
					    uint32_t away, int thread, int threads)
{
	// (n_tokens may be as large as an int: the counter is wider)
	if (a.pos || a.slot)
		for (size_t t = (size_t)want + thread; t < (size_t)a.n_tokens; t += threads) {
			if (a.pos)
				a.pos[t] = -1;
			if (a.slot)
				a.slot[t] = -1;
		}
	if (thread == 0) {
		const bool none = ring.room == 0 && ring.free == 0; // (no ring)
		const int back = (int)min(away, (uint32_t)ring.room);
		a.first[a.n_seqs] = (int)want;
		a.state_out[0] = none ? state[0] : ring_at(a, ring, (int)need);
		a.state_out[1] = none ? state[1] : ring.free - (int)need + back;
	}
}

// of requests b0 .. b0 + n - 1, a lane each
__device__ __forceinline__ PlanCounts counts_at(const PlanCounts *counts, int b0, int n)
{
	const int lane = threadIdx.x & 63;
	return lane < n ? counts[b0 + lane] : PlanCounts{0, 0, 0, 0, 0, 0};
}

__global__ __launch_bounds__(PLAN_THREADS) void plan_count_kernel(PlanArgs a, PlanWork w)
{
	__shared__ PlanCounts counts[PLAN_BLOCK];
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, b = blockIdx.x * PLAN_BLOCK + wave;
	PlanCounts n = {0, 0, 0, 0, 0, 0};
	if (b < a.n_seqs) {
		n = count_request(a, b);
		if (lane == 0)
			w.counts[b] = n;
	}
	if (lane == 0)
		counts[wave] = n;
	__syncthreads();
	if (wave == 0) {
		const PlanCounts c = counts_at(counts, 0, PLAN_BLOCK);
		const uint32_t need = running_sum(c.need), want = running_sum(c.want), away = running_sum(c.away);
		if (lane == 63) {
			w.sums[blockIdx.x * 3] = need;
			w.sums[blockIdx.x * 3 + 1] = want;
			w.sums[blockIdx.x * 3 + 2] = away;
		}
		if (blockIdx.x == 0 && lane < 2)
			w.state[lane] = a.state[lane];
	}
}

// The sums over the requests so far, and of those that are served where the sums pass
// what there is: cut is set then, and every request from there on gets nothing.
struct Before {
	uint32_t need = 0, want = 0, away = 0;
	bool cut = false;
	// the first lane where the running sums pass what there is, 64: none
	__device__ __forceinline__ int over(const PlanArgs &a, const Ring &ring, uint32_t more_need, uint32_t more_want) const
	{
		const unsigned long long set = __ballot(plus(need, more_need) > (uint32_t)ring.free || plus(want, more_want) > (uint32_t)a.n_tokens);
		return set ? __builtin_ctzll(set) : 64;
	}
	// a lane's counts added; the sums before each of them
	__device__ __forceinline__ void add(const PlanArgs &a, const Ring &ring, const PlanCounts &mine, uint32_t &my_need, uint32_t &my_want,
					    uint32_t &my_away)
	{
		const uint32_t n = running_sum(mine.need), w = running_sum(mine.want), g = running_sum(mine.away);
		my_need = plus(need, n - mine.need);
		my_want = plus(want, w - mine.want);
		my_away = plus(away, g - mine.away);
		away = plus(away, sum_at(g, 63));
		if (cut)
			return;
		const int l = over(a, ring, n, w);
		cut = l < 64;
		need = cut ? sum_at(my_need, l & 63) : plus(need, sum_at(n, 63));
		want = cut ? sum_at(my_want, l & 63) : plus(want, sum_at(w, 63));
	}
};

// of lane i
__device__ __forceinline__ PlanCounts counts_of(const PlanCounts &c, int i)
{
	auto of = [&](int x) { return __builtin_amdgcn_readlane(x, i); };
	return PlanCounts{of(c.need), of(c.want), of(c.away), of(c.held), of(c.away0), of(c.len)};
}

__global__ __launch_bounds__(PLAN_THREADS) void plan_fill_kernel(PlanArgs a, PlanWork w)
{
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, block = blockIdx.x;
	// (the loads that wait for nothing first: the counts, and the table by them)
	const int b0 = block * PLAN_BLOCK, m = min(PLAN_BLOCK, a.n_seqs - b0);
	const PlanCounts mine = counts_at(w.counts, b0, m);
	const Ring ring = ring_of(a, w.state);
	uint32_t sum0[3] = {0, 0, 0};
	if (lane < block)
		for (int i = 0; i < 3; i++)
			sum0[i] = w.sums[lane * 3 + i];
	const PlanCounts own = counts_of(mine, wave);
	const Columns k(own.len, own.want);
	const int id = wave < m ? named(a, b0 + wave, own, k, k.c0 + (own.held ? 0 : (int)blockIdx.y * 64)) : -1;
	Before s;
	// the blocks before this one, 64 at a time; the one that the cut lies in is looked at
	for (int k0 = 0; k0 < block; k0 += 64) {
		const int k = k0 + lane;
		uint32_t x[3] = {sum0[0], sum0[1], sum0[2]};
		if (k0)
			for (int i = 0; i < 3; i++)
				x[i] = k < block ? w.sums[k * 3 + i] : 0;
		const uint32_t need = running_sum(x[0]), want = running_sum(x[1]), away = plus(s.away, sum_at(running_sum(x[2]), 63));
		if (!s.cut) {
			const int l = s.over(a, ring, need, want);
			if (l < 64) {
				const int from = (k0 + l) * PLAN_BLOCK;
				// (before that block: the sums up to the lane before)
				s.need = plus(s.need, l ? sum_at(need, l - 1) : 0);
				s.want = plus(s.want, l ? sum_at(want, l - 1) : 0);
				uint32_t none[3];
				s.add(a, ring, counts_at(w.counts, from, min(PLAN_BLOCK, a.n_seqs - from)), none[0], none[1], none[2]);
			} else {
				s.need = plus(s.need, sum_at(need, 63));
				s.want = plus(s.want, sum_at(want, 63));
			}
		}
		s.away = away;
	}
	uint32_t need, want, away;
	const bool cut_before = s.cut;
	const uint32_t want_at = s.want;
	s.add(a, ring, mine, need, want, away);
	if (wave < m) {
		// (past the cut: sums that nothing fits)
		fill_request(a, b0 + wave, own, ring, cut_before ? ~0u : sum_at(need, wave), sum_at(want, wave), sum_at(away, wave), blockIdx.y,
			     gridDim.y, id);
	}
	if (blockIdx.y == 0 && wave == 0 && lane < m)
		a.first[b0 + lane] = (int)(cut_before ? want_at : min(want, s.want));
	if (block == (int)gridDim.x - 1)
		finish_plan(a, ring, w.state, s.need, s.want, s.away, blockIdx.y * PLAN_THREADS + threadIdx.x, gridDim.y * PLAN_THREADS);
}

// Few requests: all of it in one workgroup.
__global__ __launch_bounds__(1024) void plan_small_kernel(PlanArgs a)
{
	__shared__ PlanCounts counts[PLAN_SMALL];
	__shared__ int state[2];
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
	if (threadIdx.x < 2)
		state[threadIdx.x] = a.state[threadIdx.x];
	for (int b = wave; b < a.n_seqs; b += 16) {
		const PlanCounts n = count_request(a, b);
		if (lane == 0)
			counts[b] = n;
	}
	__syncthreads();
	const Ring ring = ring_of(a, state);
	Before s;
	uint32_t need, want, away;
	const PlanCounts mine = counts_at(counts, 0, a.n_seqs);
	s.add(a, ring, mine, need, want, away);
	// all waves on a few requests: each takes some of their chunks
	const int per = a.n_seqs < 16 ? 16 / max(a.n_seqs, 1) : 1;
	for (int i = wave / per; i < a.n_seqs; i += 16 / per) {
		const PlanCounts own = counts_of(mine, i);
		const Columns k(own.len, own.want);
		const int id = named(a, i, own, k, k.c0 + (own.held ? 0 : wave % per * 64));
		fill_request(a, i, own, ring, sum_at(need, i), sum_at(want, i), sum_at(away, i), wave % per, per, id);
	}
	if (wave == 0 && lane < a.n_seqs)
		a.first[lane] = (int)min(want, s.want);
	finish_plan(a, ring, state, s.need, s.want, s.away, threadIdx.x, 1024);
}

hipError_t launch_plan(const PlanArgs &a, void *work, hipStream_t st)
{
	if (a.n_seqs == 0 || (a.n_seqs <= PLAN_SMALL && a.n_tokens <= 16384 && (size_t)a.n_seqs * a.max_pages <= 32768)) {
		tie_launch(plan_small_kernel, dim3(1), dim3(1024), 0, st, a);
		return hipGetLastError();
	}
	PlanWork w;
	carve_plan(a.n_seqs, (uint8_t *)work, &w);
	const int blocks = (a.n_seqs + PLAN_BLOCK - 1) / PLAN_BLOCK, chunks = a.n_tokens / (64 * PAGE) + 1;
	tie_launch(plan_count_kernel, dim3(blocks), dim3(PLAN_THREADS), 0, st, a, w);
	tie_launch(plan_fill_kernel, dim3(blocks, chunks < 1 ? 1 : chunks < 4 ? chunks : 4), dim3(PLAN_THREADS), 0, st, a, w);
	return hipGetLastError();
}

} // namespace tie
