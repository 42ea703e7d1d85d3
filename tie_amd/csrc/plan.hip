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
// chain of loads (length, table, sums, ring) and the launches, not by bytes.
#include "kv.h"

namespace tie {

constexpr int PLAN_BLOCK = 16; // requests of a workgroup
constexpr int PLAN_SMALL = 64; // requests that one workgroup takes alone

struct PlanCounts {
	int need, want, away; // pages to take, token rows, pages to give back
	int held;             // pages of its new rows that the table names already
};

struct PlanWork {
	PlanCounts *counts; // [n_seqs]
	double *sums;       // [blocks][3] of need, want and away
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
	v.sums = (double *)take(((size_t)n_seqs + PLAN_BLOCK - 1) / PLAN_BLOCK * 3 * sizeof(double));
	v.state = (int *)take(2 * sizeof(int));
	if (w)
		*w = v;
	return off;
}

size_t plan_work_bytes(int n_seqs)
{
	return carve_plan(n_seqs, nullptr, nullptr);
}

// What a request asks for, from its length and count alone.
struct Request {
	int len, want;
	int c0, c1; // columns of its new rows' pages: all but the first may be taken from the ring
	int fresh0; // from this one on
	int r0, r1; // columns whose pages go back
};

__device__ __forceinline__ Request request(const PlanArgs &a, int b)
{
	Request r;
	r.len = a.len[b];
	const int n = a.n_new[b];
	const bool good = r.len >= 0 && n >= 0 && (long long)r.len + n <= (long long)a.max_pages * PAGE;
	r.want = good ? n : 0;
	r.c0 = r.want ? r.len / PAGE : 0;
	r.c1 = r.want ? (r.len + r.want - 1) / PAGE + 1 : 0;
	r.fresh0 = r.want ? r.c0 + (r.len % PAGE != 0) : 0;
	r.r0 = r.r1 = 0;
	if (n < 0) { // ended
		r.r1 = a.max_pages;
	} else if (a.window) {
		// (a page whose last row is below the window of the next token, at row len)
		const long long low = (long long)r.len - a.window + 1;
		r.r0 = a.sinks / PAGE + (a.sinks % PAGE != 0);
		r.r1 = low > 0 ? min((int)(low / PAGE), a.max_pages) : 0;
	}
	return r;
}

__device__ __forceinline__ bool is_page(const PlanArgs &a, int id)
{
	return id >= 0 && id < a.n_pages;
}

// A wave: the counts of request b, and its row of the table copied.
__device__ __forceinline__ PlanCounts count_request(const PlanArgs &a, int b)
{
	const Request r = request(a, b);
	const int32_t *row = a.pages + (size_t)b * a.max_pages;
	int32_t *out = a.pages_out + (size_t)b * a.max_pages;
	const int lane = threadIdx.x & 63;
	const bool copy = out != row;
	PlanCounts n = {0, r.want, 0, 0};
	auto look = [&](int from, int to) {
		for (int c0 = from; c0 < to; c0 += 64) {
			const int c = c0 + lane;
			const int id = c < to ? row[c] : -1;
			if (copy && c < to)
				out[c] = id;
			const bool page = is_page(a, id);
			n.held += __popcll(__ballot(page && c >= r.fresh0 && c < r.c1));
			n.away += __popcll(__ballot(page && c >= r.r0 && c < r.r1));
		}
	};
	if (copy) {
		look(0, a.max_pages);
	} else {
		// (the two ranges do not meet)
		look(r.r0, r.r1);
		look(r.fresh0, r.c1);
	}
	n.need = r.c1 - r.fresh0 - n.held;
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

// A wave: what request b gets, its columns' chunks y, y + ny, ... of 64.  need0, want0,
// away0: the sums over the requests before it.
__device__ __forceinline__ void fill_request(const PlanArgs &a, int b, const PlanCounts &n, const Ring &ring, double need0,
					     double want0, double away0, int y, int ny)
{
	const Request r = request(a, b);
	const int32_t *row = a.pages + (size_t)b * a.max_pages;
	int32_t *out = a.pages_out + (size_t)b * a.max_pages;
	const int lane = threadIdx.x & 63;
	if (r.want && need0 + n.need <= ring.free && want0 + r.want <= a.n_tokens) {
		const int t0 = (int)want0 - r.len; // token row of cache row 0
		// (where the table names some of the pages, the ones before are counted in turn)
		const bool all_fresh = n.held == 0;
		int taken = 0;
		for (int c = r.c0 + (all_fresh ? y * 64 : 0); c < r.c1 && (all_fresh || y == 0); c += all_fresh ? ny * 64 : 64) {
			const int col = c + lane;
			int id = -1;
			if (col < r.c1 && (!all_fresh || col < r.fresh0))
				id = row[col];
			const bool fresh = col >= r.fresh0 && col < r.c1 && !is_page(a, id);
			const unsigned long long set = __ballot(fresh);
			const int rank = all_fresh ? col - r.fresh0 : taken + __popcll(set & ((1ull << lane) - 1));
			if (fresh) {
				id = a.ring[ring_at(a, ring, (int)need0 + rank)];
				out[col] = id;
			}
			taken += __popcll(set);
			if (!a.pos && !a.slot)
				continue;
			const int from = max(r.len, c * PAGE), to = (int)min((long long)r.len + r.want, ((long long)c + 64) * PAGE);
			for (int x0 = from; x0 < to; x0 += 64) {
				const int x = x0 + lane, page = __shfl(id, x / PAGE - c);
				if (x < to) {
					if (a.pos)
						a.pos[t0 + x] = x;
					if (a.slot)
						a.slot[t0 + x] = is_page(a, page) ? page * PAGE + x % PAGE : -1;
				}
			}
		}
	}
	if (y)
		return;
	int gone = 0;
	for (int c = r.r0; c < r.r1; c += 64) {
		const int col = c + lane, id = col < r.r1 ? row[col] : -1;
		const bool away = is_page(a, id);
		const unsigned long long set = __ballot(away);
		const double place = away0 + gone + __popcll(set & ((1ull << lane) - 1));
		if (away && place < ring.room) {
			a.ring[ring_at(a, ring, ring.free + (int)place)] = id;
			out[col] = -1;
		}
		gone += __popcll(set);
	}
}

// What is known when all requests are summed: the last range's end, the token rows
// behind it and the ring's new state.
__device__ __forceinline__ void finish_plan(const PlanArgs &a, const Ring &ring, const int *state, double need, double want, double away,
					    int thread, int threads)
{
	for (int t = (int)want + thread; t < a.n_tokens; t += threads) {
		if (a.pos)
			a.pos[t] = -1;
		if (a.slot)
			a.slot[t] = -1;
	}
	if (thread == 0) {
		const bool none = ring.room == 0 && ring.free == 0; // (no ring)
		const int back = (int)(away < ring.room ? away : ring.room);
		a.first[a.n_seqs] = (int)want;
		a.state_out[0] = none ? state[0] : ring_at(a, ring, (int)need);
		a.state_out[1] = none ? state[1] : ring.free - (int)need + back;
	}
}

__global__ __launch_bounds__(256) void plan_count_kernel(PlanArgs a, PlanWork w)
{
	__shared__ double sum[4][3];
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
	double need = 0.0, want = 0.0, away = 0.0;
	for (int i = wave; i < PLAN_BLOCK; i += 4) {
		const int b = blockIdx.x * PLAN_BLOCK + i;
		if (b >= a.n_seqs)
			break;
		const PlanCounts n = count_request(a, b);
		if (lane == 0)
			w.counts[b] = n;
		need += n.need;
		want += n.want;
		away += n.away;
	}
	if (lane == 0) {
		sum[wave][0] = need;
		sum[wave][1] = want;
		sum[wave][2] = away;
	}
	__syncthreads();
	if (threadIdx.x < 3)
		w.sums[blockIdx.x * 3 + threadIdx.x] = (sum[0][threadIdx.x] + sum[1][threadIdx.x]) + (sum[2][threadIdx.x] + sum[3][threadIdx.x]);
	if (blockIdx.x == 0 && threadIdx.x < 2)
		w.state[threadIdx.x] = a.state[threadIdx.x];
}

__device__ __forceinline__ double of_last(double x)
{
	return of_lane(x, 63);
}

// The sums over the requests before block `block` (a wave, whole numbers in 64-bit
// floats), and of those that are served where the sums pass what there is: cut is set
// then, and every request from there on gets nothing.
struct Before {
	double need, want, away;
	bool cut;
};

__device__ __forceinline__ void add_requests(const PlanArgs &a, const PlanCounts *counts, int b0, int n, const Ring &ring, Before &s,
					     double &my_need, double &my_want, double &my_away, PlanCounts &mine)
{
	const int lane = threadIdx.x & 63;
	mine = PlanCounts{0, 0, 0, 0};
	if (lane < n)
		mine = counts[b0 + lane];
	const double need = running_of<64>((double)mine.need), want = running_of<64>((double)mine.want),
		     away = running_of<64>((double)mine.away);
	my_need = s.need + (need - mine.need);
	my_want = s.want + (want - mine.want);
	my_away = s.away + (away - mine.away);
	s.away += of_last(away);
	if (s.cut)
		return;
	const unsigned long long over = __ballot(s.need + need > ring.free || s.want + want > a.n_tokens);
	if (over) {
		const int l = __builtin_ctzll(over);
		s.need = of_lane(my_need, l);
		s.want = of_lane(my_want, l);
		s.cut = true;
	} else {
		s.need += of_last(need);
		s.want += of_last(want);
	}
}

__global__ __launch_bounds__(256) void plan_fill_kernel(PlanArgs a, PlanWork w)
{
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, block = blockIdx.x;
	const Ring ring = ring_of(a, w.state);
	Before s = {0.0, 0.0, 0.0, false};
	// the blocks before this one, 64 at a time; the one that the cut lies in is looked at
	for (int k0 = 0; k0 < block; k0 += 64) {
		const int k = k0 + lane;
		double x[3] = {0.0, 0.0, 0.0};
		if (k < block)
			for (int i = 0; i < 3; i++)
				x[i] = w.sums[k * 3 + i];
		const double need = running_of<64>(x[0]), want = running_of<64>(x[1]), away = running_of<64>(x[2]);
		const double away_before = s.away;
		if (!s.cut) {
			const unsigned long long over = __ballot(s.need + need > ring.free || s.want + want > a.n_tokens);
			if (over) {
				const int l = __builtin_ctzll(over), b0 = (k0 + l) * PLAN_BLOCK;
				s.need += of_lane(need - x[0], l);
				s.want += of_lane(want - x[1], l);
				double d0, d1, d2;
				PlanCounts mine;
				add_requests(a, w.counts, b0, min(PLAN_BLOCK, a.n_seqs - b0), ring, s, d0, d1, d2, mine);
			} else {
				s.need += of_last(need);
				s.want += of_last(want);
			}
		}
		s.away = away_before + of_last(away);
	}
	const int b0 = block * PLAN_BLOCK, m = min(PLAN_BLOCK, a.n_seqs - b0);
	double need, want, away;
	PlanCounts mine;
	const bool cut_before = s.cut;
	const double want_at = s.want;
	add_requests(a, w.counts, b0, m, ring, s, need, want, away, mine);
	for (int i = wave; i < m; i += 4) {
		PlanCounts n;
		n.need = __builtin_amdgcn_readlane(mine.need, i);
		n.want = __builtin_amdgcn_readlane(mine.want, i);
		n.away = __builtin_amdgcn_readlane(mine.away, i);
		n.held = __builtin_amdgcn_readlane(mine.held, i);
		// (past the cut: sums that nothing fits)
		const double over = cut_before ? __builtin_inf() : of_lane(need, i);
		fill_request(a, b0 + i, n, ring, over, of_lane(want, i), of_lane(away, i), blockIdx.y, gridDim.y);
	}
	if (blockIdx.y == 0 && wave == 0 && lane < m)
		a.first[b0 + lane] = (int)(cut_before ? want_at : want < s.want ? want : s.want);
	if (block == (int)gridDim.x - 1)
		finish_plan(a, ring, w.state, s.need, s.want, s.away, blockIdx.y * 256 + threadIdx.x, gridDim.y * 256);
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
	Before s = {0.0, 0.0, 0.0, false};
	double need, want, away;
	PlanCounts mine;
	add_requests(a, counts, 0, a.n_seqs, ring, s, need, want, away, mine);
	// all waves on a few requests: each takes some of their chunks
	const int per = a.n_seqs < 16 ? 16 / max(a.n_seqs, 1) : 1;
	for (int i = wave / per; i < a.n_seqs; i += 16 / per) {
		PlanCounts n;
		n.need = __builtin_amdgcn_readlane(mine.need, i);
		n.want = __builtin_amdgcn_readlane(mine.want, i);
		n.away = __builtin_amdgcn_readlane(mine.away, i);
		n.held = __builtin_amdgcn_readlane(mine.held, i);
		fill_request(a, i, n, ring, of_lane(need, i), of_lane(want, i), of_lane(away, i), wave % per, per);
	}
	if (wave == 0 && lane < a.n_seqs)
		a.first[lane] = (int)(want < s.want ? want : s.want);
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
	const int blocks = (a.n_seqs + PLAN_BLOCK - 1) / PLAN_BLOCK, chunks = (a.n_tokens + 64 * PAGE - 1) / (64 * PAGE);
	tie_launch(plan_count_kernel, dim3(blocks), dim3(256), 0, st, a, w);
	tie_launch(plan_fill_kernel, dim3(blocks, chunks < 1 ? 1 : chunks < 16 ? chunks : 16), dim3(256), 0, st, a, w);
	return hipGetLastError();
}

} // namespace tie
