// attention.hip -- attention of token rows (single tokens, a drafted tree, a
// causal chunk) over the paged cache, on the f16 matrix cores.
//
//   o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m)
//
// over the rows j that a token sees, in one pass with the running maximum m.
// Queries are F32 and the result is held to F32: each query row is scaled by a
// power of two and split into two f16 parts (22 bits), and so is each weight
// exp(.) before the second product; the cache's f16 values and int8 codes are
// exact in f16, so every product is exact and the sums are F32.
//
// Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T, with
// v_mfma_f32_16x16x32_f16, over 32 or 64 cache rows at a time (KT = 2 or 4
// tiles of 16).  A lane (n = lane % 16, g = lane / 16) of S^T's tiles holds
// query n, and since tile t's row 4 g + i is cache row 4 KT g + 4 t + i, the 4 KT
// rows from 4 KT g on: just what the second product's operand wants of that
// lane.  So the weights never leave their registers, the maximum and sum of a
// query are one value a lane (joined over g), and K and V^T go from the pages
// straight into operands.
//
// The maximum m is a reference only: it moves when some weight would pass
// 2^MOVE, so most steps need no exchange between lanes and leave O alone.  (int8:
// when some weight times its row's V scale would pass f16; see weigh8.)
//
// Through a window (WIN) a tile walks the pages of the first rows and those from its
// lowest visible row on, and masks what lies beside them: the same kernels, with
// the same bounds (61 f16 tokens over 4096 rows of up to 30000, 481 MB: 92 us, 5.2 TB/s;
// a chunk of 4096 over 1024, 69 GFLOP: 142 us).
#include <type_traits>

#include "kv.h"

namespace tie {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float MOVE = 3.0f;       // log2 of the largest weight
constexpr float P_LOG2 = 12.0f;    // weights times 2^12 stay below the f16 limit, their second parts above the subnormals
constexpr float V_UP = 0x1p12f;    // int8: V scales times this (those of a trained layer's values are then about 1)
constexpr float SCALE_LOW = -90.0f; // log2 of the smallest of them that the weights' reference goes by
constexpr float SUM_MOST = 0x1p107f; // of a step's weights before their V scales: 16 rows of SCALE_LOW and 2^(P_LOG2 + 1)

// four int8 codes to f16: 1024 + (code + 128) is the f16 0x6400 | byte, from
// which 1152 is taken exactly
__device__ __forceinline__ void codes4(uint32_t w, h2 &lo, h2 &hi)
{
	w ^= 0x80808080u;
	const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
	lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
	hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
}

__device__ __forceinline__ h8 codes8(uint32_t a, uint32_t b)
{
	h2 p0, p1, p2, p3;
	codes4(a, p0, p1);
	codes4(b, p2, p3);
	return (h8){p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

// x as two f16 parts, each rounded to nearest: the rest of the first is at
// most 2^-11 of x and is held to 2^-11 of itself, so hi + lo is x to 2^-22
// (rounding both toward zero is a bias of 2^-21 on weights that are all
// positive)
__device__ __forceinline__ void split2(float x0, float x1, h2 &hi, h2 &lo)
{
	typedef float f2 __attribute__((ext_vector_type(2)));
	hi = __builtin_convertvector((f2){x0, x1}, h2);
	lo = __builtin_convertvector((f2){__builtin_fmaf((float)hi.x, -1.0f, x0), __builtin_fmaf((float)hi.y, -1.0f, x1)}, h2);
}

// 16 bytes for each lane from base (the same in all lanes) + off to lds + 16 *
// lane (lds: the same in all lanes).  In assembly, so that the compiler does not
// hold back reads of the other buffer for it; the caller waits (s_waitcnt)
// before the barrier that hands the buffer over.
__device__ __forceinline__ void load_lds16(const void *base, uint32_t off, const void *lds)
{
	const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds); // (the low half of a shared address is its offset)
	asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(to) : "memory", "m0");
}

// x of lane N of the lane's group of 16
template <int N> __device__ __forceinline__ float lane16(float x)
{
	return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x150 + N, 0xf, 0xf, true));
}

// v[t][i] *= the s of lane 4 t + i of the group of 16: a lane's 4 KT rows times
// their scales, of which each lane holds one
template <int KT> __device__ __forceinline__ void times_rows(float (&v)[4 * KT], float s)
{
	v[0] *= lane16<0>(s), v[1] *= lane16<1>(s), v[2] *= lane16<2>(s), v[3] *= lane16<3>(s);
	v[4] *= lane16<4>(s), v[5] *= lane16<5>(s), v[6] *= lane16<6>(s), v[7] *= lane16<7>(s);
	if constexpr (KT == 4) {
		v[8] *= lane16<8>(s), v[9] *= lane16<9>(s), v[10] *= lane16<10>(s), v[11] *= lane16<11>(s);
		v[12] *= lane16<12>(s), v[13] *= lane16<13>(s), v[14] *= lane16<14>(s), v[15] *= lane16<15>(s);
	}
}

// a pointer that is the same in all lanes, in scalar registers
__device__ __forceinline__ const uint8_t *uniform(const uint8_t *p)
{
	const uint64_t x = (uint64_t)p;
	const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
	return (const uint8_t *)((uint64_t)hi << 32 | lo);
}

// max over the four lanes of a query (lane, +16, +32, +48)
__device__ __forceinline__ float max_g(float x)
{
	x = __builtin_fmaxf(x, __shfl_xor(x, 16));
	return __builtin_fmaxf(x, __shfl_xor(x, 32));
}

__device__ __forceinline__ float sum_g(float x)
{
	x += __shfl_xor(x, 16);
	return x + __shfl_xor(x, 32);
}

// 2^(floor(log2 x)) of a finite x > 0
__device__ __forceinline__ float pow2_below(float x)
{
	return __uint_as_float(__float_as_uint(x) & 0x7f800000u);
}

__device__ __forceinline__ int div_up(int a, int b)
{
	return (int)(((uint32_t)a + (uint32_t)b - 1) / (uint32_t)b);
}

// How the work of a call is cut: sequence b has tiles(b) row tiles for each kv
// head, each over pages(b) pages, in parts of as many pages -- one unit of work
// (a workgroup) for each.  Every workgroup finds the cut by itself from
// the lengths on the device, so that neither a copy to the host nor a launch
// for a plan stands before the attention and captured calls follow the lengths.
struct Cut {
	// (grain, least and rows are powers of two: shifts, where 64-bit divisions are a sixth of
	// the kernels' instructions, on the way to a unit's first page)
	int cap;   // units that run at once: at most so many where tiles are cut
	int full;  // so many tiles are not cut
	int grain; // pages that are not cut
	int least; // grains of a unit, at least
	int alone; // so few grains of a tile are one unit
	int whole; // tiles are not cut at all
	int rows;  // query rows of a tile
};

struct Unit {
	int b, tile, head, part, parts, t0, n, len;
	int base, tile_at; // the first unit of the sequence, and the tile's place among its tiles
};

// (in 64-bit floats: exact, and without the LDS instructions of a shuffle)
__device__ __forceinline__ int wave_sum(int x)
{
	return (int)wave_total((double)x);
}

// The first row that a token at row `stand` sees through a window, 0 or more.
__device__ __forceinline__ int window_low(int stand, int window)
{
	const long long low = (long long)stand - window + 1;
	return low > 0 ? (int)low : 0;
}

// The pages of a tile that sees nothing below row `low` but the first rows: page i
// of them is page i of the sequence below `sinks`, else i + skip.  all: the pages of
// the sequence up to the last that the tile sees.
struct Span {
	int sinks, skip, pages;
	__device__ __forceinline__ int page(int i) const
	{
		return i < sinks ? i : i + skip;
	}
};

__device__ __forceinline__ Span window_span(int low, int sinks, int all)
{
	const int from = min(low / PAGE, all);
	Span w;
	w.sinks = min(div_up(sinks, PAGE), from);
	w.skip = from - w.sinks;
	w.pages = all - w.skip;
	return w;
}

template <bool WIN>
__device__ __forceinline__ void seq_work(const KvSeqs &s, const AttnArgs &a, int b, int group, int rows, int &t0, int &n, int &len,
					 int &tiles, int &pages)
{
	t0 = n = len = tiles = pages = 0;
	if (b >= s.n_seqs)
		return;
	len = s.len[b];
	seq_tokens(s, b, t0, n);
	if (n == 0)
		return;
	tiles = (int)(((long long)n * group + rows - 1) >> __builtin_ctz(rows));
	pages = seq_fits(s, len, n) ? (len + n + PAGE - 1) / PAGE : 1;
	if (WIN && seq_fits(s, len, n)) {
		// what the first tile sees, and no tile more than these: its tokens' windows
		// together, on one page more than they fill
		const int all = pages;
		pages = window_span(window_low(len, a.window), a.sinks, all).pages;
		if (tiles > 1 && !a.mask) {
			const long long span = (long long)a.window + (rows + group - 2) / group;
			const long long most = div_up(a.sinks, PAGE) + span / PAGE + 2;
			pages = (int)(most < all ? most : all);
		}
	}
}

// x / 2^k, rounded up, for a divisor of 2^k
__device__ __forceinline__ int shift_up(int x, int by)
{
	return (int)(((uint32_t)x + (uint32_t)by - 1) >> __builtin_ctz(by));
}

// Parts of a tile for a grain of its pages, so that no more than cap units come
// (0: whole tiles; so where the tiles alone fill the card).  The first block of
// 64 sequences is in the wave's lanes already.
__device__ __forceinline__ int tile_parts(const Cut &cut, int pages, float rate)
{
	const int grains = shift_up(pages, cut.grain), most = grains >> __builtin_ctz(cut.least), p = (int)((float)grains * rate + 0.5f);
	return p < 2 || grains <= cut.alone ? 1 : p < most ? p : most;
}

template <bool WIN>
__device__ __forceinline__ float part_rate(const KvSeqs &s, const AttnArgs &a, int kvh, int group, const Cut &cut, int tiles0,
					   int pages0)
{
	if (cut.whole)
		return 0.0f;
	const int lane = threadIdx.x & 63;
	auto over = [&](auto f) { // the sum of f(tiles, pages) over all sequences
		double x = f(tiles0, pages0);
		for (int b = 64 + lane; b < s.n_seqs; b += 64) {
			int t0, n, len, tiles, pages;
			seq_work<WIN>(s, a, b, group, cut.rows, t0, n, len, tiles, pages);
			x += f(tiles, pages);
		}
		return s.n_seqs > 1 ? wave_total(x) : of_lane(x, 0);
	};
	const int cap = cut.cap / kvh > 0 ? cut.cap / kvh : 1; // for one kv head
	if (over([](int t, int) { return t; }) * kvh >= cut.full)
		return 0.0f;
	// the nearest number to each tile's share; a little less where those are too many
	float rate = (float)(cap / over([&](int t, int p) { return (double)t * shift_up(p, cut.grain); }));
	for (int i = 0; i < 16; i++) {
		if (over([&](int t, int p) { return t * tile_parts(cut, p, rate); }) <= cap)
			return rate;
		rate *= 0.92f;
	}
	return 0.0f;
}

// The unit of workgroup `index`; false past the last.  Units of a sequence:
// kv heads innermost (workgroups go to the dies in turn: a die then has few
// heads' pages in its L2), then parts, then tiles.
template <bool WIN>
__device__ __forceinline__ bool find_unit(const KvSeqs &s, const AttnArgs &a, int kvh, int group, const Cut &cut, int index, Unit &u)
{
	const int lane = threadIdx.x & 63;
	int t0, n, len, tiles, pages;
	seq_work<WIN>(s, a, lane, group, cut.rows, t0, n, len, tiles, pages);
	const float rate = part_rate<WIN>(s, a, kvh, group, cut, tiles, pages);
	int before = 0;
	for (int b0 = 0;;) {
		const int parts = tiles ? tile_parts(cut, pages, rate) : 0, mine = tiles * parts * kvh;
		const int incl = s.n_seqs > 1 ? (int)running_of<64>((double)mine) : mine;
		const unsigned long long past = __ballot(before + incl > index);
		if (past) {
			const int l = __builtin_ctzll(past);
			auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
			u.b = b0 + l;
			u.base = before + of(incl - mine);
			u.parts = of(parts);
			const int at = index - u.base;
			u.head = (uint32_t)at % (uint32_t)kvh;
			u.part = (uint32_t)at / (uint32_t)kvh % (uint32_t)u.parts;
			// (causal: the last tiles have the most pages; they start first)
			u.tile_at = (uint32_t)at / (uint32_t)kvh / (uint32_t)u.parts;
			u.tile = of(tiles) - 1 - u.tile_at;
			u.t0 = of(t0);
			u.n = of(n);
			u.len = of(len);
			u.base = __builtin_amdgcn_readfirstlane(u.base);
			u.b = __builtin_amdgcn_readfirstlane(u.b);
			u.head = __builtin_amdgcn_readfirstlane(u.head);
			u.part = __builtin_amdgcn_readfirstlane(u.part);
			u.tile = __builtin_amdgcn_readfirstlane(u.tile);
			u.tile_at = __builtin_amdgcn_readfirstlane(u.tile_at);
			return true;
		}
		before += __builtin_amdgcn_readlane(incl, 63);
		b0 += 64;
		if (b0 >= s.n_seqs)
			return false;
		seq_work<WIN>(s, a, b0 + lane, group, cut.rows, t0, n, len, tiles, pages);
	}
}

// The first page of the unit's part, and behind its last.  all: the pages that the
// tile's parts share out.
__device__ __forceinline__ void part_pages(const Cut &cut, const Unit &u, int all, int pages, int &p0, int &p1)
{
	// (in grains where a part has few of them, else to the page)
	const int grain = all / u.parts < 4 * cut.grain ? cut.grain : 1;
	const int grains = shift_up(all, grain), q = grains / u.parts, r = grains % u.parts;
	p0 = (u.part * q + min(u.part, r)) * grain;
	p1 = min(pages, p0 + (q + (u.part < r)) * grain);
}

// Which of the 64 rows of the page at row `start` a token sees: all committed
// ones, and of the sequence's own tokens those of its mask, or (causal) those
// up to itself.  node < 0: none.
__device__ __forceinline__ uint64_t sees(const AttnArgs &a, const Unit &u, int node, int start)
{
	if (node < 0)
		return 0;
	const int rel = start - u.len; // the page's first row as a node
	if (rel <= -PAGE)
		return ~0ull;
	auto below = [](long long n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
	if (!a.mask)
		return below((long long)node + 1 - rel);
	uint64_t w = 0;
	const uint64_t *m = a.mask + (size_t)(u.t0 + node) * a.mask_words;
	const int word = rel >> 6, sh = rel & 63; // (floors)
	if (word >= 0 && word < a.mask_words)
		w = m[word] >> sh;
	if (sh && word + 1 >= 0 && word + 1 < a.mask_words)
		w |= m[word + 1] << (64 - sh);
	w &= below((long long)u.n - rel); // no bit names a node that is not there
	return w | below(-(long long)rel);
}

// The same through a window whose lowest row is `low`: committed rows below it are
// not seen but the first a.sinks; of the sequence's own tokens the mask's stand as
// they are, and a causal row's go by the window too.
template <bool WIN>
__device__ __forceinline__ uint64_t sees_through(const AttnArgs &a, const Unit &u, int node, int low, int start)
{
	uint64_t w = sees(a, u, node, start);
	if (WIN && w) {
		auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
		uint64_t near = ~below(low - start) | below(a.sinks - start);
		if (a.mask)
			near |= ~below(u.len - start);
		w &= near;
	}
	return w;
}

// The lowest row that a token sees, but for the first ones.
__device__ __forceinline__ int low_of(const AttnArgs &a, const Unit &u, int node)
{
	return window_low(a.at ? a.at[u.t0 + node] : u.len + node, a.window);
}

// min and max over the wave
__device__ __forceinline__ int wave_least(int x)
{
#pragma unroll
	for (int k = 1; k < 64; k <<= 1)
		x = min(x, __shfl_xor(x, k));
	return __builtin_amdgcn_readfirstlane(x);
}

// The least and the largest `low` of a tile's tokens, nodes n0 .. n1.
__device__ __forceinline__ void tile_lows(const AttnArgs &a, const Unit &u, int n0, int n1, int &least, int &most)
{
	if (!a.at) {
		least = window_low(u.len + n0, a.window);
		most = window_low(u.len + n1, a.window);
		return;
	}
	int lo = 0x7fffffff, hi = 0;
	for (int i = n0 + (int)(threadIdx.x & 63); i <= n1; i += 64) {
		const int x = low_of(a, u, i);
		lo = min(lo, x);
		hi = max(hi, x);
	}
	least = wave_least(lo);
	most = -wave_least(-hi);
}

// Results of a part, for each row of its tile: O [HD], the maximum, the sum.
constexpr int part_row(int hd)
{
	return hd + 4; // (16-byte rows)
}

// A token row's query for one lane of an operand: 8 values of each K step.
// PAIRS: int8 rows straight from memory come 16 codes to a lane.
template <int HD, bool PAIRS>
__device__ __forceinline__ void fetch_query(const AttnArgs &a, const Unit &u, int node, int head, int g, float (&x)[HD / 32][8])
{
	const float *q = a.q + (size_t)(u.t0 + (node < 0 ? 0 : node)) * a.q_stride + (size_t)head * HD;
	const bool vec = (((uintptr_t)a.q | a.q_stride * 4) & 15) == 0;
#pragma unroll
	for (int k = 0; k < HD / 32; k++) {
		const float *from = q + (PAIRS ? (k >> 1) * 64 + g * 16 + (k & 1) * 8 : k * 32 + g * 8);
		if (vec) {
			const f4 x0 = reinterpret_cast<const f4 *>(from)[0], x1 = reinterpret_cast<const f4 *>(from)[1];
#pragma unroll
			for (int j = 0; j < 4; j++) {
				x[k][j] = x0[j];
				x[k][4 + j] = x1[j];
			}
		} else {
#pragma unroll
			for (int j = 0; j < 8; j++)
				x[k][j] = from[j];
		}
	}
}

// The operand's two parts, of the query scaled to below 2^10; qs: what the
// products are multiplied by (with log2 e: exp2 for exp), positive (the scale's
// sign is in the query).
template <int HD>
__device__ __forceinline__ void split_query(const AttnArgs &a, int node, float (&x)[HD / 32][8], h8 (&qh)[HD / 32],
					    h8 (&ql)[HD / 32], float &qs)
{
	float m = 0.0f;
#pragma unroll
	for (int k = 0; k < HD / 32; k++)
#pragma unroll
		for (int j = 0; j < 8; j++) {
			x[k][j] = node < 0 ? 0.0f : x[k][j];
			m = __builtin_fmaxf(m, __builtin_fabsf(x[k][j]));
		}
	m = max_g(m);
	const float p2 = m >= 1e-30f && m < __builtin_inff() ? pow2_below(m) : 1.0f;
	const float up = __builtin_copysignf(512.0f / p2, a.scale);
	// (not 0: the score of a row that is not seen, -inf, stays that)
	qs = __builtin_fmaxf(__builtin_fabsf(a.scale) * 1.44269504088896f * (p2 * (1.0f / 512.0f)), 1.2e-38f);
#pragma unroll
	for (int k = 0; k < HD / 32; k++)
#pragma unroll
		for (int j = 0; j < 8; j += 2) {
			h2 hi, lo;
			split2(x[k][j] * up, x[k][j + 1] * up, hi, lo);
			qh[k][j] = hi.x, qh[k][j + 1] = hi.y;
			ql[k][j] = lo.x, ql[k][j + 1] = lo.y;
		}
}

// The running state of 16 query rows: a lane's query's reference (log2 of what
// the lane's share of the sum, and O^T, are multiples of).
template <int HD>
struct Rows {
	float mx = -__builtin_inff(), sum = 0.0f;
	f4 o[HD / 16];
};

// The weights w in the two f16 parts of the second product's operand.
template <int KT> __device__ __forceinline__ void split_weights(const float (&w)[4 * KT], h8 (&ph)[KT / 2], h8 (&pl)[KT / 2])
{
#pragma unroll
	for (int e = 0; e < 4 * KT; e += 2) {
		h2 hi, lo;
		split2(w[e], w[e + 1], hi, lo);
		ph[e / 8][e % 8] = hi.x, ph[e / 8][e % 8 + 1] = hi.y;
		pl[e / 8][e % 8] = lo.x, pl[e / 8][e % 8 + 1] = lo.y;
	}
}

// f16 rows: from the products sc of 16 KT cache rows to the weights' two f16
// parts for the second product; the state's reference and sum, and O where the
// reference moved.  whole: every query of the wave sees all the rows; else bits:
// which of the lane's 4 KT rows its query sees (the weights of the others are
// 0).  Weights, O and sum carry 2^P_LOG2, by way of the exponent, until
// finish().
template <int HD, int KT>
__device__ __forceinline__ void weigh(Rows<HD> &r, const f4 (&sc)[KT], float qs, bool whole, uint32_t bits, h8 (&ph)[KT / 2],
				      h8 (&pl)[KT / 2])
{
	float w[4 * KT];
#pragma unroll
	for (int e = 0; e < 4 * KT; e++)
		w[e] = sc[e / 4][e % 4];
	if (!whole)
#pragma unroll
		for (int e = 0; e < 4 * KT; e++)
			if (!(bits >> e & 1))
				w[e] = -__builtin_inff();
	float top = -__builtin_inff();
#pragma unroll
	for (int e = 0; e < 4 * KT; e++)
		top = __builtin_fmaxf(top, w[e]);
	top *= qs;
	if (__any(top > r.mx + MOVE)) {
		top = __builtin_fmaxf(r.mx, max_g(top));
		const float f = r.mx == top ? 1.0f : __builtin_amdgcn_exp2f(r.mx - top);
		r.mx = top;
		r.sum *= f;
#pragma unroll
		for (int m = 0; m < HD / 16; m++)
			r.o[m] *= f;
	}
	const float base = (r.mx == -__builtin_inff() ? 0.0f : r.mx) - P_LOG2;
#pragma unroll
	for (int e = 0; e < 4 * KT; e++) {
		w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[e], qs, -base));
		r.sum += w[e];
	}
	split_weights<KT>(w, ph, pl);
}

// int8 rows: the same.  ks and vs are the K and V scale of the lane's row (lane
// 4 t + i of 16: row 4 t + i of the group's), vs times `up` and finite unless
// whole.  The second product's weights are y = 2^(score - mx) vs, and it is y that
// has to stay in f16's range, though V scales may lie any number of binades apart:
// so the reference is not the largest score but the largest y of the rows that the
// query sees (held at 2^P_LOG2 when it moves, and moved past 2^15).  A row that a
// query does not see, or that weighs nothing, has no part in it, whatever its
// scale.  Rows of scales below 2^SCALE_LOW count as that for the reference alone,
// so that the sum stays in F32's range.  The reference is a whole number: what
// moves with it stays exact.
//
// The weights are formed with the reference as it stands, and again where it turns
// out to have to move (a few times in a pass): no maximum of the scores is
// needed in the common path.
template <int HD, int KT>
__device__ __forceinline__ void weigh8(Rows<HD> &r, const f4 (&sc)[KT], float ks, float vs, float qs, bool whole, uint32_t bits,
				       h8 (&ph)[KT / 2], h8 (&pl)[KT / 2])
{
	float s[4 * KT], w[4 * KT], add, most;
#pragma unroll
	for (int e = 0; e < 4 * KT; e++)
		s[e] = sc[e / 4][e % 4];
	times_rows<KT>(s, ks);
	if (!whole)
#pragma unroll
		for (int e = 0; e < 4 * KT; e++)
			if (!(bits >> e & 1))
				s[e] = -__builtin_inff();
	auto weights = [&](float base) {
		add = most = 0.0f;
#pragma unroll
		for (int e = 0; e < 4 * KT; e++) {
			w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], qs, -base));
			add += w[e];
		}
		times_rows<KT>(w, vs);
#pragma unroll
		for (int e = 0; e < 4 * KT; e++)
			most = __builtin_fmaxf(most, __builtin_fabsf(w[e]));
	};
	weights(r.mx); // (before the first row: not a number, or infinite)
	if (__any(!(add <= SUM_MOST) || most > 32768.0f)) {
		// log2 of y without the reference
		float y[4 * KT], top = -__builtin_inff();
#pragma unroll
		for (int e = 0; e < 4 * KT; e++)
			y[e] = 1.0f;
		times_rows<KT>(y, __builtin_fminf(__builtin_fmaxf(__builtin_amdgcn_logf(__builtin_fabsf(vs)), SCALE_LOW), 100.0f));
#pragma unroll
		for (int e = 0; e < 4 * KT; e++)
			top = __builtin_fmaxf(top, __builtin_fmaf(s[e], qs, y[e]));
		top = __builtin_fmaxf(r.mx, __builtin_ceilf(max_g(top)) - P_LOG2);
		const float f = __builtin_ldexpf(1.0f, (int)__builtin_fmaxf(r.mx - top, -200.0f));
		r.mx = top;
		r.sum *= f;
#pragma unroll
		for (int m = 0; m < HD / 16; m++)
			r.o[m] *= f;
		weights(top == -__builtin_inff() ? 0.0f : top);
	}
	r.sum += add;
	split_weights<KT>(w, ph, pl);
}

// The V scale of a lane's row as weigh8() takes it.  Where one is above 2^60 the
// factor `up` (the same in all lanes) goes down by 2^64, once, and the references
// with it (by less where the sum would leave F32's range: then all values so far
// are below 2^SCALE_LOW of the present one).
template <int HD, int NT> __device__ __forceinline__ float scale_up(float vs, float &up, Rows<HD> (&r)[NT])
{
	if (up == V_UP && __any(__builtin_fabsf(vs) > 0x1p60f / V_UP)) {
		up = V_UP * 0x1p-64f;
#pragma unroll
		for (int t = 0; t < NT; t++) {
			const int d = min(max(104 + 127 - (int)(__float_as_uint(max_g(r[t].sum)) >> 23 & 0xff), 0), 64);
			r[t].mx -= (float)d;
			r[t].sum = __builtin_ldexpf(r[t].sum, d);
#pragma unroll
			for (int m = 0; m < HD / 16; m++)
				r[t].o[m] *= __builtin_ldexpf(1.0f, d - 64);
		}
	}
	return vs * up;
}

// At the end: the sum over a query's four lanes (returned), and what O is to be
// multiplied by.  int8: O and the sum as multiples of another 2^mx, so that the
// sum is about 1.
template <int HD, bool I8> __device__ __forceinline__ float finish(Rows<HD> &r, float up, float &back)
{
	const float total = sum_g(r.sum);
	if (!I8) {
		back = 1.0f / (1 << (int)P_LOG2);
		return total * back;
	}
	back = 1.0f;
	const bool any = total > 0.0f && total < __builtin_inff();
	const int k = any ? (int)(__float_as_uint(total) >> 23) - 127 : 0, k_up = (int)(__float_as_uint(up) >> 23) - 127;
	r.mx = any ? r.mx + (float)k : r.mx;
#pragma unroll
	for (int m = 0; m < HD / 16; m++)
#pragma unroll
		for (int i = 0; i < 4; i++)
			r.o[m][i] = __builtin_ldexpf(r.o[m][i], -k - k_up);
	return __builtin_ldexpf(total, -k);
}

// int8 rows of which some queries do not see some, or that hold nothing (!
// there): a V scale that is not finite would reach queries that do not see its
// row as 0 * inf.  The K scale takes its place, so that those that see the row
// get NaN.
__device__ __forceinline__ void guard_scales(float &ks, float &vs, bool there)
{
	if (!(__builtin_fabsf(vs) < __builtin_inff()) || !there) {
		vs = 0.0f;
		ks = __builtin_nanf("");
	}
}

// f16 values w of 32 rows that not every query sees, an operand of column tile
// m: a value that is not finite would reach queries that do not see its row as 0
// * inf.  Such values are taken out and come back for those that see them.  v:
// the page's values of this head, the rows from `row0` on, `end` of which hold
// anything; vis: the rows of these 32 that the lane's query sees.
template <int HD, int NT>
__device__ __forceinline__ void guard_values(u4 &w, const uint8_t *v, int row0, int m, int g, int end,
					     const uint32_t (&vis)[NT], Rows<HD> (&r)[NT])
{
	uint32_t odd = 0;
#pragma unroll
	for (int e = 0; e < 4; e++) {
		uint32_t x = w[e];
		if ((x & 0x7c00u) == 0x7c00u) {
			x &= 0xffff0000u;
			odd |= 1u << (2 * e);
		}
		if ((x & 0x7c000000u) == 0x7c000000u) {
			x &= 0xffffu;
			odd |= 2u << (2 * e);
		}
		w[e] = x;
	}
	if (!__any(odd != 0))
		return;
	for (int row = 0; row < min(end, 32); row++) {
		const int src = (row >> 3) * 16; // the lane group that has the row
#pragma unroll
		for (int i = 0; i < 4; i++) {
			// (column 4 g + i of the tile: this lane's in O^T)
			if (!(__shfl(odd, src + 4 * g + i) >> (row & 7) & 1))
				continue;
			const float x = (float)reinterpret_cast<const _Float16 *>(v)[(m * 16 + 4 * g + i) * PAGE + row0 + row];
#pragma unroll
			for (int t = 0; t < NT; t++)
				if (vis[t] >> row & 1)
					r[t].o[m][i] = x != x ? x : r[t].o[m][i] + x;
		}
	}
}

// The values of a page that are not finite, to the queries that see their
// rows (inf and NaN stay what they are whatever a weight).
template <int HD, int NT>
__device__ __forceinline__ void give_back(const uint8_t *v, int g, int end, const uint64_t (&vis)[NT], Rows<HD> (&r)[NT])
{
	for (int row = 0; row < min(end, PAGE); row++)
#pragma unroll
		for (int m = 0; m < HD / 16; m++)
#pragma unroll
			for (int i = 0; i < 4; i++) {
				const float x = (float)reinterpret_cast<const _Float16 *>(v)[(m * 16 + 4 * g + i) * PAGE + row];
				if (__builtin_fabsf(x) < __builtin_inff())
					continue;
#pragma unroll
				for (int t = 0; t < NT; t++)
					if (vis[t] >> row & 1)
						r[t].o[m][i] += x;
			}
}

// ---------------------------------------------------------------- few rows
// A workgroup: 16 query rows (a row: a token and one query head of the unit's
// kv head), its 8 waves taking the unit's pages in turn.  Bound by the stream of
// pages: a wave requests a page's K as soon as the products with the last one's
// are done and its V as soon as O has taken the last one's, so that one of the
// two is always under way, at 2 waves on a SIMD (16 tokens over 32000 int8 rows,
// 276 MB: 55 us, 5.0 TB/s).  Short ones: by the chain of lengths, page numbers,
// pages, products, join (one token over 500 rows 11 us, of which the eight waves'
// 128 KB are 2 us of loads into one CU).
constexpr int FEW_ROWS = 16, FEW_WAVES = 8, FEW_CAP = 256;
constexpr int FEW_PARTS = FEW_CAP + 32; // parts of a tile, at most

// two floats past the dies' caches
__device__ __forceinline__ void put_pair(uint64_t *p, float x, float y)
{
	__hip_atomic_store(p, (uint64_t)__float_as_uint(x) | (uint64_t)__float_as_uint(y) << 32, __ATOMIC_RELAXED,
			   __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void get_pair(const uint64_t *p, float &x, float &y)
{
	const uint64_t v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
	x = __uint_as_float((uint32_t)v);
	y = __uint_as_float((uint32_t)(v >> 32));
}

template <int HD, bool I8, bool WIN>
__global__ __launch_bounds__(64 * FEW_WAVES, 2) void attn_few_kernel(KvLayer c, KvSeqs s, AttnArgs a, Cut cut, float *part,
								       int *count)
{
	constexpr int KS = HD / 32, MT = HD / 16, R = FEW_ROWS, WK = FEW_WAVES;
	constexpr int KT = I8 ? 4 : 2;       // a step: a page of int8, half a page of f16 (16 KB of K and V at HD = 128)
	constexpr int SP = 4 / KT;           // steps of a page
	constexpr int KL = I8 ? KS / 2 : KS; // 16-byte loads of a lane for one of a step's K tiles
	extern __shared__ __attribute__((aligned(16))) float lds[];
	const int group = a.n_heads / c.kvh;
	Unit u;
	if (!find_unit<WIN>(s, a, c.kvh, group, cut, blockIdx.x, u))
		return;
	const int lane = threadIdx.x & 63, n16 = lane & 15, g = lane >> 4;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	bool bad = !seq_fits(s, u.len, u.n); // the rows cannot be read: the result is NaN

	const int row = u.tile * R + n16;
	const int node = row / group < u.n ? row / group : -1;
	// (causal: nothing behind the tile's last token is seen)
	const int last = a.mask ? u.n : min(u.n, (u.tile * R + R - 1) / group + 1);
	int pages = bad ? 0 : (u.len + last + PAGE - 1) / PAGE, shared = (u.len + u.n + PAGE - 1) / PAGE;
	Span span = {0, 0, 0};
	int low = 0;
	if (WIN) {
		int least, most;
		const int n0 = u.tile * R / group, n1 = min(u.n, (u.tile * R + R - 1) / group + 1) - 1;
		tile_lows(a, u, n0, n1, least, most);
		low = node < 0 ? 0 : low_of(a, u, node);
		// (a mask names its own tokens whatever the window)
		span = window_span(a.mask ? min(least, u.len) : least, a.sinks, pages);
		shared = pages = span.pages;
	}
	int p0, p1;
	part_pages(cut, u, shared, pages, p0, p1);
	const int steps = (p1 - p0) * SP;

	u4 kr[KT][KL], vr[MT];
	float ks = 0.0f, vs = 0.0f; // int8: the scales of the lane's row
	size_t at = 0; // of the page whose V is in (or on its way to) vr
	auto page = [&](int step) {
		const int p = WIN ? span.page(p0 + step / SP) : p0 + step / SP;
		const int id = __builtin_amdgcn_readfirstlane(page_of(s, c.n_pages, u.b, p * PAGE));
		bad = bad || id < 0;
		return (size_t)(id < 0 ? 0 : id) * c.kvh + u.head;
	};
	auto get_k = [&](size_t pg, int step) {
		const int row0 = step % SP * 32;
#pragma unroll
		for (int kt = 0; kt < KT; kt++) {
			const int q = row0 + (n16 >> 2) * 4 * KT + kt * 4 + (n16 & 3);
			const u4 *p = reinterpret_cast<const u4 *>(c.k + (pg * PAGE + q) * HD * (I8 ? 1 : 2)) + g;
#pragma unroll
			for (int e = 0; e < KL; e++)
				kr[kt][e] = p[e * 4];
		}
		if (I8)
			ks = c.ks[pg * PAGE + lane];
	};
	auto get_v = [&](size_t pg, int step) {
#pragma unroll
		for (int m = 0; m < MT; m++)
			vr[m] = reinterpret_cast<const u4 *>(c.v + (pg * HD + m * 16 + n16) * PAGE * (I8 ? 1 : 2))[step % SP * 4 + g];
		if (I8)
			vs = c.vs[pg * PAGE + lane];
	};
	float x[KS][8];
	fetch_query<HD, I8>(a, u, node, u.head * group + row % group, g, x);
	if (wave < steps) {
		at = page(wave);
		get_k(at, wave);
		get_v(at, wave);
	}
	h8 qh[KS], ql[KS];
	float qs;
	split_query<HD>(a, node, x, qh, ql, qs);
	Rows<HD> r[1];
#pragma unroll
	for (int m = 0; m < MT; m++)
		r[0].o[m] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
	float up = V_UP;

	for (int step = wave; step < steps; step += WK) {
		const int start = (WIN ? span.page(p0 + step / SP) : p0 + step / SP) * PAGE, row0 = step % SP * 32;
		const int end = u.len + u.n - start - row0;
		const uint64_t vis = sees_through<WIN>(a, u, node, low, start) >> row0;
		constexpr uint64_t all = KT == 4 ? ~0ull : 0xffffffffull;
		const bool whole = __all((vis & all) == all || node < 0);
		const bool more = step + WK < steps;
		const size_t next = more ? page(step + WK) : at;
		f4 sc[KT];
#pragma unroll
		for (int kt = 0; kt < KT; kt++) {
			f4 lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
#pragma unroll
			for (int k = 0; k < KS; k++) {
				h8 kf;
				if constexpr (I8) {
					const u4 w = kr[kt][k >> 1];
					kf = k & 1 ? codes8(w.z, w.w) : codes8(w.x, w.y);
				} else {
					kf = __builtin_bit_cast(h8, kr[kt][k]);
				}
				lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[k], lo, 0, 0, 0);
				hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[k], hi, 0, 0, 0);
			}
			sc[kt] = lo + hi;
		}
		float kk = ks;
		if (more)
			get_k(next, step + WK);
		h8 ph[KT / 2], pl[KT / 2];
		if (I8) {
			if (!whole)
				guard_scales(kk, vs, lane < end);
			weigh8<HD, KT>(r[0], sc, kk, scale_up<HD, 1>(vs, up, r), qs, whole, (uint32_t)(vis >> (4 * KT * g)), ph, pl);
		} else {
			weigh<HD, KT>(r[0], sc, qs, whole, (uint32_t)(vis >> (4 * KT * g)), ph, pl);
		}
#pragma unroll
		for (int m = 0; m < MT; m++) {
			if constexpr (I8) {
				const h8 v0 = codes8(vr[m].x, vr[m].y), v1 = codes8(vr[m].z, vr[m].w);
				r[0].o[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0], r[0].o[m], 0, 0, 0);
				r[0].o[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[KT / 2 - 1], r[0].o[m], 0, 0, 0);
				r[0].o[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0], r[0].o[m], 0, 0, 0);
				r[0].o[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[KT / 2 - 1], r[0].o[m], 0, 0, 0);
			} else {
				u4 w = vr[m];
				if (!whole) {
					const uint32_t seen[1] = {(uint32_t)vis};
					guard_values<HD, 1>(w, c.v + at * HD * PAGE * 2, row0, m, g, end, seen, r);
				}
				const h8 v0 = __builtin_bit_cast(h8, w);
				r[0].o[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0], r[0].o[m], 0, 0, 0);
				r[0].o[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0], r[0].o[m], 0, 0, 0);
			}
		}
		if (more)
			get_v(next, step + WK);
		at = next;
	}
	float back;
	const float total = finish<HD, I8>(r[0], up, back);

	// join the waves: each puts its rows into LDS ([wave][row][HD + 4])
	constexpr int LR = part_row(HD);
	float *mine = lds + ((size_t)wave * R + n16) * LR;
#pragma unroll
	for (int m = 0; m < MT; m++)
		*reinterpret_cast<f4 *>(mine + m * 16 + 4 * g) = r[0].o[m] * back;
	if (g == 0) {
		mine[HD] = bad ? __builtin_nanf("") : r[0].mx;
		mine[HD + 1] = bad ? __builtin_nanf("") : total;
	}
	__syncthreads();
	// (pairs of columns: a part's values go by 8 bytes)
	auto out_at = [&](int q) {
		const int to = u.tile * R + q;
		return a.out + (size_t)(u.t0 + to / group) * a.o_stride + (size_t)(u.head * group + to % group) * HD;
	};
	const int live = min(R, u.n * group - u.tile * R); // rows of the tile
	uint64_t *mine64 = reinterpret_cast<uint64_t *>(part + (size_t)blockIdx.x * R * LR);
	for (int e = threadIdx.x; e < live * HD / 2; e += 64 * WK) {
		const int q = e / (HD / 2), i = e % (HD / 2);
		float m = -__builtin_inff(), l = 0.0f, x0 = 0.0f, x1 = 0.0f;
#pragma unroll
		for (int w = 0; w < WK; w++)
			m = __builtin_fmaxf(m, lds[((size_t)w * R + q) * LR + HD]);
		const float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
		for (int w = 0; w < WK; w++) {
			const float *from = lds + ((size_t)w * R + q) * LR;
			const float f = __builtin_amdgcn_exp2f(from[HD] - base);
			l += from[HD + 1] * f;
			x0 += from[2 * i] * f;
			x1 += from[2 * i + 1] * f;
		}
		if (u.parts == 1) {
			float *o = out_at(q) + 2 * i;
			o[0] = l == 0.0f ? 0.0f : x0 / l;
			o[1] = l == 0.0f ? 0.0f : x1 / l;
		} else {
			put_pair(mine64 + q * (LR / 2) + i, x0, x1);
			if (i == 0)
				put_pair(mine64 + q * (LR / 2) + HD / 2, m, l);
		}
	}
	if (u.parts == 1)
		return;
	// The last of the tile's parts joins them.  What the parts wrote went past
	// the dies' caches (agent-scope accesses) and is there once the writer's
	// loads and stores are done, which each wave waits for before its
	// workgroup counts; the last one to count leaves the counter as it was, 0.
	asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
	__syncthreads();
	const int u0 = u.base + u.tile_at * u.parts * c.kvh + u.head; // unit of part q: u0 + q kvh
	if ((long long)u0 + (long long)(u.parts - 1) * c.kvh >= gridDim.x || u0 >= WORK_COUNTERS || u.parts > FEW_PARTS)
		return; // (sequences that overlap: more units than the rows can have)
	int *last_one = reinterpret_cast<int *>(lds);
	if (threadIdx.x == 0)
		*last_one = __hip_atomic_fetch_add(count + u0, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == u.parts - 1;
	__syncthreads();
	if (!*last_one)
		return;
	if (threadIdx.x == 0)
		__hip_atomic_store(count + u0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
	__syncthreads();
	const uint64_t *from64 = reinterpret_cast<const uint64_t *>(part + (size_t)u0 * R * LR);
	const size_t step64 = (size_t)c.kvh * R * LR / 2;
	// first the rows' maxima and sums: a row's 32 lanes take parts in turn
	float *fac = lds; // [live][parts up to FEW_PARTS] the parts' factors
	{
		const int q = threadIdx.x / 32, l32 = threadIdx.x % 32;
		if (q < live) {
			float pm[FEW_PARTS / 32], pl[FEW_PARTS / 32], m = -__builtin_inff(), l = 0.0f;
#pragma unroll
			for (int e = 0; e < FEW_PARTS / 32; e++) {
				const int k = e * 32 + l32;
				pm[e] = -__builtin_inff();
				pl[e] = 0.0f;
				if (k < u.parts)
					get_pair(from64 + k * step64 + q * (LR / 2) + HD / 2, pm[e], pl[e]);
			}
#pragma unroll
			for (int e = 0; e < FEW_PARTS / 32; e++)
				m = __builtin_fmaxf(m, pm[e]);
#pragma unroll
			for (int k = 1; k < 32; k <<= 1)
				m = __builtin_fmaxf(m, __shfl_xor(m, k));
			const float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
			for (int e = 0; e < FEW_PARTS / 32; e++) {
				pm[e] = __builtin_amdgcn_exp2f(pm[e] - base);
				l += pl[e] * pm[e];
			}
#pragma unroll
			for (int k = 1; k < 32; k <<= 1)
				l += __shfl_xor(l, k);
			const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
			for (int e = 0; e < FEW_PARTS / 32; e++)
				if (e * 32 + l32 < u.parts)
					fac[q * FEW_PARTS + e * 32 + l32] = l == 0.0f ? 0.0f : pm[e] * inv;
		}
	}
	__syncthreads();
	for (int e = threadIdx.x; e < live * HD / 2; e += 64 * WK) {
		const int q = e / (HD / 2), i = e % (HD / 2);
		float x0 = 0.0f, x1 = 0.0f;
		for (int k0 = 0; k0 < u.parts; k0 += 16) {
			float y0[16], y1[16];
#pragma unroll
			for (int k = 0; k < 16; k++)
				get_pair(from64 + min(k0 + k, u.parts - 1) * step64 + q * (LR / 2) + i, y0[k], y1[k]);
#pragma unroll
			for (int k = 0; k < 16; k++) {
				const float f = k0 + k < u.parts ? fac[q * FEW_PARTS + k0 + k] : 0.0f;
				x0 += k0 + k < u.parts ? y0[k] * f : 0.0f;
				x1 += k0 + k < u.parts ? y1[k] * f : 0.0f;
			}
		}
		float *o = out_at(q) + 2 * i;
		o[0] = x0;
		o[1] = x1;
	}
}

// ---------------------------------------------------------------- many rows
// A workgroup: 32 RG query rows of one kv head, 32 to a wave, all over the same
// pages: a page comes into LDS once (int8 codes as f16), while the one before
// is worked on.  RG = 2: a wave takes half of a page for its rows, and two waves'
// rows are joined at the end.  Bound by the matrix cores and the weights'
// arithmetic: two workgroups on a CU hide less of each other's waits than their
// waves' turns suggest (2.05 us a page of 128 rows for a CU with two, 2.26 alone;
// the matrix instructions are 0.86 of them).
//
// LDS rows are swizzled in 16-byte pieces so that the 8 lanes that read
// together touch all banks: K row r's piece q lies at q ^ f(r), f the lane of
// the operand that reads the row; V column i's at q ^ (i % 8).
constexpr int MANY_WAVES = 4;

// The page table's entries of a unit, a lane each, 64 pages at a time: a page's
// number is then a register away (a load of it stands before the page's own loads
// otherwise: 800 cycles a page; the kernel of few rows has eight waves to hide
// that, and is 0.6 us slower this way).
struct PageIds {
	int first, ids; // pages first .. first + 63
	__device__ __forceinline__ void get(const KvSeqs &s, const Unit &u, const Span &w, int p)
	{
		first = p;
		const int at = w.page(p + (int)(threadIdx.x & 63));
		ids = at < s.max_pages ? s.pages[(size_t)u.b * s.max_pages + at] : -1;
	}
	// the number of page p, p not below the last one asked for; bad: it is none
	__device__ __forceinline__ int of(const KvSeqs &s, const Unit &u, const Span &w, int n_pages, int p, bool &bad)
	{
		if (p - first >= 64)
			get(s, u, w, p);
		const int id = __builtin_amdgcn_readlane(ids, p - first);
		const bool ok = id >= 0 && id < n_pages;
		bad = bad || !ok;
		return ok ? id : 0;
	}
};

template <int HD, bool I8, int RG, bool WIN>
__global__ __launch_bounds__(64 * MANY_WAVES, 2) void attn_many_kernel(KvLayer c, KvSeqs s, AttnArgs a, Cut cut, float *part)
{
	constexpr int KS = HD / 32, MT = HD / 16, R = 32 * RG, NT = 2, KT = 2, E = I8 ? 1 : 2;
	constexpr int NL = PAGE * HD * E / 16 / 256; // 16-byte pieces of a page's K (and V) for a thread
	constexpr int KP = HD / 8, VP = PAGE / 8;    // pieces of a K row and of a V column in LDS
	__shared__ __attribute__((aligned(1024))) _Float16 lk[2][PAGE * HD], lv[2][PAGE * HD];
	__shared__ __attribute__((aligned(16))) float lsc[2][2][PAGE];
	const int group = a.n_heads / c.kvh;
	Unit u;
	// (whole tiles in causal order, two to a CU: the longest with the shortest)
	int index = blockIdx.x;
	if (cut.whole && (int)gridDim.x <= cut.cap && index >= cut.cap / 2)
		index = (int)gridDim.x - 1 - (index - cut.cap / 2);
	if (!find_unit<WIN>(s, a, c.kvh, group, cut, index, u))
		return;
	const int tid = threadIdx.x, lane = tid & 63, n16 = lane & 15, g = lane >> 4;
	const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	bool bad = !seq_fits(s, u.len, u.n);

	const int last = a.mask ? u.n : min(u.n, (u.tile * R + R - 1) / group + 1);
	int pages = bad ? 0 : (u.len + last + PAGE - 1) / PAGE, shared = (u.len + u.n + PAGE - 1) / PAGE;
	const int all_below = u.len + (a.mask ? 0 : u.tile * R / group + 1); // rows below it every query of the tile sees
	Span span = {0, 0, 0};
	int all_above = 0; // (a window: and from it on)
	if (WIN) {
		int least;
		const int n0 = u.tile * R / group, n1 = min(u.n, (u.tile * R + R - 1) / group + 1) - 1;
		tile_lows(a, u, n0, n1, least, all_above);
		span = window_span(a.mask ? min(least, u.len) : least, a.sinks, pages);
		shared = pages = span.pages;
	}
	int p0, p1;
	part_pages(cut, u, shared, pages, p0, p1);
	PageIds ids;
	ids.get(s, u, span, p0);
	u4 codes[I8 ? NL : 1];
	float sr = 0.0f;
	auto page = [&](int p) {
		return (size_t)ids.of(s, u, span, c.n_pages, p, bad) * c.kvh + u.head;
	};
	// where a K row's and a V column's pieces lie
	auto kx = [](int row) { return ((row & 3) | (row >> 3 & 3) << 2) & (KP - 1); };
	auto vx = [](int col) { return col & (VP - 1); };
	// f16: a page's pieces straight to LDS (a thread's piece e there comes from
	// the place that the swizzle names)
	uint32_t ko[NL], vo[NL];
	if (!I8)
#pragma unroll
		for (int q = 0; q < NL; q++) {
			const int e = tid + q * 256;
			ko[q] = 16 * (e / KP * KP + (e % KP ^ kx(e / KP)));
			vo[q] = 16 * (e / VP * VP + (e % VP ^ vx(e / VP)));
		}
	// f16: request a page, to buffer b
	auto get = [&](size_t pg, int b) {
		const uint8_t *k = uniform(c.k + pg * PAGE * HD * E), *v = uniform(c.v + pg * PAGE * HD * E);
#pragma unroll
		for (int q = 0; q < NL; q++) {
			load_lds16(k, ko[q], lk[b] + (q * 256 + wave * 64) * 8);
			load_lds16(v, vo[q], lv[b] + (q * 256 + wave * 64) * 8);
		}
	};
	// int8: a page's codes by way of registers, K and the scales (half 0) and then
	// V (both at once would be more registers than there are)
	auto get8 = [&](size_t pg, int half) {
		const uint8_t *from = uniform((half ? c.v : c.k) + pg * PAGE * HD);
#pragma unroll
		for (int q = 0; q < NL; q++)
			codes[q] = reinterpret_cast<const u4 *>(from)[tid + q * 256];
		if (!half && tid < 2 * PAGE)
			sr = tid < PAGE ? c.ks[pg * PAGE + tid] : c.vs[pg * PAGE + tid - PAGE];
	};
	auto put8 = [&](int b, int half) {
		if (!half) {
#pragma unroll
			for (int q = 0; q < NL; q++) {
				const int e = tid + q * 256; // piece of 16 codes: two of f16
				const int row = e / (KP / 2), kp = e % (KP / 2) * 2;
				h8 *kl = reinterpret_cast<h8 *>(lk[b] + row * HD);
				kl[kp ^ kx(row)] = codes8(codes[q].x, codes[q].y);
				kl[(kp + 1) ^ kx(row)] = codes8(codes[q].z, codes[q].w);
			}
			if (tid < 2 * PAGE)
				lsc[b][tid >> 6][tid & 63] = sr;
		} else {
#pragma unroll
			for (int q = 0; q < NL; q++) {
				const int e = tid + q * 256;
				const int col = e / (VP / 2), vp = e % (VP / 2) * 2;
				h8 *vl = reinterpret_cast<h8 *>(lv[b] + col * PAGE);
				vl[vp ^ vx(col)] = codes8(codes[q].x, codes[q].y);
				vl[(vp + 1) ^ vx(col)] = codes8(codes[q].z, codes[q].w);
			}
		}
	};
	size_t at = 0;
	u4 first[I8 ? NL : 1]; // of K: all that a unit begins with is under way at once
	if (p0 < p1) {
		at = page(p0);
		if (I8) {
			get8(at, 0);
#pragma unroll
			for (int q = 0; q < NL; q++)
				first[q] = codes[q];
			get8(at, 1);
		} else {
			get(at, 0);
		}
	}

	int node[NT];
	h8 qh[NT][KS], ql[NT][KS];
	float qs[NT], x[NT][KS][8];
	Rows<HD> r[NT];
#pragma unroll
	for (int t = 0; t < NT; t++) {
		const int row = u.tile * R + wave % RG * 32 + 16 * t + n16;
		node[t] = row / group < u.n ? row / group : -1;
		fetch_query<HD, false>(a, u, node[t], u.head * group + row % group, g, x[t]);
	}
#pragma unroll
	for (int t = 0; t < NT; t++) {
		split_query<HD>(a, node[t], x[t], qh[t], ql[t], qs[t]);
#pragma unroll
		for (int m = 0; m < MT; m++)
			r[t].o[m] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
	}
	float up = V_UP;
	if (I8) {
		put8(0, 1);
#pragma unroll
		for (int q = 0; q < NL; q++)
			codes[q] = first[q];
		put8(0, 0);
	} else {
		__builtin_amdgcn_s_waitcnt(0); // the pieces under way to LDS
	}
	__syncthreads();

	for (int p = p0; p < p1; p++) {
		const int b = (p - p0) & 1, start = (WIN ? span.page(p) : p) * PAGE, end = u.len + u.n - start;
		const bool more = p + 1 < p1;
		const size_t next = more ? page(p + 1) : at;
		if (!I8 && more)
			get(next, b ^ 1); // (all waves left that buffer at the last barrier)
		const bool seen_all = start + PAGE <= all_below && (!WIN || start >= all_above || start + PAGE <= a.sinks);
		uint64_t vis[NT];
#pragma unroll
		for (int t = 0; t < NT; t++)
			vis[t] = ~0ull;
		if (!seen_all)
#pragma unroll
			for (int t = 0; t < NT; t++)
				vis[t] = sees_through<WIN>(a, u, node[t], WIN && node[t] >= 0 ? low_of(a, u, node[t]) : 0, start);
		// a page that not all of the tile sees: f16 values that are not finite
		// are taken out first (see guard_values), and come back below
		if (!I8 && !seen_all) {
			uint32_t odd = 0;
#pragma unroll
			for (int q = 0; q < NL; q++) {
				u4 *x = reinterpret_cast<u4 *>(lv[b]) + tid + q * 256;
				u4 y = *x;
				uint32_t here = 0;
#pragma unroll
				for (int e = 0; e < 4; e++) {
					here |= ((y[e] & 0x7c00u) == 0x7c00u) | ((y[e] & 0x7c000000u) == 0x7c000000u);
					y[e] = ((y[e] & 0x7c00u) == 0x7c00u ? 0u : y[e] & 0xffffu) |
					       ((y[e] & 0x7c000000u) == 0x7c000000u ? 0u : y[e] & 0xffff0000u);
				}
				if (here)
					*x = y;
				odd |= here;
			}
			if (__syncthreads_or(odd)) {
				uint64_t mine[NT];
#pragma unroll
				for (int t = 0; t < NT; t++)
					mine[t] = RG == MANY_WAVES ? vis[t] : vis[t] & 0xffffffffull << wave / RG * 32;
				give_back<HD, NT>(c.v + at * HD * PAGE * 2, g, end, mine, r);
			}
		}
		// (between: what is done between the products and the weights)
		auto weigh_half = [&](int row0, h8 (&ph)[NT][1], h8 (&pl)[NT][1], auto between) {
			uint32_t seen[NT];
			bool whole = seen_all;
#pragma unroll
			for (int t = 0; t < NT; t++)
				seen[t] = (uint32_t)(vis[t] >> row0);
			if (!seen_all) {
				bool all = true, any = false;
#pragma unroll
				for (int t = 0; t < NT; t++) {
					all = all && (seen[t] == ~0u || node[t] < 0);
					any = any || seen[t] != 0;
				}
				if (!__any(any)) {
					between();
					return false;
				}
				whole = __all(all);
			}
			h8 kf[KT][KS];
#pragma unroll
			for (int kt = 0; kt < KT; kt++) {
				const h8 *kl = reinterpret_cast<const h8 *>(lk[b] + (row0 + (n16 >> 2) * 8 + kt * 4 + (n16 & 3)) * HD);
#pragma unroll
				for (int k = 0; k < KS; k++)
					kf[kt][k] = kl[(k * 4 + g) ^ (n16 & (KP - 1))];
			}
			f4 sc[NT][KT];
			// (the wave that feeds the matrix cores goes before the other: 2%)
			__builtin_amdgcn_s_setprio(1);
#pragma unroll
			for (int kt = 0; kt < KT; kt++)
#pragma unroll
				for (int t = 0; t < NT; t++)
					sc[t][kt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
			for (int k = 0; k < KS; k++)
#pragma unroll
				for (int e = 0; e < 2; e++)
#pragma unroll
					for (int kt = 0; kt < KT; kt++)
#pragma unroll
						for (int t = 0; t < NT; t++)
							sc[t][kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[kt][k], e ? qh[t][k] : ql[t][k],
													   sc[t][kt], 0, 0, 0);
			__builtin_amdgcn_s_setprio(0);
			between();
			float ks = 0.0f, vs = 0.0f;
			if constexpr (I8) {
				const int row = row0 + g * 8 + (n16 & 7);
				ks = lsc[b][0][row];
				vs = lsc[b][1][row];
				if (!whole)
					guard_scales(ks, vs, row < end);
				vs = scale_up<HD, NT>(vs, up, r);
			}
#pragma unroll
			for (int t = 0; t < NT; t++)
				if (I8)
					weigh8<HD, KT>(r[t], sc[t], ks, vs, qs[t], whole, seen[t] >> (8 * g), ph[t], pl[t]);
				else
					weigh<HD, KT>(r[t], sc[t], qs[t], whole, seen[t] >> (8 * g), ph[t], pl[t]);
			return true;
		};
		auto add_half = [&](int row0, const h8 (&ph)[NT][1], const h8 (&pl)[NT][1]) {
			__builtin_amdgcn_s_setprio(1);
#pragma unroll
			for (int m = 0; m < MT; m++) {
				const h8 vf = reinterpret_cast<const h8 *>(lv[b] + (m * 16 + n16) * PAGE)[(row0 / 8 + g) ^ (n16 & (VP - 1))];
#pragma unroll
				for (int t = 0; t < NT; t++)
					r[t].o[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[t][0], r[t].o[m], 0, 0, 0);
#pragma unroll
				for (int t = 0; t < NT; t++)
					r[t].o[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[t][0], r[t].o[m], 0, 0, 0);
			}
			__builtin_amdgcn_s_setprio(0);
		};
		h8 ph[NT][1], pl[NT][1];
		if constexpr (RG == MANY_WAVES) {
#pragma unroll 1
			for (int row0 = 0; row0 < PAGE; row0 += 32) {
				if (I8 && more)
					get8(next, row0 >> 5);
				if (weigh_half(row0, ph, pl, [] {}))
					add_half(row0, ph, pl);
				if (I8 && more)
					put8(b ^ 1, row0 >> 5);
			}
		} else {
			const int row0 = wave / RG * 32;
			if (I8 && more)
				get8(next, 0);
			const bool any = weigh_half(row0, ph, pl, [&] {
				if (I8 && more) {
					put8(b ^ 1, 0);
					get8(next, 1);
				}
			});
			if (any)
				add_half(row0, ph, pl);
			if (I8 && more)
				put8(b ^ 1, 1);
		}
		if (!I8)
			__builtin_amdgcn_s_waitcnt(0);
		__syncthreads();
		at = next;
	}
	float back, total[NT];
#pragma unroll
	for (int t = 0; t < NT; t++)
		total[t] = finish<HD, I8>(r[t], up, back);
	if constexpr (RG < MANY_WAVES) {
		// the waves of the pages' second halves hand their rows to the others:
		// O ([wave][t][m][lane], in K's buffers) and the maxima and sums
		static_assert(RG == MANY_WAVES / 2, "a row group: two waves");
		f4 *lo = reinterpret_cast<f4 *>(&lk[0][0]) + (size_t)wave % RG * NT * MT * 64 + lane;
		float *lm = &lsc[0][0][0] + wave % RG * 64 + n16;
		if (wave >= RG)
#pragma unroll
			for (int t = 0; t < NT; t++) {
#pragma unroll
				for (int m = 0; m < MT; m++)
					lo[(t * MT + m) * 64] = r[t].o[m] * back;
				if (g == 0) {
					lm[t * 32] = r[t].mx;
					lm[t * 32 + 16] = total[t];
				}
			}
		__syncthreads();
		if (wave >= RG)
			return;
#pragma unroll
		for (int t = 0; t < NT; t++) {
			const float om = lm[t * 32], top = __builtin_fmaxf(r[t].mx, om), base = top == -__builtin_inff() ? 0.0f : top;
			const float f0 = __builtin_amdgcn_exp2f(r[t].mx - base), f1 = __builtin_amdgcn_exp2f(om - base);
			r[t].mx = top;
			total[t] = total[t] * f0 + lm[t * 32 + 16] * f1;
#pragma unroll
			for (int m = 0; m < MT; m++)
				r[t].o[m] = r[t].o[m] * (back * f0) + lo[(t * MT + m) * 64] * f1;
		}
		back = 1.0f;
	}
#pragma unroll
	for (int t = 0; t < NT; t++) {
		const int q = wave * 32 + 16 * t + n16, to = u.tile * R + q;
		if (node[t] < 0)
			continue;
		float *o = part + ((size_t)index * R + q) * part_row(HD);
		float f = back;
		if (u.parts == 1) {
			o = a.out + (size_t)(u.t0 + to / group) * a.o_stride + (size_t)(u.head * group + to % group) * HD;
			f = bad ? __builtin_nanf("") : total[t] == 0.0f ? 0.0f : back / total[t];
		} else if (g == 0) {
			o[HD] = bad ? __builtin_nanf("") : r[t].mx;
			o[HD + 1] = bad ? __builtin_nanf("") : total[t];
		}
		const bool vec = ((uintptr_t)o & 15) == 0;
#pragma unroll
		for (int m = 0; m < MT; m++) {
			const f4 x = total[t] == 0.0f && u.parts == 1 && !bad ? (f4){0.0f, 0.0f, 0.0f, 0.0f} : r[t].o[m] * f;
			if (vec) {
				// (past the caches: what lies there at a launch's end is written back first,
				// 3 us of a tree's parts)
				__builtin_nontemporal_store(x, reinterpret_cast<f4 *>(o + m * 16 + 4 * g));
			} else {
#pragma unroll
				for (int i = 0; i < 4; i++)
					o[m * 16 + 4 * g + i] = x[i];
			}
		}
	}
}

// ---------------------------------------------------------------- join
// A workgroup: JOIN_HEADS query heads of one token, HD / 4 lanes to a head: first
// the parts' maxima and sums, a lane to a part, then their rows, 16 under way
// at once.  Bound by the parts' bytes and the chain of steps: 26 tokens of 64 heads
// in 18 parts (16 MB) 8.9 us, of which 2 find the parts.
constexpr int JOIN_HEADS = 8;
template <int HD, bool WIN>
__global__ __launch_bounds__(JOIN_HEADS *HD / 4) void attn_join_kernel(KvLayer c, KvSeqs s, AttnArgs a, Cut cut, int units,
								       const float *part)
{
	constexpr int L = HD / 4, PR = part_row(HD);
	const int group = a.n_heads / c.kvh, blocks = div_up(a.n_heads, JOIN_HEADS);
	const int t = blockIdx.x / blocks, h = blockIdx.x % blocks * JOIN_HEADS + threadIdx.x / L, head = min(h, a.n_heads - 1) / group;
	int st0, sn;
	const int b = seq_of_token(s, t, st0, sn);
	if (b < 0)
		return;
	// the sequence's units: those of the sequences before it come first
	const int lane = threadIdx.x & 63;
	int t0, n, len, tiles, pages;
	seq_work<WIN>(s, a, lane, group, cut.rows, t0, n, len, tiles, pages);
	const float rate = part_rate<WIN>(s, a, c.kvh, group, cut, tiles, pages);
	int before = 0;
	for (int b0 = 0; b0 <= b; b0 += 64) {
		if (b0)
			seq_work<WIN>(s, a, b0 + lane, group, cut.rows, t0, n, len, tiles, pages);
		before += s.n_seqs > 1 ? wave_sum(b0 + lane < b && tiles ? tiles * tile_parts(cut, pages, rate) * c.kvh : 0) : 0;
	}
	seq_work<WIN>(s, a, b, group, cut.rows, t0, n, len, tiles, pages);
	const int parts = tile_parts(cut, pages, rate);
	if (parts == 1)
		return;
	const int row = (t - t0) * group + h % group, tile = row / cut.rows;
	const int u0 = before + ((tiles - 1 - tile) * parts) * c.kvh + head; // unit of part q: u0 + q kvh
	if (h >= a.n_heads || u0 < 0 || (long long)u0 + (long long)(parts - 1) * c.kvh >= units)
		return; // (sequences that overlap: more units than the rows can have)
	const float *from = part + ((size_t)u0 * cut.rows + row % cut.rows) * PR;
	const size_t step = (size_t)c.kvh * cut.rows * PR;
	const int i = threadIdx.x % L;
	float m = -__builtin_inff(), l = 0.0f;
	f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
	for (int q0 = 0; q0 < parts; q0 += L) {
		float pm = -__builtin_inff(), pl = 0.0f;
		if (q0 + i < parts) {
			const float *pr = from + (q0 + i) * step;
			pm = pr[HD];
			pl = pr[HD + 1];
		}
		float top = __builtin_fmaxf(m, pm);
#pragma unroll
		for (int k = 1; k < L; k <<= 1)
			top = __builtin_fmaxf(top, __shfl_xor(top, k, L));
		const float base = top == -__builtin_inff() ? 0.0f : top;
		const float back = __builtin_amdgcn_exp2f(m - base);
		const float f = __builtin_amdgcn_exp2f(pm - base);
		m = top;
		float sum = pl * f;
#pragma unroll
		for (int k = 1; k < L; k <<= 1)
			sum += __shfl_xor(sum, k, L);
		l = l * back + sum;
		x *= back;
		const int n8 = min(L, parts - q0);
		for (int q = 0; q < n8; q += 16) {
			f4 o[16];
#pragma unroll
			for (int k = 0; k < 16; k++)
				o[k] = reinterpret_cast<const f4 *>(from + (q0 + min(q + k, n8 - 1)) * step)[i];
#pragma unroll
			for (int k = 0; k < 16; k++) {
				const float fk = __shfl(f, min(q + k, n8 - 1), L);
				x += q + k < n8 ? o[k] * fk : (f4){0.0f, 0.0f, 0.0f, 0.0f};
			}
		}
	}
	float *out = a.out + (size_t)t * a.o_stride + (size_t)h * HD + 4 * i;
#pragma unroll
	for (int q = 0; q < 4; q++)
		out[q] = l == 0.0f ? 0.0f : x[q] / l;
}

// ---------------------------------------------------------------- launch
// a tile for every CU, and none is cut (600 tokens over 1100 rows, 300 tiles, 54 us; cut in two 68)
constexpr int MANY_FULL = 256, MANY_CAP = 512;

struct Shape {
	bool few;
	Cut cut;
	size_t units; // at most
};

// Whether `rows` query rows (of one kv head) of n_seqs sequences go to the kernel of few rows.
static bool few_of(const KvLayer &c, int max_pages, size_t rows, size_t n_seqs)
{
	// The kernel of few rows reads a page again for each 16 of them, but its parts
	// are joined in the same launch and a wave waits for none: small trees take it
	// too, int8 ones (half the bytes; codes are converted for every 16 rows) up to
	// larger sizes.  int8: 5 tokens of 32 heads over 8000 rows 17 us (by the other
	// kernel 26), 26 over 8000 26.5 (31), over 32000 61 (59), 16 sequences of 16
	// over 8000 70 (64).  f16: 8 tokens over 1000 rows 16.7 (18.6), over 8000 20 (27),
	// 16 over 8000 26 (31), 8 sequences of 8 over 8000 38 (31); with 8 kv heads of 64
	// 26 over 2000 13 (16), over 8000 23.5 (23), but over 30000, which a die's cache
	// does not hold, 60 (34): more than 64 f16 rows only where the page table, all
	// that is known here of the lengths, ends at 10000.
	const size_t most = c.i8 ? 256 : max_pages * PAGE <= 10240 ? 128 : 64, units = c.i8 ? 448 : 64;
	return rows <= FEW_ROWS * n_seqs || (rows <= most * n_seqs && rows * c.kvh <= units * FEW_ROWS);
}

static Shape attn_shape(const KvLayer &c, const KvSeqs &s, const AttnArgs &a)
{
	const size_t group = a.n_heads / c.kvh, rows = (size_t)s.n_tokens * group;
	Shape h;
	// (what is known here of the pages that a tile sees: the table's columns, or the
	// window's)
	size_t columns = s.max_pages;
	if (a.window) {
		const size_t seen = ((size_t)a.sinks + PAGE - 1) / PAGE + ((size_t)a.window + PAGE - 2) / PAGE + 1;
		columns = seen < columns ? seen : columns;
	}
	h.few = few_of(c, (int)columns, rows, s.n_seqs);
	// Through a window a tile has few pages, so that reading them again for each 16 rows
	// costs less than the other kernel's second launch, as long as no CU has two tiles (100
	// f16 tokens over a window of 200 15 us, by the other kernel 23; 48 tokens of 64 heads over
	// 1000 24.5 and 28; 200 int8 tokens over 200 58 and 27).  f16: up to 640 KB of them (26 tokens
	// of four sequences, 8 kv heads of 64, over 2000 22.5 and 26, over 4000 36 and 31); int8,
	// whose codes the other kernel converts first: to 1280 (32 tokens of four sequences over 4000
	// 37.5 both, 26 of one 30 and 36).
	if (a.window && rows * c.kvh <= (size_t)FEW_CAP * FEW_ROWS && columns * PAGE * c.hd * 2 <= (c.i8 ? 1280u : 320u) * 1024)
		h.few = true;
	// many: 128 rows where such tiles fill the card (4096 tokens of 32 heads 240
	// us, by 64 rows 257), or 64: as many units and half the parts' bytes, less
	// left of tiles that a mask or a sequence's end cuts (1000 tokens over 2000
	// rows 55 us, by 128 rows 89)
	h.cut.rows = h.few ? FEW_ROWS : rows * c.kvh < (size_t)MANY_FULL * 128 ? 64 : 128;
	// one workgroup of 8 waves on a CU, or two of 4
	h.cut.cap = h.few ? FEW_CAP : MANY_CAP;
	h.cut.full = h.few ? FEW_CAP : MANY_FULL;
	// (few: a grain is a round of the waves; a second one costs as much as joining
	// two parts: one f16 token over 300 rows of 8 kv heads of 64 7.8 us, in two parts
	// 10.2, over 1000 10.7, in two parts of two rounds 11.6; one int8 token over 600
	// rows of 4 kv heads of 128 12.5, in two parts 14.4, over 1000 14.7 either way, of
	// 8 kv heads of 64 8.6, in two parts 10.7, over 1000 9.9 and 10.8)
	h.cut.grain = !h.few ? 1 : c.i8 ? FEW_WAVES : FEW_WAVES / 2;
	h.cut.least = h.few ? 1 : 2;
	h.cut.alone = h.few ? 2 : 3;
	const size_t seqs = s.n_seqs < s.n_tokens ? s.n_seqs : s.n_tokens; // that have tokens, at most
	const size_t tiles = (rows + seqs * (h.cut.rows - 1)) / h.cut.rows;
	// as many tiles as fill the card are not cut: no parts, no join
	h.cut.whole = rows / h.cut.rows * c.kvh >= (size_t)h.cut.full;
	// Nor are tiles that a window leaves few pages: a cut saves the pages of all but one part,
	// at 2 us each (int8 more), and the join costs 10 us.  f16: 200 tokens of 32 heads over 200 21.7
	// us (cut 28.0), over 500 27.8 (28.3), 175 of 64 in eight sequences over 700 34.5 (42.8);
	// int8: 70 of 64 in four over 300 27.2 (27.4), over 500 32.5 (29.5).
	const size_t all = tiles * c.kvh;
	if (a.window && !h.few && all < MANY_CAP && columns * (MANY_CAP - all) <= (size_t)(c.i8 ? 6 : 10) * MANY_CAP)
		h.cut.whole = 1;
	// (a share that is rounded down can make one more part)
	h.units = (h.cut.whole ? 0 : h.cut.cap + c.kvh) + tiles * c.kvh;
	// (not with a kv head for every 8 rows or more, and then: whole tiles)
	if (h.few && h.units > WORK_COUNTERS)
		h.cut.whole = 1;
	return h;
}

// Enough for this call and for every one of the same heads and type with no more
// tokens, sequences and columns of the page table.  (Calls whose tiles fill the
// card have no parts, smaller ones do: memory for a prompt's chunk is memory for
// the tokens decoded behind it.)
size_t attention_work_bytes(const KvLayer &c, const KvSeqs &s, const AttnArgs &a)
{
	const size_t group = a.n_heads / c.kvh, rows = (size_t)s.n_tokens * group;
	const size_t seqs = s.n_seqs < s.n_tokens ? s.n_seqs : s.n_tokens;
	// rows of the largest such call whose tiles are cut, 0: there is none
	auto most_rows = [&](size_t tile, size_t full) {
		const size_t below = tile * ((full + c.kvh - 1) / c.kvh) - 1;
		return (rows < below ? rows : below) / group * group;
	};
	auto values = [&](size_t r, size_t n, size_t tile, size_t cap) {
		n = n < r / group ? n : r / group;
		return r == 0 ? 0 : (cap + c.kvh + (r + n * (tile - 1)) / tile * c.kvh) * tile * part_row(c.hd);
	};
	size_t most = values(most_rows(FEW_ROWS, FEW_CAP), seqs, FEW_ROWS, FEW_CAP);
	for (size_t tile = 64; tile <= 128; tile *= 2) {
		const size_t r = most_rows(tile, MANY_FULL);
		// (one sequence's rows are the first that this kernel takes, and it takes
		// more than FEW_ROWS for each sequence; with a window it takes them for the
		// window's sake, which another call may have otherwise)
		if ((!a.window && few_of(c, s.max_pages, r, 1)) || (tile == 128 && r * c.kvh < (size_t)MANY_FULL * 128))
			continue;
		const size_t by_rows = (r - 1) / FEW_ROWS, v = values(r, seqs < by_rows ? seqs : by_rows, tile, MANY_CAP);
		most = most > v ? most : v;
	}
	return WORK_COUNTERS * sizeof(int) + most * sizeof(float);
}

template <int HD, bool I8, bool WIN>
static hipError_t go(const Shape &h, const KvLayer &c, const KvSeqs &s, const AttnArgs &a, int *count, hipStream_t st)
{
	float *part = reinterpret_cast<float *>(count + WORK_COUNTERS);
	if (h.few) {
		const size_t lds = (size_t)FEW_WAVES * FEW_ROWS * part_row(HD) * sizeof(float);
		const hipError_t e = ensure_lds_limit((const void *)attn_few_kernel<HD, I8, WIN>, lds);
		if (e != hipSuccess)
			return e;
		tie_launch(attn_few_kernel<HD, I8, WIN>, dim3(h.units), dim3(64 * FEW_WAVES), lds, st, c, s, a, h.cut,
			   part, count);
		return hipGetLastError();
	}
	tie_launch(h.cut.rows == 64 ? attn_many_kernel<HD, I8, 2, WIN> : attn_many_kernel<HD, I8, 4, WIN>, dim3(h.units),
		   dim3(64 * MANY_WAVES), 0, st, c, s, a, h.cut, part);
	if (!h.cut.whole)
		tie_launch(attn_join_kernel<HD, WIN>, dim3((size_t)s.n_tokens * ((a.n_heads + JOIN_HEADS - 1) / JOIN_HEADS)),
			   dim3(JOIN_HEADS * HD / 4), 0, st, c, s, a, h.cut, (int)h.units, (const float *)part);
	return hipGetLastError();
}

hipError_t launch_attention(const KvLayer &c, const KvSeqs &s, const AttnArgs &a, void *work, hipStream_t st)
{
	const Shape h = attn_shape(c, s, a);
	int *count = reinterpret_cast<int *>(work);
	auto by_window = [&](auto win) {
		constexpr bool W = decltype(win)::value;
		if (c.hd == 128)
			return c.i8 ? go<128, true, W>(h, c, s, a, count, st) : go<128, false, W>(h, c, s, a, count, st);
		return c.i8 ? go<64, true, W>(h, c, s, a, count, st) : go<64, false, W>(h, c, s, a, count, st);
	};
	return a.window ? by_window(std::true_type()) : by_window(std::false_type());
}

} // namespace tie
