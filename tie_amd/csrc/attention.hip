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
// v_mfma_f32_16x16x32_f16.  A lane (n = lane % 16, g = lane / 16) of S^T's
// four 16-row tiles holds query n and, since tile t's row 4 g + i is page row
// 16 g + 4 t + i, the 16 rows 16 g .. 16 g + 15 of a page: just what the second
// product's operand wants of that lane.  So the weights never leave their
// registers, the running maximum and sum of a query are one value a lane
// (joined over g), and K and V^T go from the pages straight into operands.
#include "kv.h"

namespace tie {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float P_SCALE = 4096.0f; // weights are at most 1; their second f16 part stays above the subnormals
constexpr int ATTN_UNITS = 512;    // workgroups that the work is cut for

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
	lo = __builtin_convertvector((f2){x0 - (float)hi.x, x1 - (float)hi.y}, h2);
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

// How the work of a call is cut: sequence b has tiles(b) row tiles for each kv
// head, each over pages(b) pages, in chunks of `chunk` pages -- one unit of
// work (a workgroup) for each.  Every workgroup finds the cut by itself from
// the lengths on the device.
struct Unit {
	int b, tile, head, part, parts, chunk, t0, n, len, index;
};

__device__ __forceinline__ long long wave_sum(long long x)
{
#pragma unroll
	for (int m = 1; m < 64; m <<= 1)
		x += __shfl_xor(x, m);
	return x;
}

__device__ __forceinline__ void seq_work(const KvSeqs &s, int b, int group, int rows, int &tiles, int &pages)
{
	int t0, n;
	tiles = pages = 0;
	if (b >= s.n_seqs)
		return;
	seq_tokens(s, b, t0, n);
	if (n == 0)
		return;
	const int len = s.len[b];
	tiles = (int)(((long long)n * group + rows - 1) / rows);
	pages = seq_fits(s, len, n) ? (len + n + PAGE - 1) / PAGE : 1;
}

// pages of a unit: as many as leave about ATTN_UNITS of them
__device__ __forceinline__ int unit_chunk(const KvSeqs &s, int kvh, int group, int rows, int least)
{
	const int lane = threadIdx.x & 63;
	long long w = 0;
	for (int b = lane; b < s.n_seqs; b += 64) {
		int tiles, pages;
		seq_work(s, b, group, rows, tiles, pages);
		w += (long long)tiles * pages;
	}
	w = wave_sum(w) * kvh;
	const long long c = (w + ATTN_UNITS - 1) / ATTN_UNITS;
	return (int)(c < least ? least : c);
}

// the unit of workgroup `index`; false past the last
__device__ __forceinline__ bool find_unit(const KvSeqs &s, int kvh, int group, int rows, int least, int index, Unit &u)
{
	const int lane = threadIdx.x & 63;
	u.chunk = unit_chunk(s, kvh, group, rows, least);
	u.index = index;
	long long before = 0;
	for (int b0 = 0; b0 < s.n_seqs; b0 += 64) {
		int tiles, pages;
		seq_work(s, b0 + lane, group, rows, tiles, pages);
		const int parts = (pages + u.chunk - 1) / u.chunk;
		const long long mine = (long long)tiles * parts * kvh;
		long long incl = mine;
#pragma unroll
		for (int m = 1; m < 64; m <<= 1) {
			const long long o = __shfl_up(incl, m);
			if (lane >= m)
				incl += o;
		}
		const unsigned long long past = __ballot(before + incl > index);
		if (past) {
			const int l = __builtin_ctzll(past);
			const int at = (int)(index - (before + __shfl(incl - mine, l)));
			u.b = b0 + l;
			u.parts = __shfl(parts, l);
			// (a kv head's parts of a tile lie side by side)
			u.part = at % u.parts;
			u.head = at / u.parts % kvh;
			u.tile = at / u.parts / kvh;
			seq_tokens(s, u.b, u.t0, u.n);
			u.len = s.len[u.b];
			return true;
		}
		before += __shfl(incl, 63);
	}
	return false;
}

// Which of the 64 rows of the page at row `start` a token sees: all committed
// ones, and of the sequence's own tokens those of its mask, or (causal) those
// up to itself.  node < 0: none.
__device__ __forceinline__ uint64_t sees(const AttnArgs &a, const Unit &u, int node, int start)
{
	if (node < 0)
		return 0;
	const int rel = start - u.len; // the page's first row as a node
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

// Partial results of a unit: its rows' maximum and sum, then O.
constexpr int part_floats(int rows, int hd)
{
	return rows * (hd + 2);
}

// A workgroup: NT tiles of 16 query rows (a row: a token and one query head
// of the unit's kv head), its WK waves taking the unit's pages in turn.
template <int HD, bool I8, int NT, int WK>
__global__ __launch_bounds__(64 * WK) void attn_kernel(KvLayer c, KvSeqs s, AttnArgs a, int least, float *part)
{
	constexpr int KS = HD / 32, MT = HD / 16, R = 16 * NT;
	extern __shared__ __attribute__((aligned(16))) float lds[];
	const int group = a.n_heads / c.kvh;
	Unit u;
	if (!find_unit(s, c.kvh, group, R, least, blockIdx.x, u))
		return;
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n16 = lane & 15, g = lane >> 4;
	bool bad = !seq_fits(s, u.len, u.n); // the rows cannot be read: the result is NaN

	// the queries, scaled to below 2^10 and split
	h8 qh[NT][KS], ql[NT][KS];
	float qs[NT]; // what a score is multiplied by: exp2 instead of exp
	int node[NT];
#pragma unroll
	for (int t = 0; t < NT; t++) {
		const int r = u.tile * R + 16 * t + n16;
		node[t] = r / group < u.n ? r / group : -1;
		float x[KS][8], m = 0.0f;
		const float *q = a.q + (size_t)(u.t0 + (node[t] < 0 ? 0 : node[t])) * a.q_stride +
				 (size_t)(u.head * group + r % group) * HD;
#pragma unroll
		for (int k = 0; k < KS; k++)
#pragma unroll
			for (int j = 0; j < 8; j++) {
				// int8 rows come 16 codes to a lane and load, f16 rows 8
				const int at = I8 ? (k >> 1) * 64 + g * 16 + (k & 1) * 8 + j : k * 32 + g * 8 + j;
				x[k][j] = node[t] < 0 ? 0.0f : q[at];
				m = __builtin_fmaxf(m, __builtin_fabsf(x[k][j]));
			}
		m = max_g(m);
		const float p2 = m >= 1e-30f && m < 1e30f ? pow2_below(m) : 1.0f;
		const float up = 512.0f / p2;
		qs[t] = a.scale * 1.44269504088896f * (p2 * (1.0f / 512.0f));
#pragma unroll
		for (int k = 0; k < KS; k++)
#pragma unroll
			for (int j = 0; j < 8; j += 2) {
				h2 hi, lo;
				split2(x[k][j] * up, x[k][j + 1] * up, hi, lo);
				qh[t][k][j] = hi.x, qh[t][k][j + 1] = hi.y;
				ql[t][k][j] = lo.x, ql[t][k][j + 1] = lo.y;
			}
	}

	f4 o[NT][MT];
	float mx[NT], sum[NT];
#pragma unroll
	for (int t = 0; t < NT; t++) {
		mx[t] = -__builtin_inff();
		sum[t] = 0.0f;
#pragma unroll
		for (int m = 0; m < MT; m++)
			o[t][m] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
	}
	// int8: the weights carry their row's V scale, over the largest power of
	// two among the scales so far
	float vtop = 1e-30f;

	// (causal: nothing behind the tile's last token is seen)
	const int last = a.mask ? u.n : min(u.n, (u.tile * R + R - 1) / group + 1);
	const int pages = bad ? 0 : (u.len + last + PAGE - 1) / PAGE;
	const int p1 = min(pages, (u.part + 1) * u.chunk);
	for (int p = u.part * u.chunk + wave; p < p1; p += WK) {
		const int start = p * PAGE, id = page_of(s, c.n_pages, u.b, start);
		if (id < 0) {
			bad = true;
			continue;
		}
		const size_t at = (size_t)id * c.kvh + u.head;
		uint64_t vis[NT];
		bool whole = true;
#pragma unroll
		for (int t = 0; t < NT; t++) {
			vis[t] = sees(a, u, node[t], start);
			whole = whole && (vis[t] == ~0ull || node[t] < 0);
		}
		whole = __all(whole);
		const int end = u.len + u.n - start; // rows of the page that hold anything

		// S^T
		f4 sc[NT][4];
#pragma unroll
		for (int kt = 0; kt < 4; kt++) {
			const int row = (n16 >> 2) * 16 + kt * 4 + (n16 & 3);
			h8 kf[KS];
			if constexpr (I8) {
				const u4 *kr = reinterpret_cast<const u4 *>(c.k + (at * PAGE + row) * HD) + g;
#pragma unroll
				for (int q = 0; q < KS / 2; q++) {
					const u4 w = kr[q * 4];
					kf[2 * q] = codes8(w.x, w.y);
					kf[2 * q + 1] = codes8(w.z, w.w);
				}
			} else {
				const u4 *kr = reinterpret_cast<const u4 *>(c.k + (at * PAGE + row) * HD * 2) + g;
#pragma unroll
				for (int q = 0; q < KS; q++)
					kf[q] = __builtin_bit_cast(h8, kr[q * 4]);
			}
#pragma unroll
			for (int t = 0; t < NT; t++) {
				f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
				for (int k = 0; k < KS; k++)
					acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[k], ql[t][k], acc, 0, 0, 0);
#pragma unroll
				for (int k = 0; k < KS; k++)
					acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[k], qh[t][k], acc, 0, 0, 0);
				sc[t][kt] = acc;
			}
		}

		// the scales of this lane's 16 rows
		f4 vsc[4];
		float vinv = P_SCALE;
		if constexpr (I8) {
			const f4 *ks = reinterpret_cast<const f4 *>(c.ks + at * PAGE + g * 16);
			const f4 *vs = reinterpret_cast<const f4 *>(c.vs + at * PAGE + g * 16);
			float top = 0.0f;
#pragma unroll
			for (int kt = 0; kt < 4; kt++) {
				const f4 k4 = ks[kt];
				vsc[kt] = vs[kt];
#pragma unroll
				for (int i = 0; i < 4; i++) {
					const bool there = g * 16 + kt * 4 + i < end;
					top = __builtin_fmaxf(top, there ? vsc[kt][i] : 0.0f);
#pragma unroll
					for (int t = 0; t < NT; t++)
						sc[t][kt][i] *= k4[i];
				}
			}
			top = max_g(top);
			if (top > vtop) { // (the same in every lane)
				const float to = pow2_below(top) * 2.0f, f = vtop / to;
				vtop = to;
#pragma unroll
				for (int t = 0; t < NT; t++)
#pragma unroll
					for (int m = 0; m < MT; m++)
						o[t][m] *= f;
			}
			vinv = P_SCALE / vtop;
		}

		// weights, in two f16 parts
		h8 ph[NT][2], pl[NT][2];
#pragma unroll
		for (int t = 0; t < NT; t++) {
			float top = -__builtin_inff();
			const uint32_t bits = (uint32_t)(vis[t] >> (16 * g)) & 0xffffu;
#pragma unroll
			for (int kt = 0; kt < 4; kt++)
#pragma unroll
				for (int i = 0; i < 4; i++) {
					float z = sc[t][kt][i] * qs[t];
					if (!whole && !(bits >> (4 * kt + i) & 1))
						z = -__builtin_inff();
					sc[t][kt][i] = z;
					top = __builtin_fmaxf(top, z);
				}
			top = __builtin_fmaxf(mx[t], max_g(top));
			const float base = top == -__builtin_inff() ? 0.0f : top;
			const float f = __builtin_amdgcn_exp2f(mx[t] - base);
			mx[t] = top;
			float add = 0.0f;
#pragma unroll
			for (int kt = 0; kt < 4; kt++) {
				float w[4];
#pragma unroll
				for (int i = 0; i < 4; i++) {
					w[i] = __builtin_amdgcn_exp2f(sc[t][kt][i] - base);
					add += w[i];
					if constexpr (I8) {
						w[i] *= vsc[kt][i] * vinv;
						if (!whole && !(bits >> (4 * kt + i) & 1))
							w[i] = 0.0f;
					} else {
						w[i] *= P_SCALE;
					}
				}
#pragma unroll
				for (int i = 0; i < 4; i += 2) {
					h2 hi, lo;
					split2(w[i], w[i + 1], hi, lo);
					const int e = (kt & 1) * 4 + i;
					ph[t][kt >> 1][e] = hi.x, ph[t][kt >> 1][e + 1] = hi.y;
					pl[t][kt >> 1][e] = lo.x, pl[t][kt >> 1][e + 1] = lo.y;
				}
			}
			sum[t] = sum[t] * f + add;
			if (!__all(f == 1.0f))
#pragma unroll
				for (int m = 0; m < MT; m++)
					o[t][m] *= f;
		}

		// O^T
#pragma unroll
		for (int m = 0; m < MT; m++) {
			const size_t col = at * HD + m * 16 + n16;
			h8 vf[2];
			if constexpr (I8) {
				const u4 w = *(reinterpret_cast<const u4 *>(c.v + col * PAGE) + g);
				vf[0] = codes8(w.x, w.y);
				vf[1] = codes8(w.z, w.w);
			} else {
				const u4 *vr = reinterpret_cast<const u4 *>(c.v + col * PAGE * 2) + 2 * g;
				u4 w[2] = {vr[0], vr[1]};
				if (!whole) {
					// a value that is not finite in a row that a token does
					// not see would reach it as 0 * inf: such values are
					// taken out here and come back for those that see them
					uint32_t odd = 0;
#pragma unroll
					for (int q = 0; q < 2; q++)
#pragma unroll
						for (int e = 0; e < 4; e++) {
							uint32_t x = w[q][e];
							if ((x & 0x7c00u) == 0x7c00u) {
								x &= 0xffff0000u;
								odd |= 1u << (8 * q + 2 * e);
							}
							if ((x & 0x7c000000u) == 0x7c000000u) {
								x &= 0xffffu;
								odd |= 2u << (8 * q + 2 * e);
							}
							w[q][e] = x;
						}
					if (__any(odd != 0)) {
						for (int r = 0; r < min(end, PAGE); r++) {
							const int src = (r >> 4) * 16; // the lane group that has row r
#pragma unroll
							for (int i = 0; i < 4; i++) {
								// (column 4 g + i of the tile: a lane of the O^T layout)
								if (!(__shfl(odd, src + 4 * g + i) >> (r & 15) & 1))
									continue;
								const float v = (float)reinterpret_cast<const _Float16 *>(
									c.v)[(at * HD + m * 16 + 4 * g + i) * PAGE + r];
#pragma unroll
								for (int t = 0; t < NT; t++)
									if (vis[t] >> r & 1)
										o[t][m][i] = v != v ? v : o[t][m][i] + v;
							}
						}
					}
				}
				vf[0] = __builtin_bit_cast(h8, w[0]);
				vf[1] = __builtin_bit_cast(h8, w[1]);
			}
#pragma unroll
			for (int t = 0; t < NT; t++)
#pragma unroll
				for (int q = 0; q < 2; q++) {
					o[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[q], pl[t][q], o[t][m], 0, 0, 0);
					o[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[q], ph[t][q], o[t][m], 0, 0, 0);
				}
		}
	}
	const float back = I8 ? vtop / P_SCALE : 1.0f / P_SCALE;

	// join the waves: each puts its rows into LDS ([wave][row][HD + 2])
	constexpr int LR = HD + 4;
	float *mine = lds + (size_t)wave * R * LR;
#pragma unroll
	for (int t = 0; t < NT; t++) {
		const float total = sum_g(sum[t]);
		float *row = mine + (16 * t + n16) * LR;
#pragma unroll
		for (int m = 0; m < MT; m++)
			*reinterpret_cast<f4 *>(row + m * 16 + 4 * g) = o[t][m] * back;
		if (g == 0) {
			row[HD] = bad ? __builtin_nanf("") : mx[t];
			row[HD + 1] = bad ? __builtin_nanf("") : total;
		}
	}
	__syncthreads();
	for (int e = threadIdx.x; e < R * HD; e += 64 * WK) {
		const int r = e / HD, i = e % HD, at = u.tile * R + r;
		if (at / group >= u.n)
			continue;
		float m = -__builtin_inff(), l = 0.0f, x = 0.0f;
#pragma unroll
		for (int w = 0; w < WK; w++)
			m = __builtin_fmaxf(m, lds[((size_t)w * R + r) * LR + HD]);
		const float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
		for (int w = 0; w < WK; w++) {
			const float *row = lds + ((size_t)w * R + r) * LR;
			const float f = __builtin_amdgcn_exp2f(row[HD] - base);
			l += row[HD + 1] * f;
			x += row[i] * f;
		}
		if (u.parts == 1) {
			a.out[(size_t)(u.t0 + at / group) * a.o_stride + (size_t)(u.head * group + at % group) * HD + i] =
				l == 0.0f ? 0.0f : x / l;
		} else {
			float *pr = part + (size_t)u.index * part_floats(R, HD) + (size_t)r * (HD + 2);
			pr[i] = x;
			if (i == 0) {
				pr[HD] = m;
				pr[HD + 1] = l;
			}
		}
	}
}

// Join the parts of a tile: one workgroup for each unit that is a tile's
// first part (a token row and head: HD threads at a time).
template <int HD>
__global__ __launch_bounds__(256) void attn_join_kernel(KvLayer c, KvSeqs s, AttnArgs a, int least, int R, const float *part)
{
	const int group = a.n_heads / c.kvh;
	Unit u;
	if (!find_unit(s, c.kvh, group, R, least, blockIdx.x, u) || u.part != 0 || u.parts == 1)
		return;
	if ((size_t)u.index + u.parts > gridDim.x)
		return; // (sequences that overlap: more units than the rows can have)
	for (int e = threadIdx.x; e < R * HD; e += 256) {
		const int r = e / HD, i = e % HD, at = u.tile * R + r;
		if (at / group >= u.n)
			break;
		const float *row = part + (size_t)u.index * part_floats(R, HD) + (size_t)r * (HD + 2);
		const size_t step = part_floats(R, HD);
		float m = -__builtin_inff(), l = 0.0f, x = 0.0f;
		for (int q = 0; q < u.parts; q++)
			m = __builtin_fmaxf(m, row[q * step + HD]);
		const float base = m == -__builtin_inff() ? 0.0f : m;
		for (int q = 0; q < u.parts; q++) {
			const float f = __builtin_amdgcn_exp2f(row[q * step + HD] - base);
			l += row[q * step + HD + 1] * f;
			x += row[q * step + i] * f;
		}
		a.out[(size_t)(u.t0 + at / group) * a.o_stride + (size_t)(u.head * group + at % group) * HD + i] =
			l == 0.0f ? 0.0f : x / l;
	}
}

// ---------------------------------------------------------------- launch
struct Shape {
	int nt, wk, least;
	size_t units; // at most
};

static Shape attn_shape(const KvLayer &c, const KvSeqs &s, const AttnArgs &a)
{
	const size_t group = a.n_heads / c.kvh, rows = (size_t)s.n_tokens * group;
	Shape h;
	const size_t avg = rows / s.n_seqs;
	h.nt = avg <= 16 ? 1 : avg <= 32 ? 2 : 4;
	h.wk = h.nt == 1 ? 8 : 4;
	h.least = h.wk;
	h.units = ATTN_UNITS + (rows / (16 * h.nt) + s.n_seqs) * c.kvh;
	return h;
}

size_t attention_work_bytes(const KvLayer &c, const KvSeqs &s, const AttnArgs &a)
{
	const Shape h = attn_shape(c, s, a);
	return h.units * part_floats(16 * h.nt, c.hd) * sizeof(float);
}

template <int HD, bool I8, int NT, int WK>
static hipError_t go(const Shape &h, const KvLayer &c, const KvSeqs &s, const AttnArgs &a, float *part, hipStream_t st)
{
	const size_t lds = (size_t)WK * 16 * NT * (HD + 4) * sizeof(float);
	const hipError_t e = ensure_lds_limit((const void *)attn_kernel<HD, I8, NT, WK>, lds);
	if (e != hipSuccess)
		return e;
	tie_launch(attn_kernel<HD, I8, NT, WK>, dim3(h.units), dim3(64 * WK), lds, st, c, s, a, h.least, part);
	tie_launch(attn_join_kernel<HD>, dim3(h.units), dim3(256), 0, st, c, s, a, h.least, 16 * NT, (const float *)part);
	return hipGetLastError();
}

hipError_t launch_attention(const KvLayer &c, const KvSeqs &s, const AttnArgs &a, void *work, hipStream_t st)
{
	const Shape h = attn_shape(c, s, a);
	float *part = reinterpret_cast<float *>(work);
#define TIE_ATTN(HD, I8)                                                             \
	(h.nt == 1 ? go<HD, I8, 1, 8>(h, c, s, a, part, st)                         \
	 : h.nt == 2 ? go<HD, I8, 2, 4>(h, c, s, a, part, st) : go<HD, I8, 4, 4>(h, c, s, a, part, st))
	if (c.hd == 128)
		return c.i8 ? TIE_ATTN(128, true) : TIE_ATTN(128, false);
	return c.i8 ? TIE_ATTN(64, true) : TIE_ATTN(64, false);
#undef TIE_ATTN
}

} // namespace tie
