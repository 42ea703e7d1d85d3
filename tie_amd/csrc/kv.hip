// kv.hip -- the cache around the attention: norm and rotation of queries and
// keys with the quantised write (append), reading back, and moving the
// accepted path's rows (keep).
#include "kv.h"

namespace tie {

typedef float f4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- append
// int8 code of x for a row's scale (0 for a row of zeros, whose scale is 0,
// and for a row that is not finite, whose scale is NaN).
__device__ __forceinline__ int8_t code_of(float x, float scale)
{
	if (!(scale > 0.0f))
		return 0;
	const float r = __builtin_rintf(x / scale);
	return (int8_t)(int)__builtin_fminf(__builtin_fmaxf(r, -127.0f), 127.0f);
}

// f16 of x, the largest finite value where it would become infinite (a cache
// row then spoils one weight, not its whole column); NaN stays.
__device__ __forceinline__ _Float16 half_of(float x)
{
	if (__builtin_fabsf(x) > 65504.0f)
		x = __builtin_copysignf(65504.0f, x);
	return (_Float16)x;
}

// A workgroup has one token; its waves take heads in turn, HD / 2 lanes each: a
// lane holds the pair (x[i], x[i + HD / 2]) that the rotation turns, and its
// cosine and sine stay with it.  All of it in 64 bits up to the one rounding to
// F32: positions reach where a 32-bit angle is off by a thousandth, and a key's
// code must not depend on the order of a 32-bit sum.  One token: bound by its
// chain of steps (position, angle, sincos; row, norm, code), 3.6 us (on the default
// stream 4.1).  Many: by the bytes, the 64-bit arithmetic (about 60 instructions
// for 64 pairs) and the V columns' pieces (a row's values lie PAGE apart) together:
// 2048 tokens of 40 heads 22.5 us, 3.5 TB/s; 20 to 21.5 without any one of them.
constexpr int DIES = 8;

template <int HD, bool I8>
__global__ __launch_bounds__(256) void kv_append_kernel(KvLayer c, KvSeqs s, AppendArgs a, int per_wave)
{
	constexpr int L = HD / 2, G = 64 / L; // lanes of a head, heads of a wave at a time
	// (workgroups go to the dies in turn: each die has neighbouring tokens)
	const int t = blockIdx.x % DIES * (gridDim.x / DIES) + blockIdx.x / DIES;
	const int lane = threadIdx.x & 63, i = lane % L, part = lane / L;
	if (t >= s.n_tokens)
		return;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	int t0, n;
	const int b = seq_of_token(s, t, t0, n);
	if (b < 0)
		return;
	const int n_all = a.n_heads + 2 * c.kvh;
	const int u0 = blockIdx.y * per_wave * 4 + wave; // this wave's units: u0, u0 + 4, ...
	auto source = [&](int h, int &kv) {
		kv = h - a.n_heads;
		return kv < 0 ? a.q + (size_t)t * a.q_stride + (size_t)h * HD
		       : kv < c.kvh ? a.k + (size_t)t * a.k_stride + (size_t)kv * HD
				    : a.v + (size_t)t * a.v_stride + (size_t)(kv - c.kvh) * HD;
	};
	// the first head's row and the norms' weights are requested before the
	// position is known
	float n0 = 0.0f, n1 = 0.0f;
	auto fetch = [&](int u) {
		int kv;
		const int h = u * G + part;
		if (h < n_all) {
			const float *p = source(h, kv);
			n0 = p[i];
			n1 = p[i + L];
		}
	};
	fetch(u0);
	const double wq0 = a.q_norm ? (double)a.q_norm[i] : 1.0, wq1 = a.q_norm ? (double)a.q_norm[i + L] : 1.0;
	const double wk0 = a.k_norm ? (double)a.k_norm[i] : 1.0, wk1 = a.k_norm ? (double)a.k_norm[i + L] : 1.0;
	const int len = s.len[b];
	const bool fits = seq_fits(s, len, n);
	const int row = fits ? len + (t - t0) : 0;
	const int page = fits ? page_of(s, c.n_pages, b, row) : -1, r = row % PAGE;
	// (no row: no position)
	const double at = a.pos ? (double)a.pos[t] : fits ? (double)row : __builtin_nan("");
	double cs, sn;
	sincos(at * exp2((double)i * (-2.0 / HD) * a.log2_theta), &sn, &cs);
	for (int u = 0; u < per_wave; u++) {
		const int h = (u0 + 4 * u) * G + part;
		if ((u0 + 4 * u) * G >= n_all)
			break;
		const bool on = h < n_all;
		const int kv = h - a.n_heads, head = kv < 0 ? h : kv < c.kvh ? kv : kv - c.kvh;
		const bool is_q = kv < 0, is_v = kv >= c.kvh;
		float x0 = n0, x1 = n1;
		if (u + 1 < per_wave)
			fetch(u0 + 4 * (u + 1));
		if (!__all(is_v)) {
			double y0 = x0, y1 = x1;
			if (is_q ? a.q_norm != nullptr : a.k_norm != nullptr) {
				// (a head's sum lies in its last lane)
				const double ss = running_of<L>(__builtin_fma(y0, y0, y1 * y1));
				const double total = G == 1 ? of_lane(ss, 63) : part ? of_lane(ss, 63) : of_lane(ss, 31);
				const double f = rsqrt(__builtin_fma(total, 1.0 / HD, a.eps));
				y0 *= f * (is_q ? wq0 : wk0);
				y1 *= f * (is_q ? wq1 : wk1);
			}
			const float z0 = (float)__builtin_fma(y0, cs, -(y1 * sn)), z1 = (float)__builtin_fma(y1, cs, y0 * sn);
			x0 = is_v ? x0 : z0;
			x1 = is_v ? x1 : z1;
		}
		if (on && is_q) {
			float *o = a.q_out + (size_t)t * a.qo_stride + (size_t)head * HD;
			o[i] = x0;
			o[i + L] = x1;
		}
		if (__all(is_q))
			continue;
		// (every lane of a head takes part in its row's largest magnitude)
		float scale = 0.0f;
		if (I8) {
			const float big = __builtin_fmaxf(__builtin_fabsf(x0), __builtin_fabsf(x1));
			const unsigned long long mine = G == 1 ? ~0ull : part ? 0xffffffff00000000ull : 0xffffffffull;
			const bool bad = (__ballot(!(__builtin_fabsf(x0) < __builtin_inff()) || !(__builtin_fabsf(x1) < __builtin_inff())) & mine) != 0;
			const float m = running_max_of<L>(big);
			const int top = G == 1 || part ? 63 : 31;
			const float most = __shfl(m, top);
			scale = bad ? __builtin_nanf("") : most / 127.0f;
		}
		if (!on || is_q || page < 0)
			continue;
		const size_t at = (size_t)page * c.kvh + head; // this page's rows of this kv head
		if (I8 && i == 0)
			(is_v ? c.vs : c.ks)[at * PAGE + r] = scale;
		const size_t e0 = at * PAGE * HD + (is_v ? (size_t)i * PAGE + r : (size_t)r * HD + i);
		const size_t e1 = e0 + (is_v ? (size_t)L * PAGE : (size_t)L);
		if (I8) {
			int8_t *o = reinterpret_cast<int8_t *>(is_v ? c.v : c.k);
			o[e0] = code_of(x0, scale);
			o[e1] = code_of(x1, scale);
		} else {
			_Float16 *o = reinterpret_cast<_Float16 *>(is_v ? c.v : c.k);
			o[e0] = half_of(x0);
			o[e1] = half_of(x1);
		}
	}
}

hipError_t launch_kv_append(const KvLayer &c, const KvSeqs &s, const AppendArgs &a, hipStream_t st)
{
	const int units = (a.n_heads + 2 * c.kvh + 128 / c.hd - 1) / (128 / c.hd); // a wave's share at a time: a head of 128, two of 64
	// a wave takes one unit where there are few tokens, else as many as leave
	// 4096 waves: the angles' cosines are the same for all of them
	const size_t all = (size_t)s.n_tokens * units;
	int per = all > 4096 ? (int)(all / 4096) : 1;
	per = per > (units + 3) / 4 ? (units + 3) / 4 : per;
	const dim3 grid((s.n_tokens + DIES - 1) / DIES * DIES, (units + 4 * per - 1) / (4 * per));
	auto go = [&](auto kern) { tie_launch(kern, grid, dim3(256), 0, st, c, s, a, per); };
	if (c.hd == 128)
		c.i8 ? go(kv_append_kernel<128, true>) : go(kv_append_kernel<128, false>);
	else
		c.i8 ? go(kv_append_kernel<64, true>) : go(kv_append_kernel<64, false>);
	return hipGetLastError();
}

// ---------------------------------------------------------------- read
// A workgroup has the rows of one sequence in one page, of one kv head and layer.
// K rows go through as they lie; V columns come into LDS in 16-byte pieces and
// leave it as rows (columns 4 bytes further apart than they are long: the lanes
// of a row read different banks).  Bound by the F32 rows written, which go past
// the caches (nontemporal stores: 30001 int8 rows 26.5 us, 5.8 TB/s; else 41.4).
// Rows that the table does not reach read as NaN.
template <int HD, bool I8>
__global__ __launch_bounds__(256) void kv_read_kernel(KvLayer c, KvSeqs s, float *k_out, float *v_out)
{
	constexpr int E = I8 ? 1 : 2, CS = PAGE * E + 4; // bytes of a column in LDS
	__shared__ __attribute__((aligned(16))) uint8_t tile[HD * CS];
	__shared__ float scale[PAGE];
	const int lane = threadIdx.x & 63, h = blockIdx.y, layer = blockIdx.z;
	// the sequence and page of this workgroup
	int b = -1, t0 = 0, n = 0, len = 0, p = 0;
	for (int b0 = 0, before = 0; b0 < s.n_seqs; b0 += 64) {
		int st0 = 0, sn = 0, sl = 0, pages = 0;
		if (b0 + lane < s.n_seqs) {
			sl = s.len[b0 + lane];
			seq_tokens(s, b0 + lane, st0, sn);
			if (sn > 0) {
				// (rows that do not fit: one workgroup for each 64 of them)
				const int from = seq_fits(s, sl, sn) ? sl % PAGE : 0;
				pages = (from + sn + PAGE - 1) / PAGE;
			}
		}
		const int incl = s.n_seqs > 1 ? (int)running_of<64>((double)pages) : pages;
		const unsigned long long past = __ballot(before + incl > (int)blockIdx.x);
		if (past) {
			const int l = __builtin_ctzll(past);
			b = b0 + l;
			t0 = __builtin_amdgcn_readlane(st0, l);
			n = __builtin_amdgcn_readlane(sn, l);
			len = __builtin_amdgcn_readlane(sl, l);
			p = (int)blockIdx.x - before - __builtin_amdgcn_readlane(incl - pages, l);
			break;
		}
		before += __builtin_amdgcn_readlane(incl, 63);
	}
	if (b < 0)
		return;
	const bool fits = seq_fits(s, len, n);
	// rows [r0, r1) of the page are token rows t0 + first ...
	const int from = fits ? len % PAGE : 0;
	const int r0 = p == 0 ? from : 0, r1 = min(PAGE, from + n - p * PAGE), first = t0 + p * PAGE + r0 - from;
	const int page = fits ? page_of(s, c.n_pages, b, len - from + p * PAGE) : -1;
	const size_t width = (size_t)c.kvh * HD;
	const size_t o = ((size_t)layer * s.n_tokens + first) * width + (size_t)h * HD;
	if (page < 0) {
		for (int e = threadIdx.x; e < (r1 - r0) * HD; e += 256)
			k_out[o + e / HD * width + e % HD] = v_out[o + e / HD * width + e % HD] = __builtin_nanf("");
		return;
	}
	const size_t at = (size_t)page * c.kvh + h;
	const uint8_t *k = c.k + layer * c.layer_bytes + at * PAGE * HD * E, *v = c.v + layer * c.layer_bytes + at * PAGE * HD * E;
	const float *ks = I8 ? c.ks + layer * c.layer_scales + at * PAGE : nullptr;
	constexpr int VP = PAGE * E / 16; // pieces of a column
	for (int e = threadIdx.x; e < HD * VP; e += 256) {
		const int col = e / VP, q = e % VP;
		if ((q + 1) * 16 / E <= r0 || q * 16 / E >= r1)
			continue;
		const uint4 x = reinterpret_cast<const uint4 *>(v)[e];
		uint32_t *to = reinterpret_cast<uint32_t *>(tile + col * CS + q * 16);
		to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
	}
	if (I8 && threadIdx.x < PAGE)
		scale[threadIdx.x] = c.vs[layer * c.layer_scales + at * PAGE + threadIdx.x];
	// K: 4 values of a row to a thread
	for (int e = threadIdx.x; e < (r1 - r0) * (HD / 4); e += 256) {
		const int r = r0 + e / (HD / 4), i = e % (HD / 4) * 4;
		float x[4];
		if (I8) {
			const uint32_t w = *reinterpret_cast<const uint32_t *>(k + r * HD + i);
			const float f = ks[r];
#pragma unroll
			for (int q = 0; q < 4; q++)
				x[q] = sbyte_f(w, q) * f;
		} else {
			typedef _Float16 h4 __attribute__((ext_vector_type(4)));
			const h4 w = *reinterpret_cast<const h4 *>(k + (r * HD + i) * 2);
#pragma unroll
			for (int q = 0; q < 4; q++)
				x[q] = (float)w[q];
		}
		float *to = k_out + o + (size_t)(r - r0) * width + i;
		if (((uintptr_t)to & 15) == 0) {
			__builtin_nontemporal_store((f4){x[0], x[1], x[2], x[3]}, reinterpret_cast<f4 *>(to));
		} else {
#pragma unroll
			for (int q = 0; q < 4; q++)
				to[q] = x[q];
		}
	}
	__syncthreads();
	// V: a column to a thread, a word's rows at a time
	constexpr int W = 4 / E;
	for (int e = threadIdx.x; e < (PAGE / W) * HD; e += 256) {
		const int i = e % HD, r = e / HD * W;
		if (r + W <= r0 || r >= r1)
			continue;
		const uint32_t w = *reinterpret_cast<const uint32_t *>(tile + i * CS + r * E);
#pragma unroll
		for (int q = 0; q < W; q++)
			if (r + q >= r0 && r + q < r1) {
				const float x = I8 ? sbyte_f(w, q) * scale[r + q]
						   : (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> (16 * q)));
				__builtin_nontemporal_store(x, v_out + o + (size_t)(r + q - r0) * width + i);
			}
	}
}

hipError_t launch_kv_read(const KvLayer &c, int n_layers, const KvSeqs &s, float *k_out, float *v_out, hipStream_t st)
{
	// pages: a sequence's rows fill n / 64 of them, less what is left at both ends
	const size_t seqs = s.n_seqs < s.n_tokens ? s.n_seqs : s.n_tokens;
	const dim3 grid((uint32_t)((s.n_tokens + seqs * 2 * (PAGE - 1)) / PAGE), c.kvh, n_layers);
	auto go = [&](auto kern) { tie_launch(kern, grid, dim3(256), 0, st, c, s, k_out, v_out); };
	if (c.hd == 128)
		c.i8 ? go(kv_read_kernel<128, true>) : go(kv_read_kernel<128, false>);
	else
		c.i8 ? go(kv_read_kernel<64, true>) : go(kv_read_kernel<64, false>);
	return hipGetLastError();
}

// ---------------------------------------------------------------- keep
// Row len + path[j] to row len + j for j < n_keep, in every layer.  A workgroup
// has one kv head and layer of a sequence, a thread one column of K or V: it
// moves its rows in order, KEEP_BATCH loads before their stores.  A path ascends,
// so path[j] >= j and no store reaches a row that a later load wants.  Where the
// rows lie is worked out once, by the first wave.  Bound by V's lines (a row's values
// lie in one for each column): 16 paths in 48 layers of 4 heads 16 us; one path 4.3,
// the chain of its steps.
constexpr int KEEP_BATCH = 8;
constexpr int KEEP_TABLE = 64; // path entries at a time

// How many entries of sequence b's path can be moved: up to the first that
// does not ascend, is none of its n nodes, or lies on no page or is to.  A wave,
// whose lanes have the first entries already (they are requested with the
// lengths), and get those entries' pages, before and after.  len + n lies within
// the page table.
__device__ __forceinline__ int keep_count(const KvSeqs &s, int n_pages, int b, int len, const int32_t *path, int mine, int want,
					  int n, int &from, int &to)
{
	const int lane = threadIdx.x & 63;
	from = to = -1;
	for (int j0 = 0; j0 < want; j0 += 64) {
		const int j = j0 + lane;
		const bool in = j < want;
		const int p = j0 == 0 ? mine : in ? path[j] : 0;
		// (both pages requested before anything else is known of the entry; the
		// first row's stand for those of an entry that names no node)
		const bool node = in && p >= 0 && p < n && j < n;
		const int f = page_of(s, n_pages, b, node ? len + p : 0), t = page_of(s, n_pages, b, node ? len + j : 0);
		const int before = __shfl_up(p, 1), prev = lane > 0 ? before : j0 > 0 ? path[j0 - 1] : -1;
		if (j0 == 0) {
			from = f;
			to = t;
		}
		const unsigned long long bad = __ballot(in && !(node && p > prev && f >= 0 && t >= 0));
		if (bad)
			return j0 + __builtin_ctzll(bad);
	}
	return want > 0 ? want : 0;
}

__device__ __forceinline__ int first_entry(const int32_t *path, int max_path)
{
	const int lane = threadIdx.x & 63;
	return path[lane < max_path ? lane : max_path - 1];
}

template <typename T>
__global__ __launch_bounds__(256) void kv_keep_kernel(KvLayer c, KvSeqs s, const int32_t *path, int max_path,
						      const int32_t *n_keep, int32_t *len_out)
{
	// source and target, as page * PAGE + row; target -1: nothing to move
	__shared__ int from[KEEP_TABLE], to[KEEP_TABLE], rows;
	const int h = blockIdx.x % c.kvh, layer = blockIdx.x / c.kvh, b = blockIdx.y, i = threadIdx.x % c.hd;
	const bool is_v = (int)threadIdx.x >= c.hd;
	const int32_t *pb = path + (size_t)b * max_path;
	const int len = s.len[b];
	// entry j of the path, a thread's: its pages are fp and tp
	auto put = [&](int j, int p, int fp, int tp) {
		from[threadIdx.x] = fp * PAGE + (len + p) % PAGE;
		to[threadIdx.x] = p == j ? -1 : tp;
	};
	if (threadIdx.x < 64) {
		int t0, n, fp, tp;
		const int entry = first_entry(pb, max_path), want = min(n_keep[b], max_path);
		seq_tokens(s, b, t0, n);
		const int count = seq_fits(s, len, n) ? keep_count(s, c.n_pages, b, len, pb, entry, want, n, fp, tp) : 0;
		if ((int)threadIdx.x < count)
			put(threadIdx.x, entry, fp, tp);
		if (threadIdx.x == 0) {
			rows = count;
			if (len_out && blockIdx.x == 0)
				len_out[b] = len + count;
		}
	}
	__syncthreads();
	const int count = rows;
	T *base = reinterpret_cast<T *>((is_v ? c.v : c.k) + (size_t)layer * c.layer_bytes) + (size_t)h * PAGE * c.hd;
	float *scales = (is_v ? c.vs : c.ks) + (size_t)layer * c.layer_scales + (size_t)h * PAGE;
	const size_t page = (size_t)c.kvh * PAGE * c.hd;
	for (int j1 = 0; j1 < count; j1 += KEEP_TABLE) {
		const int m = min(KEEP_TABLE, count - j1);
		if (j1) {
			__syncthreads();
			if ((int)threadIdx.x < m) {
				const int j = j1 + threadIdx.x, p = pb[j];
				put(j, p, page_of(s, c.n_pages, b, len + p), page_of(s, c.n_pages, b, len + j));
			}
			__syncthreads();
		}
		for (int j0 = 0; j0 < m; j0 += KEEP_BATCH) {
			T x[KEEP_BATCH];
			float f[KEEP_BATCH];
#pragma unroll
			for (int q = 0; q < KEEP_BATCH; q++) {
				const int j = j0 + q;
				if (j >= m || to[j] < 0)
					continue;
				const int fp = from[j] / PAGE, fr = from[j] % PAGE;
				x[q] = base[fp * page + (is_v ? i * PAGE + fr : fr * c.hd + i)];
				if (sizeof(T) == 1 && i == 0)
					f[q] = scales[(size_t)fp * c.kvh * PAGE + fr];
			}
#pragma unroll
			for (int q = 0; q < KEEP_BATCH; q++) {
				const int j = j0 + q;
				if (j >= m || to[j] < 0)
					continue;
				const int tr = (len + j1 + j) % PAGE;
				base[to[j] * page + (is_v ? i * PAGE + tr : tr * c.hd + i)] = x[q];
				if (sizeof(T) == 1 && i == 0)
					scales[(size_t)to[j] * c.kvh * PAGE + tr] = f[q];
			}
		}
	}
}

__global__ __launch_bounds__(64) void kv_keep_len_kernel(KvSeqs s, int n_pages, const int32_t *path, int max_path,
							 const int32_t *n_keep, int32_t *len_out)
{
	const int b = blockIdx.x;
	int t0, n;
	seq_tokens(s, b, t0, n);
	const int len = s.len[b];
	const int32_t *pb = path + (size_t)b * max_path;
	const int entry = first_entry(pb, max_path), want = min(n_keep[b], max_path);
	int from, to;
	const int count = seq_fits(s, len, n) ? keep_count(s, n_pages, b, len, pb, entry, want, n, from, to) : 0;
	if (threadIdx.x == 0)
		len_out[b] = len + count;
}

hipError_t launch_kv_keep(const KvLayer &c, int n_layers, const KvSeqs &s, const int32_t *path, int max_path,
			  const int32_t *n_keep, int32_t *len_out, hipStream_t st)
{
	const dim3 grid(n_layers * c.kvh, s.n_seqs), block(2 * c.hd);
	// (lengths updated in place: by a launch behind the one that reads them)
	int32_t *now = len_out == s.len ? nullptr : len_out;
	if (c.i8)
		tie_launch(kv_keep_kernel<uint8_t>, grid, block, 0, st, c, s, path, max_path, n_keep, now);
	else
		tie_launch(kv_keep_kernel<uint16_t>, grid, block, 0, st, c, s, path, max_path, n_keep, now);
	if (len_out && !now)
		tie_launch(kv_keep_len_kernel, dim3(s.n_seqs), dim3(64), 0, st, s, c.n_pages, path, max_path, n_keep,
			   len_out);
	return hipGetLastError();
}

} // namespace tie
