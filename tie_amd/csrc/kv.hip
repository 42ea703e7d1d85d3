// kv.hip -- the cache around the attention: norm and rotation of queries and
// keys with the quantised write (append), reading back, and moving the
// accepted path's rows (keep).
#include "kv.h"

namespace tie {

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

// A wave takes heads of one token, HD / 2 lanes each: a lane holds the pair
// (x[i], x[i + HD / 2]) that the rotation turns.  All of it in 64 bits up to
// the one rounding to F32: positions reach where a 32-bit angle is off by a
// thousandth, and a key's code must not depend on the order of a 32-bit sum.
template <int HD, bool I8>
__global__ __launch_bounds__(256) void kv_append_kernel(KvLayer c, KvSeqs s, AppendArgs a, int per_wave)
{
	constexpr int L = HD / 2, G = 64 / L; // lanes of a head, heads of a wave at a time
	const int t = blockIdx.x, lane = threadIdx.x & 63, i = lane % L;
	const int wave = blockIdx.y * 4 + (threadIdx.x >> 6);
	int t0, n;
	const int b = seq_of_token(s, t, t0, n);
	if (b < 0)
		return;
	const int len = s.len[b], row = len + (t - t0);
	const bool fits = seq_fits(s, len, n);
	const int page = fits ? page_of(s, c.n_pages, b, row) : -1, r = fits ? row % PAGE : 0;
	const int n_all = a.n_heads + 2 * c.kvh;
	double cs = 0.0, sn = 0.0;
	{
		const int pos = a.pos ? a.pos[t] : row;
		const double angle = (double)pos * exp2((double)i * (-2.0 / HD) * a.log2_theta);
		sincos(angle, &sn, &cs);
	}
	for (int u = 0; u < per_wave; u++) {
		const int h = (wave * per_wave + u) * G + lane / L;
		const bool on = h < n_all;
		const int kv = h - a.n_heads, head = kv < 0 ? h : kv < c.kvh ? kv : kv - c.kvh;
		const bool is_q = kv < 0, is_v = kv >= c.kvh;
		float x0 = 0.0f, x1 = 0.0f;
		if (on) {
			const float *p = (is_q ? a.q + (size_t)t * a.q_stride
				       : is_v  ? a.v + (size_t)t * a.v_stride
					       : a.k + (size_t)t * a.k_stride) +
					 (size_t)head * HD;
			x0 = p[i];
			x1 = p[i + L];
		}
		const float *w = is_q ? a.q_norm : a.k_norm;
		if (!is_v) {
			double y0 = x0, y1 = x1;
			double ss = y0 * y0 + y1 * y1;
#pragma unroll
			for (int m = 1; m < L; m <<= 1)
				ss += __shfl_xor(ss, m);
			if (w) {
				const double f = 1.0 / sqrt(ss / HD + a.eps);
				y0 = y0 * f * (double)w[i];
				y1 = y1 * f * (double)w[i + L];
			}
			x0 = (float)(y0 * cs - y1 * sn);
			x1 = (float)(y1 * cs + y0 * sn);
		}
		if (on && is_q) {
			float *o = a.q_out + (size_t)t * a.qo_stride + (size_t)head * HD;
			o[i] = x0;
			o[i + L] = x1;
		}
		// (every lane of a head takes part in its row's largest magnitude)
		float scale = 0.0f;
		if (I8) {
			float m = __builtin_fmaxf(__builtin_fabsf(x0), __builtin_fabsf(x1));
			bool bad = !(__builtin_fabsf(x0) < __builtin_inff()) || !(__builtin_fabsf(x1) < __builtin_inff());
#pragma unroll
			for (int q = 1; q < L; q <<= 1) {
				m = __builtin_fmaxf(m, __shfl_xor(m, q));
				bad |= __shfl_xor((int)bad, q) != 0;
			}
			scale = bad ? __builtin_nanf("") : m / 127.0f;
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
	const int units = (a.n_heads + 2 * c.kvh + 128 / c.hd - 1) / (128 / c.hd); // waves with a head (pair) each
	// a wave takes one unit where there are few tokens, else several: the
	// angles' cosines are the same for all of them
	int per = 1;
	while (per < 16 && (size_t)s.n_tokens * units > (size_t)4096 * per)
		per *= 2;
	const dim3 grid(s.n_tokens, (units + 4 * per - 1) / (4 * per));
	auto go = [&](auto kern) { tie_launch(kern, grid, dim3(256), 0, st, c, s, a, per); };
	if (c.hd == 128)
		c.i8 ? go(kv_append_kernel<128, true>) : go(kv_append_kernel<128, false>);
	else
		c.i8 ? go(kv_append_kernel<64, true>) : go(kv_append_kernel<64, false>);
	return hipGetLastError();
}

// ---------------------------------------------------------------- read
// One workgroup a token row and layer.  A row that the table does not reach
// reads as NaN.
template <bool I8>
__global__ __launch_bounds__(256) void kv_read_kernel(KvLayer c, KvSeqs s, float *k_out, float *v_out)
{
	const int t = blockIdx.x, layer = blockIdx.y, w = c.kvh * c.hd;
	int t0, n;
	const int b = seq_of_token(s, t, t0, n);
	if (b < 0)
		return;
	const int len = s.len[b], row = len + (t - t0);
	const int page = seq_fits(s, len, n) ? page_of(s, c.n_pages, b, row) : -1, r = page < 0 ? 0 : row % PAGE;
	const size_t o = ((size_t)layer * s.n_tokens + t) * w;
	for (int e = threadIdx.x; e < w; e += 256) {
		if (page < 0) {
			k_out[o + e] = v_out[o + e] = __builtin_nanf("");
			continue;
		}
		const int h = e / c.hd, i = e % c.hd;
		const size_t at = (size_t)page * c.kvh + h;
		const size_t ek = (size_t)layer * c.layer_bytes + (at * PAGE + r) * c.hd + i,
			     ev = (size_t)layer * c.layer_bytes + (at * c.hd + i) * PAGE + r;
		if (I8) {
			const size_t sc = (size_t)layer * c.layer_scales + at * PAGE + r;
			k_out[o + e] = (float)reinterpret_cast<const int8_t *>(c.k)[ek] * c.ks[sc];
			v_out[o + e] = (float)reinterpret_cast<const int8_t *>(c.v)[ev] * c.vs[sc];
		} else {
			// (layer_bytes counts two for an element)
			const size_t half = (size_t)layer * (c.layer_bytes / 2);
			k_out[o + e] = (float)reinterpret_cast<const _Float16 *>(c.k)[half + (at * PAGE + r) * c.hd + i];
			v_out[o + e] = (float)reinterpret_cast<const _Float16 *>(c.v)[half + (at * c.hd + i) * PAGE + r];
		}
	}
}

hipError_t launch_kv_read(const KvLayer &c, int n_layers, const KvSeqs &s, float *k_out, float *v_out, hipStream_t st)
{
	const dim3 grid(s.n_tokens, n_layers);
	if (c.i8)
		tie_launch(kv_read_kernel<true>, grid, dim3(256), 0, st, c, s, k_out, v_out);
	else
		tie_launch(kv_read_kernel<false>, grid, dim3(256), 0, st, c, s, k_out, v_out);
	return hipGetLastError();
}

// ---------------------------------------------------------------- keep
// Row len + path[j] to row len + j for j < n_keep, in every layer.  A thread
// has one column (or the two scales) of one kv head and layer and moves its
// rows in order, KEEP_BATCH loads before their stores: a path ascends, so
// path[j] >= j and no store reaches a row that a later load wants.
constexpr int KEEP_BATCH = 8;

// How many entries of sequence b's path can be moved: up to the first that
// does not ascend or is none of its n nodes.
__device__ __forceinline__ int keep_count(const int32_t *path, int want, int n)
{
	int prev = -1, j = 0;
	for (; j < want; j++) {
		const int p = path[j];
		if (p <= prev || p >= n)
			break;
		prev = p;
	}
	return j;
}

template <typename T>
__device__ __forceinline__ void keep_rows(T *base, size_t page_stride, int row_stride, const KvLayer &c, const KvSeqs &s,
					  int b, int len, const int32_t *path, int count)
{
	for (int j0 = 0; j0 < count; j0 += KEEP_BATCH) {
		T v[KEEP_BATCH];
		int to[KEEP_BATCH];
#pragma unroll
		for (int q = 0; q < KEEP_BATCH; q++) {
			const int j = j0 + q;
			to[q] = -1;
			if (j < count && path[j] != j) {
				const int from = page_of(s, c.n_pages, b, len + path[j]);
				to[q] = page_of(s, c.n_pages, b, len + j);
				if (from < 0)
					to[q] = -1;
				else
					v[q] = base[from * page_stride + (size_t)((len + path[j]) % PAGE) * row_stride];
			}
		}
#pragma unroll
		for (int q = 0; q < KEEP_BATCH; q++)
			if (to[q] >= 0)
				base[to[q] * page_stride + (size_t)((len + j0 + q) % PAGE) * row_stride] = v[q];
	}
}

template <typename T>
__global__ __launch_bounds__(256) void kv_keep_kernel(KvLayer c, KvSeqs s, const int32_t *path, int max_path,
						      const int32_t *n_keep, int32_t *len_out)
{
	const int h = blockIdx.x % c.kvh, layer = blockIdx.x / c.kvh, b = blockIdx.y, i = threadIdx.x % c.hd;
	const bool is_v = (int)threadIdx.x >= c.hd;
	int t0, n;
	seq_tokens(s, b, t0, n);
	const int len = s.len[b];
	const int32_t *pb = path + (size_t)b * max_path;
	const int count = seq_fits(s, len, n) ? keep_count(pb, min(n_keep[b], max_path), n) : 0;
	T *base = reinterpret_cast<T *>((is_v ? c.v : c.k) + (size_t)layer * c.layer_bytes) + (size_t)h * PAGE * c.hd;
	keep_rows(base + (is_v ? i * PAGE : i), (size_t)c.kvh * PAGE * c.hd, is_v ? 1 : c.hd, c, s, b, len, pb, count);
	if (c.i8 && i == 0)
		keep_rows((is_v ? c.vs : c.ks) + (size_t)layer * c.layer_scales + (size_t)h * PAGE, (size_t)c.kvh * PAGE, 1, c, s,
			  b, len, pb, count);
	// (written last by a workgroup of its own that moves nothing: len_out may
	// be len itself, which the others read)
}

__global__ __launch_bounds__(64) void kv_keep_len_kernel(KvSeqs s, const int32_t *path, int max_path,
							 const int32_t *n_keep, int32_t *len_out)
{
	const int b = blockIdx.x * 64 + threadIdx.x;
	if (b >= s.n_seqs)
		return;
	int t0, n;
	seq_tokens(s, b, t0, n);
	const int len = s.len[b];
	len_out[b] = len + (seq_fits(s, len, n) ? keep_count(path + (size_t)b * max_path, min(n_keep[b], max_path), n) : 0);
}

hipError_t launch_kv_keep(const KvLayer &c, int n_layers, const KvSeqs &s, const int32_t *path, int max_path,
			  const int32_t *n_keep, int32_t *len_out, hipStream_t st)
{
	const dim3 grid(n_layers * c.kvh, s.n_seqs), block(2 * c.hd);
	if (c.i8)
		tie_launch(kv_keep_kernel<uint8_t>, grid, block, 0, st, c, s, path, max_path, n_keep, len_out);
	else
		tie_launch(kv_keep_kernel<uint16_t>, grid, block, 0, st, c, s, path, max_path, n_keep, len_out);
	if (len_out)
		tie_launch(kv_keep_len_kernel, dim3((s.n_seqs + 63) / 64), dim3(64), 0, st, s, path, max_path, n_keep, len_out);
	return hipGetLastError();
}

} // namespace tie
