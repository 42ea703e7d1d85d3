// kv.h -- the paged key/value cache and its sequences, as the kernels of the
// attention half see them (kv.hip, attention.hip).
#pragma once
#include "common.h"

namespace tie {

constexpr int PAGE = TIE_HIP_PAGE_ROWS; // rows of a page: one 64-bit mask word, four 16-row matrix-core tiles
constexpr int MAX_PAGES = 1 << 25; // of a layer: page * PAGE + row is an int (256 GiB of one int8 kv head of 64)

// One layer of a cache.  K [page][kv head][PAGE][hd] and V [page][kv
// head][hd][PAGE]: a V column's rows are contiguous, so that both products of
// the attention take their operands from memory in 16-byte pieces as they lie.
// Scales [page][kv head][PAGE], int8 only.
struct KvLayer {
	uint8_t *k = nullptr, *v = nullptr;
	float *ks = nullptr, *vs = nullptr;
	int n_pages = 0, kvh = 0, hd = 0, i8 = 0;
	// bytes (and scales) of a layer: the kernels of several layers step by them
	size_t layer_bytes = 0, layer_scales = 0;
};

// The sequences of a call: device arrays, read by the kernels only after the
// bounds checks below.
struct KvSeqs {
	const int32_t *pages = nullptr; // [n_seqs][max_pages]
	const int32_t *len = nullptr;   // [n_seqs]
	const int32_t *first = nullptr; // [n_seqs + 1], or null: a token each
	int n_seqs = 0, max_pages = 0, n_tokens = 0;
};

// The scratch memory of the attention and verification calls begins with this
// many counters, which every call finds at 0 and leaves at 0 (the rest of it a
// call may find as it likes).
constexpr int WORK_COUNTERS = 8192;

struct AppendArgs {
	const float *q, *k, *v;
	size_t q_stride, k_stride, v_stride; // floats from a token's row to the next
	float *q_out;
	size_t qo_stride;
	const float *q_norm, *k_norm; // [hd], or null: no norm
	const int32_t *pos;           // [n_tokens], or null: the cache row
	int n_heads;
	double eps, log2_theta;
	// several axes: pos [axes][n_tokens], and two bits for each pair of a head that name its axis
	int axes = 1;
	uint64_t axis[2] = {0, 0};
};

struct AttnArgs {
	const float *q = nullptr;
	size_t q_stride = 0;
	float *out = nullptr;
	size_t o_stride = 0;
	const uint64_t *mask = nullptr; // [n_tokens][mask_words], or null: causal
	int mask_words = 0, n_heads = 0;
	float scale = 0.0f;
	// a window: rows below `sinks`, and above the row that the token stands at less `window`
	int window = 0, sinks = 0;
	const int32_t *at = nullptr; // [n_tokens], or null: the token's own row
};

hipError_t launch_kv_append(const KvLayer &c, const KvSeqs &s, const AppendArgs &a, hipStream_t st);
hipError_t launch_kv_read(const KvLayer &c, int n_layers, const KvSeqs &s, float *k_out, float *v_out, hipStream_t st);
hipError_t launch_kv_keep(const KvLayer &c, int n_layers, const KvSeqs &s, const int32_t *path, int max_path,
			  const int32_t *n_keep, int32_t *len_out, hipStream_t st);
// (a.window 0: none)
size_t attention_work_bytes(const KvLayer &c, const KvSeqs &s, const AttnArgs &a);
hipError_t launch_attention(const KvLayer &c, const KvSeqs &s, const AttnArgs &a, void *work, hipStream_t st);

struct VerifyArgs {
	const float *logits, *draft; // draft null: proposed without probabilities
	size_t l_stride, d_stride;
	const int32_t *first, *tokens, *parent;
	const float *u_accept, *u_sample;
	int vocab, n_seqs, n_tokens, max_children, max_path;
	float temperature;
	int32_t *path, *n_keep, *next;
};
constexpr int VERIFY_KIDS = 16; // children of a node that are tried, at most
size_t verify_work_bytes(const VerifyArgs &a, bool with_draft);
hipError_t launch_verify(const VerifyArgs &a, void *work, hipStream_t st);

// The pages of a step (plan.hip).
struct PlanArgs {
	const int32_t *pages, *len, *n_new; // [n_seqs][max_pages], [n_seqs], [n_seqs]
	int32_t *pages_out;                 // may be pages
	int32_t *ring;                      // [n_pages]
	const int32_t *state;               // [2]
	int32_t *state_out;                 // may be state
	int n_pages, n_seqs, max_pages, n_tokens, window, sinks;
	int32_t *first;      // [n_seqs + 1]
	int32_t *pos, *slot; // [n_tokens], or null
};
size_t plan_work_bytes(int n_seqs);
hipError_t launch_plan(const PlanArgs &a, void *work, hipStream_t st);

// Log-probabilities of tokens (logprobs.hip).
struct LogprobArgs {
	const float *logits;
	size_t stride;
	int vocab, n_rows, n_top;
	const int32_t *tokens; // [n_rows], or null
	double rate, inv; // log2 e / temperature, 1 / temperature
	float *logprob, *entropy; // [n_rows], or null
	int32_t *rank;            // [n_rows], or null
	int32_t *top_tokens;      // [n_rows][n_top]
	float *top_logprobs;      // [n_rows][n_top]
};
constexpr int LOGPROB_TOP = 64; // alternatives, at most
size_t logprobs_work_bytes(int vocab, int n_rows, int n_top);
hipError_t launch_logprobs(const LogprobArgs &a, void *work, hipStream_t st);

#if defined(__HIPCC__)
// x moved across lanes by a DPP control; lanes that get nothing: `none`
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp(float none, float x)
{
	return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, x), CTRL,
								     ROWS, 0xf, false));
}
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp(double none, double x)
{
	const uint64_t n = (uint64_t)__double_as_longlong(none), v = (uint64_t)__double_as_longlong(x);
	const uint32_t lo = __builtin_amdgcn_update_dpp((int)(uint32_t)n, (int)(uint32_t)v, CTRL, ROWS, 0xf, false),
		       hi = __builtin_amdgcn_update_dpp((int)(n >> 32), (int)(v >> 32), CTRL, ROWS, 0xf, false);
	return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// x of a lane (the same in all lanes), whether it is active here or not
__device__ __forceinline__ double of_lane(double x, int lane)
{
	const uint64_t v = (uint64_t)__double_as_longlong(x);
	const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
	return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// The running sum, or maximum, over groups of L = 64 or 32 lanes (a group's last
// lane has the whole), in registers: within rows of 16 by shifts, then the rows'
// ends into the rows behind.
template <int L> __device__ __forceinline__ double running_of(double x)
{
	x = x + dpp<0x111, 0xf>(0.0, x);
	x = x + dpp<0x112, 0xf>(0.0, x);
	x = x + dpp<0x114, 0xf>(0.0, x);
	x = x + dpp<0x118, 0xf>(0.0, x);
	x = x + dpp<0x142, 0xa>(0.0, x);
	return L == 64 ? x + dpp<0x143, 0xc>(0.0, x) : x;
}
template <int L> __device__ __forceinline__ float running_max_of(float x)
{
	const float none = -__builtin_inff();
	x = __builtin_fmaxf(x, dpp<0x111, 0xf>(none, x));
	x = __builtin_fmaxf(x, dpp<0x112, 0xf>(none, x));
	x = __builtin_fmaxf(x, dpp<0x114, 0xf>(none, x));
	x = __builtin_fmaxf(x, dpp<0x118, 0xf>(none, x));
	x = __builtin_fmaxf(x, dpp<0x142, 0xa>(none, x));
	return L == 64 ? __builtin_fmaxf(x, dpp<0x143, 0xc>(none, x)) : x;
}

__device__ __forceinline__ double wave_total(double x)
{
	return of_lane(running_of<64>(x), 63);
}

__device__ __forceinline__ float wave_max(float x)
{
	return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, running_max_of<64>(x)), 63));
}

// The token rows of sequence b: [t0, t0 + n), n = 0 where the arrays say
// something that lies outside the call's own sizes.
__device__ __forceinline__ void seq_tokens(const KvSeqs &s, int b, int &t0, int &n)
{
	t0 = b;
	n = 1;
	if (s.first) {
		t0 = s.first[b];
		const int t1 = s.first[b + 1];
		n = t0 >= 0 && t1 >= t0 && t1 <= s.n_tokens ? t1 - t0 : 0;
	}
}

// Whether sequence b's rows, n of them behind the committed ones, lie within
// its page table.
__device__ __forceinline__ bool seq_fits(const KvSeqs &s, int len, int n)
{
	return len >= 0 && (long long)len + n <= (long long)s.max_pages * PAGE;
}

// The page of row `row` of sequence b, -1 where the table names none.
__device__ __forceinline__ int page_of(const KvSeqs &s, int n_pages, int b, int row)
{
	const int p = s.pages[(size_t)b * s.max_pages + row / PAGE];
	return p >= 0 && p < n_pages ? p : -1;
}

// The sequence of token row t (the last b with first[b] <= t), -1 when none
// holds it.  A wave: the ranges a lane each, after bisection down to 64 of them.
__device__ __forceinline__ int seq_of_token(const KvSeqs &s, int t, int &t0, int &n)
{
	if (!s.first) {
		t0 = t;
		n = 1;
		return t < s.n_seqs ? t : -1;
	}
	int lo = 0, hi = s.n_seqs;
	while (hi - lo > 64) {
		const int mid = (lo + hi) >> 1;
		if (s.first[mid] <= t)
			lo = mid;
		else
			hi = mid;
	}
	const int b = lo + (int)(threadIdx.x & 63);
	const int from = b < hi ? s.first[b] : 0x7fffffff, to = b < hi ? s.first[b + 1] : 0;
	const unsigned long long below = __ballot(from <= t);
	if (!below)
		return -1;
	const int l = 63 - __builtin_clzll(below), t1 = __builtin_amdgcn_readlane(to, l);
	t0 = __builtin_amdgcn_readlane(from, l);
	n = t1 - t0;
	return t0 >= 0 && t < t1 && t1 <= s.n_tokens ? lo + l : -1;
}
#endif

} // namespace tie
