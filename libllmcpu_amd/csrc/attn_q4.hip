// Split-K attention over the 4-bit cache (kv_q4.h): decode and session batches,
// and every batch in exact mode.
//
// S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_f16, the keys' values as
// the format defines them (fp16, exact), Q and P as fp16 hi + lo: 22 significant
// bits, so scores and outputs have the error of fp32 sums. A product's 16
// columns are 8 (token, query head) pairs, their hi parts in columns 0 .. 7 and
// their lo parts in columns 8 .. 15; one rotation by half a row adds the two.
// Every pair goes through the same instructions in whatever column and batch it
// lies, and a group of keys outside its span changes nothing in it (weights
// exactly 0, factors exactly 1), so a token's bits depend on its own split grid
// alone.
//
// A work-group of four wavefronts owns one KV head, one range of keys and T
// tiles of 8 pairs; its wavefronts take groups of 32 keys in turn
// (record by record, straight into operand registers), keep running maxima and
// sums of their own, and meet in LDS at the end.
//
// Bound: HBM for long spans (five bits an element, K and V once: 32 768 keys of 8 x
// 128, 42 MB, 10.5 us a call of three streams; 131 072 of 8 x 64, 84 MB, 17.7:
// 4.0 and 4.7 TB/s, a large copy's rate is 4.76), beside the VALU work that makes
// fp16 of the codes (13 operations for eight); the launch and its chain of loads,
// softmax and merge for short ones (1024 keys of one head of 256: 9.8 us alone,
// 5.0 in flight, of which the host's call is 4.1).
#include "kernels.h"
#include "kv_q4.h"

namespace nnchip
{
	namespace
	{
		constexpr int kW = kQ4Waves;
		// A pair's weights are 2^(score - offset). The offset is raised, to kBelow
		// under the largest score so far, when a score passes it by more than kRaise:
		// weights stay under 2^kRaise (fp16 holds them) and a pair's largest weight is
		// at least 2^kBelow, so the steps of fp16's lo part (2^-25 at the least) are
		// 2^-31 of it.
		constexpr float kRaise = 14.0f, kBelow = 6.0f;

		__device__ __forceinline__ float ror8(float x)
		{
			return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false));
		}
		__device__ __forceinline__ float max_other_row(float x)
		{
			const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
			return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
		}
		__device__ __forceinline__ float row_max(float x) // over 16 lanes
		{
			x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xf, 0xf, false)));
			x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xf, 0xf, false)));
			x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xf, 0xf, false)));
			return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xf, 0xf, false)));
		}
		// Over the four lanes of a column.
		__device__ __forceinline__ float column_max(float x) { return max_with_other_half(max_other_row(x)); }
		__device__ __forceinline__ float column_sum(float x) { return add_with_other_half(add_with_other_row(x)); }

		// One record's registers: 32 rows, 32 columns of K and V.
		struct record
		{
			u32x4 code;
			u32x2 ksz;
			u32x4 vs, vz;
		};

		__device__ __forceinline__ record load_record(const unsigned char* rec, int lane)
		{
			record r;
			r.code = load_stream(rec + 16 * lane);
			r.ksz = *reinterpret_cast<const u32x2*>(rec + kQ4KScales + 8 * (lane & 15));
			r.vs = *reinterpret_cast<const u32x4*>(rec + kQ4VScales + 32 * (lane >> 4));
			r.vz = *reinterpret_cast<const u32x4*>(rec + kQ4VScales + 32 * (lane >> 4) + 16);
			return r;
		}

		// hi (is_lo false) or lo part of two weights.
		__device__ __forceinline__ uint32_t part_of(float a, float b, bool is_lo)
		{
			const f16x2 h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
			const f16x2 l = {static_cast<_Float16>(a - static_cast<float>(h.x)), static_cast<_Float16>(b - static_cast<float>(h.y))};
			return as_u32(is_lo ? l : h);
		}

		// From the largest magnitude of a pair's q: the power of two (with the scale's
		// sign: a masked score must stay the least) that brings it under 2^15, and
		// what its scores are multiplied with afterwards. 0, infinity and NaN stay as
		// they are.
		__device__ __forceinline__ void q_scale(float qscale, float m, float& back, float& up)
		{
			int e = m > 0.0f && m < INFINITY ? 14 - ilogbf(m) : 0;
			e = e < 126 ? e : 126;
			back = fmaxf(ldexpf(fabsf(qscale), -e), 1.17549435e-38f);
			up = ldexpf(qscale < 0.0f ? -1.0f : 1.0f, e);
		}

		__device__ __forceinline__ void add_scaled(float4& acc, const float4& v, float w)
		{
			acc.x = fmaf(v.x, w, acc.x);
			acc.y = fmaf(v.y, w, acc.y);
			acc.z = fmaf(v.z, w, acc.z);
			acc.w = fmaf(v.w, w, acc.w);
		}

		// Four outputs at element `at`: sums over their weights' sum.
		__device__ __forceinline__ void write_out(const decode_params& p, size_t at, const float4& acc, float sum)
		{
			const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
			float4 y = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
			if (p.gate) y = float4{gated(y.x, p.gate, at), gated(y.y, p.gate, at + 1), gated(y.z, p.gate, at + 2), gated(y.w, p.gate, at + 3)};
			*reinterpret_cast<float4*>(p.out + at) = y;
		}

		// What the wavefronts (classes) of a work-group add up to, in their order.
		struct joined
		{
			float m = -INFINITY, l = 0.0f;
			float4 o = {0, 0, 0, 0};
			__device__ __forceinline__ void factors(float mv, float& fa, float& fb)
			{
				const float now = fmaxf(m, mv), at = now == -INFINITY ? 0.0f : now;
				fa = fast_exp2(m - at);
				fb = fast_exp2(mv - at);
				m = now;
			}
			__device__ __forceinline__ void add(float mv, float lv, const float4& v)
			{
				float fa, fb;
				factors(mv, fa, fb);
				l = fmaf(lv, fb, l * fa);
				o = join4(o, fa, v, fb);
			}
			static __device__ __forceinline__ float4 join4(const float4& a, float fa, const float4& b, float fb)
			{
				return float4{fmaf(b.x, fb, a.x * fa), fmaf(b.y, fb, a.y * fa), fmaf(b.z, fb, a.z * fa), fmaf(b.w, fb, a.w * fa)};
			}
		};

		// Elements d .. d + 3 of a pair's result over the split: its partial, or with
		// one split the output.
		template <int HD>
		__device__ __forceinline__ void write_pair(const decode_params& p, int tok, int kvh, int h, int group, int split, int d,
		                                           const float4& o, float m, float l)
		{
			if (p.n_split > 1)
			{
				float* dst = p.part + (((static_cast<size_t>(tok) * p.n_kv + kvh) * p.n_split + split) * group + h) * (HD + 4);
				*reinterpret_cast<float4*>(dst + d) = o;
				if (d == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(m, l);
			}
			else
				write_out(p, (static_cast<size_t>(tok) * p.n_head + kvh * group + h) * HD + d, o, l);
		}

		// The ordered merge of a pair's splits: M = the largest offset; o and l
		// relative to it, summed over the splits of a slice in ascending order, then
		// over the slices in order. Split s (its absolute number: keys / split_keys)
		// belongs to slice s % merge_slices, so a batch whose first split lies before a
		// token's own gives the token the same sums (those splits add exact zeros).
		constexpr int kMergeThreads = 256, kMergeAhead = 8;
		static_assert(kDecodeMaxSplits == kMergeThreads, "a thread per split");
		__host__ __device__ constexpr int merge_slices(int hd) { return kMergeThreads / (hd / 4); }

		// By 256 threads per pair: every split's offset in one load per thread, outputs
		// in float4 columns times slices.
		__global__ __launch_bounds__(kMergeThreads) void merge_q4_kernel(const decode_params p, int hd, int group)
		{
			__shared__ float s_f[kDecodeMaxSplits], s_lf[kDecodeMaxSplits];
			__shared__ float s_red[kMergeThreads / 64];
			__shared__ float s_l[kMergeThreads];
			__shared__ float4 s_o[kMergeThreads];
			const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
			const int qh = blockIdx.x, tok = blockIdx.y, kvh = qh / group, h = qh % group;
			const int ns = p.n_split, cols = hd / 4, n_slices = merge_slices(hd);
			const int c = tid % cols, slice = tid / cols;
			const int base = p.split_base / p.split_keys; // the first split's number
			const int s0 = n_slices - 1 - (base + n_slices - 1 - slice) % n_slices; // the slice's first split
			const float* part = p.part + ((static_cast<size_t>(tok) * p.n_kv + kvh) * ns * group + h) * (hd + 4);
			const size_t step = static_cast<size_t>(group) * (hd + 4);

			float2 ml = make_float2(-INFINITY, 0.0f);
			if (tid < ns) ml = *reinterpret_cast<const float2*>(part + tid * step + hd);
			float4 o[kMergeAhead]; // the slice's first splits, on their way meanwhile
#pragma unroll
			for (int i = 0; i < kMergeAhead; ++i)
			{
				const int s = s0 + i * n_slices;
				o[i] = float4{0, 0, 0, 0};
				if (slice < n_slices && s < ns) o[i] = *reinterpret_cast<const float4*>(part + s * step + 4 * c);
			}
			float mx = max_with_other_half(max_other_row(row_max(ml.x)));
			if (lane == 0) s_red[wave] = mx;
			__syncthreads();
			mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
			const float f = fast_exp2(ml.x - (mx == -INFINITY ? 0.0f : mx));
			s_f[tid] = f;
			s_lf[tid] = ml.y;
			__syncthreads();
			float4 acc = {0, 0, 0, 0};
			float l = 0.0f;
			if (slice < n_slices)
			{
#pragma unroll
				for (int i = 0; i < kMergeAhead; ++i)
				{
					const int s = s0 + i * n_slices;
					if (s >= ns) continue;
					add_scaled(acc, o[i], s_f[s]);
					l = fmaf(s_lf[s], s_f[s], l);
				}
				for (int s = s0 + kMergeAhead * n_slices; s < ns; s += n_slices)
				{
					add_scaled(acc, *reinterpret_cast<const float4*>(part + s * step + 4 * c), s_f[s]);
					l = fmaf(s_lf[s], s_f[s], l);
				}
			}
			s_o[tid] = acc;
			s_l[tid] = l;
			__syncthreads();
			if (tid >= cols) return;
			acc = float4{0, 0, 0, 0};
			l = 0.0f;
			for (int i = 0; i < n_slices; ++i)
			{
				add_scaled(acc, s_o[i * cols + tid], 1.0f);
				l += s_l[i * cols + tid];
			}
			write_out(p, (static_cast<size_t>(tok) * p.n_head + qh) * hd + 4 * tid, acc, l);
		}

		// The same within the split launch, for one token's pairs and at most
		// kFuseSplits splits: a work-group's partial is stored with device scope (sc1:
		// through its XCD's L2, acknowledged once every XCD can see it), then the
		// work-group counts itself in; the last of its KV head to do so resets the
		// count and merges, a float4 column of a pair per thread, every split's loads
		// at once and with device scope.
		constexpr int kAuxDevice = 16, kFuseSplits = 8;
		__device__ __forceinline__ __amdgpu_buffer_rsrc_t head_partials(const decode_params& p, int kvh, int group, int hd)
		{
			const size_t floats = static_cast<size_t>(p.n_split) * group * (hd + 4);
			return __builtin_amdgcn_make_buffer_rsrc(p.part + kvh * floats, 0, static_cast<int>(floats * 4), 0x00020000);
		}
		__device__ __forceinline__ void store_device(__amdgpu_buffer_rsrc_t r, int at, const float4& v)
		{
			__builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, 4 * at, 0, kAuxDevice);
		}
		template <int HD>
		__device__ __forceinline__ void merge_last(const decode_params& p, int kvh, int group)
		{
			constexpr int COLS = HD / 4, SLICES = merge_slices(HD), CLASSES = SLICES < kFuseSplits ? SLICES : kFuseSplits;
			const auto rs = head_partials(p, kvh, group, HD);
			const int base = p.split_base / p.split_keys, ns = p.n_split;
			for (int x = threadIdx.x; x < group * COLS; x += 64 * kW)
			{
				const int h = x / COLS, c = x % COLS;
				float4 o[kFuseSplits];
				float2 ml[kFuseSplits];
#pragma unroll
				for (int s = 0; s < kFuseSplits; ++s) // (past the last split: past the descriptor, zeros)
				{
					const int at = 4 * (s * group + h) * (HD + 4);
					o[s] = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(rs, at + 16 * c, 0, kAuxDevice));
					ml[s] = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(rs, at + 4 * HD, 0, kAuxDevice));
				}
				float mx = -INFINITY;
#pragma unroll
				for (int s = 0; s < kFuseSplits; ++s)
				{
					if (s >= ns) ml[s].x = -INFINITY;
					mx = fmaxf(mx, ml[s].x);
				}
				const float off = mx == -INFINITY ? 0.0f : mx;
				// Class k: splits k, k + SLICES, ..., which are slice (base + k) % SLICES.
				float4 part[CLASSES];
				float l[CLASSES];
#pragma unroll
				for (int k = 0; k < CLASSES; ++k)
				{
					part[k] = float4{0, 0, 0, 0};
					l[k] = 0.0f;
#pragma unroll
					for (int s = k; s < kFuseSplits; s += SLICES)
					{
						if (s >= ns) continue;
						const float f = fast_exp2(ml[s].x - off);
						add_scaled(part[k], o[s], f);
						l[k] = fmaf(ml[s].y, f, l[k]);
					}
				}
				// The slices in order: from the class of slice 0 on, then the classes
				// before it.
				const int c0 = (SLICES - base % SLICES) % SLICES;
				float4 acc = {0, 0, 0, 0};
				float sum = 0.0f;
#pragma unroll
				for (int pass = 0; pass < 2; ++pass)
#pragma unroll
					for (int k = 0; k < CLASSES; ++k)
						if ((k >= c0) == (pass == 0))
						{
							add_scaled(acc, part[k], 1.0f);
							sum += l[k];
						}
				write_out(p, static_cast<size_t>(kvh * group + h) * HD + 4 * c, acc, sum);
			}
		}

		// Two wavefronts per SIMD where their registers fit (256 each).
		constexpr int q4_per_simd(int nb) { return nb <= 4 ? 2 : 1; }

		template <int NB, int T, bool FUSE>
		__global__ __launch_bounds__(64 * kW, q4_per_simd(NB)) void decode_q4_kernel(
			const decode_params p, int group)
		{
			constexpr int HD = NB * kQ4Block;
			const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
			const int split = blockIdx.x, kvh = blockIdx.y;
			const int c8 = lane & 7, g = lane >> 4;
			const bool is_lo = (lane & 8) != 0;
			const int n_pairs = p.n_tok * group;

			__shared__ float s_o[kW][8][HD + 4]; // a tile's outputs (relative to its offset), offset, sum

			// The keys any pair of the launch attends to, within the split.
			int kmin, kmax, unused;
			attn_span(p.causal, p.window, p.pos0, p.n_seq, kmin, unused);
			attn_span(p.causal, p.window, p.pos0 + p.n_tok - 1, p.n_seq, unused, kmax);
			const int k0 = p.split_base + split * p.split_keys;
			const int g_first = (kmin > k0 ? kmin : k0) / kQ4Rows;
			const int g_last = (kmax < k0 + p.split_keys - 1 ? kmax : k0 + p.split_keys - 1) / kQ4Rows;
			const int row_groups = p.rows / kQ4Rows, blocks = p.kv_dim / kQ4Block;
			const unsigned char* recs = static_cast<const unsigned char*>(p.K) + static_cast<size_t>(kvh) * NB * kQ4Record;
			const size_t group_bytes = static_cast<size_t>(blocks) * kQ4Record;
			// (wavefront w takes the groups whose number in the split is w modulo kW)
			int kg = k0 / kQ4Rows + wave;
			if (kg < g_first) kg += (g_first - kg + kW - 1) / kW * kW;

			// Records in flight: kDepth - 1 groups ahead of the one worked on. (At 16
			// blocks a group's registers do not fit twice.)
			constexpr int kDepth = NB <= 4 && T == 1 ? 3 : NB <= 8 ? 2 : 1;
			int row_group = kg % row_groups; // of the group loaded next
			const int hop = kW % row_groups;
			record r[kDepth][NB];
			auto load_next = [&](record* to)
			{
				const unsigned char* at = recs + static_cast<size_t>(row_group) * group_bytes;
#pragma unroll
				for (int b = 0; b < NB; ++b) to[b] = load_record(at + b * kQ4Record, lane);
				row_group += hop;
				if (row_group >= row_groups) row_group -= row_groups;
			};
#pragma unroll
			for (int i = 0; i + 1 < kDepth; ++i)
				if (kg + i * kW <= g_last) load_next(r[i]);

			// Q: per pair brought under 2^15 by a power of two, then fp16 hi or lo.
			f16x8 q[T][NB];
			float back[T];
			int first[T], last[T];
#pragma unroll
			for (int i = 0; i < T; ++i)
			{
				const int pair = (blockIdx.z * T + i) * 8 + c8;
				const bool real = pair < n_pairs;
				const int tok = real ? pair / group : 0, h = real ? pair % group : 0;
				attn_span(p.causal, p.window, p.pos0 + tok, p.n_seq, first[i], last[i]);
				if (!real) last[i] = -1, first[i] = 0;
				const float* src = p.q + (static_cast<size_t>(tok) * p.n_head + kvh * group + h) * HD + 8 * g;
				float x[NB][8];
				float m = 0.0f;
#pragma unroll
				for (int b = 0; b < NB; ++b)
				{
					const float4 u = *reinterpret_cast<const float4*>(src + 32 * b), v = *reinterpret_cast<const float4*>(src + 32 * b + 4);
					// k slot order: columns 0, 4, 1, 5, 2, 6, 3, 7
					x[b][0] = u.x, x[b][1] = v.x, x[b][2] = u.y, x[b][3] = v.y;
					x[b][4] = u.z, x[b][5] = v.z, x[b][6] = u.w, x[b][7] = v.w;
#pragma unroll
					for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[b][j]));
				}
				m = column_max(m);
				float up;
				q_scale(p.qscale, m, back[i], up);
#pragma unroll
				for (int b = 0; b < NB; ++b)
				{
					u32x4 w;
#pragma unroll
					for (int j = 0; j < 4; ++j) w[j] = part_of(x[b][2 * j] * up, x[b][2 * j + 1] * up, is_lo);
					q[i][b] = as_f16x8(w);
				}
			}

			f32x4 o[T][NB][2] = {};
			float m_off[T], l[T];
#pragma unroll
			for (int i = 0; i < T; ++i) m_off[i] = -INFINITY, l[i] = 0.0f;

			// Every pair of tile i sees the keys full_from[i] .. full_to[i].
			int full_from[T], full_to[T];
#pragma unroll
			for (int i = 0; i < T; ++i)
			{
				const int a = (blockIdx.z * T + i) * 8, z = a + 7 < n_pairs ? a + 7 : n_pairs - 1;
				attn_span(p.causal, p.window, p.pos0 + z / group, p.n_seq, full_from[i], unused);
				attn_span(p.causal, p.window, p.pos0 + (a < n_pairs ? a : 0) / group, p.n_seq, unused, full_to[i]);
			}
			const q4_masks masks;
			auto work = [&](const record* r)
			{
				f32x4 s[T][2] = {};
#pragma unroll
				for (int b = 0; b < NB; ++b)
#pragma unroll
					for (int t = 0; t < 2; ++t)
					{
						const f16x8 a = q4_k(t ? r[b].code.y : r[b].code.x, t ? r[b].ksz.y : r[b].ksz.x, masks);
#pragma unroll
						for (int i = 0; i < T; ++i) s[i][t] = mfma16x16x32(a, q[i][b], s[i][t]);
					}

				f16x8 w[T];
#pragma unroll
				for (int i = 0; i < T; ++i)
				{
					float sc[8]; // tile t, row j: 4 t + j; key 32 kg + 16 t + 4 g + j
#pragma unroll
					for (int j = 0; j < 8; ++j)
					{
						const float d = s[i][j >> 2][j & 3];
						sc[j] = d + ror8(d);
					}
					if (kg * kQ4Rows < full_from[i] || kg * kQ4Rows + kQ4Rows - 1 > full_to[i])
					{
						asm volatile(""); // (a branch: most groups lie within every span)
#pragma unroll
						for (int j = 0; j < 8; ++j)
						{
							const int key = kg * kQ4Rows + 16 * (j >> 2) + 4 * g + (j & 3);
							if (key < first[i] || key > last[i]) sc[j] = -INFINITY;
						}
					}
					float m = sc[0];
#pragma unroll
					for (int j = 1; j < 8; ++j) m = fmaxf(m, sc[j]);
					m = column_max(m) * back[i];
					const bool up = m > m_off[i] + kRaise; // (the first keys of a span too: from -inf)
					if (__any(up))
					{
						const float now = up ? m - kBelow : m_off[i];
						const float f = up ? fast_exp2(m_off[i] - now) : 1.0f;
						if (!__all(m_off[i] == -INFINITY)) // (else nothing has been added yet)
						{
							l[i] *= f;
#pragma unroll
							for (int b = 0; b < NB; ++b) o[i][b][0] *= f, o[i][b][1] *= f;
						}
						m_off[i] = now;
					}
					const float off = m_off[i] == -INFINITY ? 0.0f : m_off[i];
#pragma unroll
					for (int j = 0; j < 8; ++j)
					{
						sc[j] = fast_exp2(fmaf(sc[j], back[i], -off));
						l[i] += sc[j];
					}
					u32x4 f;
#pragma unroll
					for (int j = 0; j < 4; ++j) f[j] = part_of(sc[j], sc[4 + j], is_lo);
					w[i] = as_f16x8(f);
				}

#pragma unroll
				for (int b = 0; b < NB; ++b)
#pragma unroll
					for (int t = 0; t < 2; ++t)
					{
						const f16x8 a = q4_v(t ? r[b].code.w : r[b].code.z, r[b].vs, r[b].vz, masks);
#pragma unroll
						for (int i = 0; i < T; ++i) o[i][b][t] = mfma16x16x32(a, w[i], o[i][b][t]);
					}
			};
			for (; kg <= g_last;)
			{
#pragma unroll
				for (int i = 0; i < kDepth; ++i)
				{
					if (kg > g_last) break;
					if (kDepth == 1 || kg + (kDepth - 1) * kW <= g_last) load_next(r[(i + kDepth - 1) % kDepth]);
					work(r[i]);
					kg += kW;
				}
			}

			// The wavefronts' parts of each tile, joined in wavefront order.
#pragma unroll
			for (int i = 0; i < T; ++i)
			{
				if (i) __syncthreads();
				l[i] = column_sum(l[i]);
#pragma unroll
				for (int b = 0; b < NB; ++b)
#pragma unroll
					for (int t = 0; t < 2; ++t)
					{
						float4 v;
						v.x = o[i][b][t][0] + ror8(o[i][b][t][0]);
						v.y = o[i][b][t][1] + ror8(o[i][b][t][1]);
						v.z = o[i][b][t][2] + ror8(o[i][b][t][2]);
						v.w = o[i][b][t][3] + ror8(o[i][b][t][3]);
						if (!is_lo) *reinterpret_cast<float4*>(&s_o[wave][c8][32 * b + 16 * t + 4 * g]) = v;
					}
				if (lane < 8) s_o[wave][c8][HD] = m_off[i], s_o[wave][c8][HD + 1] = l[i];
				__syncthreads();
				const int pair0 = (blockIdx.z * T + i) * 8;
				const int n_here = n_pairs - pair0 < 8 ? n_pairs - pair0 : 8;
				for (int x = threadIdx.x; x < n_here * (HD / 4); x += 64 * kW) // a float4 of a pair
				{
					const int c = x / (HD / 4), d = 4 * (x % (HD / 4)), pair = pair0 + c;
					const int tok = p.n_tok == 1 ? 0 : pair / group, h = pair - tok * group;
					joined y;
#pragma unroll
					for (int v = 0; v < kW; ++v)
						y.add(s_o[v][c][HD], s_o[v][c][HD + 1], *reinterpret_cast<const float4*>(&s_o[v][c][d]));
					if constexpr (FUSE)
					{
						const auto rs = head_partials(p, kvh, group, HD);
						const int at = (split * group + h) * (HD + 4);
						store_device(rs, at + d, y.o);
						if (d == 0) store_device(rs, at + HD, float4{y.m, y.l, 0, 0});
					}
					else
						write_pair<HD>(p, tok, kvh, h, group, split, d, y.o, y.m, y.l);
				}
			}
			if constexpr (FUSE)
			{
				__shared__ int s_last;
				asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the thread's stores are seen everywhere
				__syncthreads();
				if (threadIdx.x == 0)
				{
					unsigned* count = p.counts + kvh;
					const bool is_last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
					                     static_cast<unsigned>(p.n_split - 1);
					if (is_last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
					s_last = is_last;
				}
				__syncthreads();
				if (!s_last) return;
				merge_last<HD>(p, kvh, group);
			}
		}

		// Many pairs (session batches, exact mode): a wavefront takes 16 pairs, one per
		// column, their hi and lo parts in products of their own, and the work-group's
		// four wavefronts share every value: each turns a quarter of a group's words
		// into operands in LDS while they compute on the group before. The classes
		// that decode_q4_kernel's wavefronts are (groups by their number in the split
		// modulo kW) follow one another, with sums of their own, and join in the same
		// order, so a pair gets the same bits. Bound: VALU (the softmax of 16 pairs in
		// fp16 parts, and every class's sums joined: some 300 operations per group of 32
		// keys; matrix units 18 % busy) and the partials, written and read as many bytes as
		// the records. (13 tokens of 32 over 8 x 128 at 20k keys: 20.9 us a call; with the kernel
		// above, two tiles of 8 pairs per wavefront, every tile's weights computed twice
		// and every value made four times, 68.)
		template <int NB>
		__global__ __launch_bounds__(64 * kW, NB <= 4 ? 2 : 1) void decode_q4_multi_kernel(const decode_params p, int group)
		{
			constexpr int HD = NB * kQ4Block, OWN = (NB + 1) / 2, PER = NB <= 6 ? 2 : 1; // groups at a time
			// Two buffers of PER groups: K and V of each block, two operands of 1 KB.
			__shared__ __align__(16) unsigned char s_op[2][PER][2][NB][2048];
			const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
			const int split = blockIdx.x, kvh = blockIdx.y;
			const int c = lane & 15, g = lane >> 4;
			const int n_pairs = p.n_tok * group, pair0 = blockIdx.z * (16 * kW), mine0 = pair0 + 16 * wave;
			const bool any = mine0 < n_pairs, real = mine0 + c < n_pairs;
			const int pair = real ? mine0 + c : n_pairs - 1;
			const int tok = pair / group, h = pair - tok * group;
			int first, last, full_from, full_to, kmin, kmax, unused;
			attn_span(p.causal, p.window, p.pos0 + tok, p.n_seq, first, last);
			auto clamped = [&](int x) { return (x < n_pairs ? x : n_pairs - 1) / group; };
			attn_span(p.causal, p.window, p.pos0 + clamped(mine0 + 15), p.n_seq, full_from, unused);
			attn_span(p.causal, p.window, p.pos0 + clamped(mine0), p.n_seq, unused, full_to);
			attn_span(p.causal, p.window, p.pos0 + clamped(pair0), p.n_seq, kmin, unused);
			attn_span(p.causal, p.window, p.pos0 + clamped(pair0 + 16 * kW - 1), p.n_seq, unused, kmax);

			const int k0 = p.split_base + split * p.split_keys;
			const int g_base = k0 / kQ4Rows;
			const int g_first = (kmin > k0 ? kmin : k0) / kQ4Rows;
			const int g_last = (kmax < k0 + p.split_keys - 1 ? kmax : k0 + p.split_keys - 1) / kQ4Rows;
			const int row_groups = p.rows / kQ4Rows, blocks = p.kv_dim / kQ4Block;
			const unsigned char* recs = static_cast<const unsigned char*>(p.K) + static_cast<size_t>(kvh) * NB * kQ4Record;
			const size_t group_bytes = static_cast<size_t>(blocks) * kQ4Record;
			// The groups class by class.
			auto class_first = [&](int cls)
			{
				const int at = g_base + cls;
				return at >= g_first ? at : at + (g_first - at + kW - 1) / kW * kW;
			};
			struct place
			{
				int cls, kg;
			};
			auto next_of = [&](place x)
			{
				x.kg += kW;
				while (x.kg > g_last && x.cls < kW - 1) x.kg = class_first(++x.cls);
				if (x.kg > g_last) x.cls = kW;
				return x;
			};
			place at{0, class_first(0) - kW};
			at = next_of(at); // (cls kW: none)

			// Wavefronts 0 and 2 make K's operands, 1 and 3 V's, of every other block.
			const bool is_v = wave & 1;
			const int block0 = wave >> 1;
			struct unit_regs
			{
				u32x2 code[OWN], ksz[OWN];
				u32x4 s[OWN], z[OWN];
			};
			auto load = [&](const place& x, unit_regs& r)
			{
				if (x.cls >= kW) return;
				const unsigned char* rec = recs + static_cast<size_t>(x.kg % row_groups) * group_bytes + block0 * kQ4Record;
				if (is_v)
				{
#pragma unroll
					for (int n = 0; n < OWN; ++n)
						if (block0 + 2 * n < NB)
						{
							r.code[n] = *reinterpret_cast<const u32x2*>(rec + 2 * n * kQ4Record + 16 * lane + 8);
							r.s[n] = *reinterpret_cast<const u32x4*>(rec + 2 * n * kQ4Record + kQ4VScales + 32 * g);
							r.z[n] = *reinterpret_cast<const u32x4*>(rec + 2 * n * kQ4Record + kQ4VScales + 32 * g + 16);
						}
				}
				else
				{
#pragma unroll
					for (int n = 0; n < OWN; ++n)
						if (block0 + 2 * n < NB)
						{
							r.code[n] = *reinterpret_cast<const u32x2*>(rec + 2 * n * kQ4Record + 16 * lane);
							r.ksz[n] = *reinterpret_cast<const u32x2*>(rec + 2 * n * kQ4Record + kQ4KScales + 8 * c);
						}
				}
			};
			const q4_masks masks;
			auto convert = [&](const place& x, const unit_regs& r, int buf, int slot)
			{
				if (x.cls >= kW) return;
				if (is_v)
				{
#pragma unroll
					for (int n = 0; n < OWN; ++n)
						if (block0 + 2 * n < NB)
						{
							f16x8* to = reinterpret_cast<f16x8*>(&s_op[buf][slot][1][block0 + 2 * n][16 * lane]);
							to[0] = q4_v(r.code[n].x, r.s[n], r.z[n], masks);
							to[64] = q4_v(r.code[n].y, r.s[n], r.z[n], masks);
						}
				}
				else
				{
#pragma unroll
					for (int n = 0; n < OWN; ++n)
						if (block0 + 2 * n < NB)
						{
							f16x8* to = reinterpret_cast<f16x8*>(&s_op[buf][slot][0][block0 + 2 * n][16 * lane]);
							to[0] = q4_k(r.code[n].x, r.ksz[n].x, masks);
							to[64] = q4_k(r.code[n].y, r.ksz[n].y, masks);
						}
				}
			};
			// The groups PER at a time: now (in LDS), ahead (in registers).
			auto after = [&](const place& x) { return x.cls < kW ? next_of(x) : x; };
			place now[PER], ahead[PER];
			auto follow = [&](place x, place* to)
			{
#pragma unroll
				for (int i = 0; i < PER; ++i) to[i] = x = after(x);
			};
			unit_regs regs[PER];
			now[0] = at;
			if constexpr (PER == 2) now[1] = after(at);
#pragma unroll
			for (int i = 0; i < PER; ++i) load(now[i], regs[i]);

			// Q, as in decode_q4_kernel.
			f16x8 qh[NB], ql[NB];
			float back;
			{
				const float* src = p.q + (static_cast<size_t>(tok) * p.n_head + kvh * group + h) * HD + 8 * g;
				float x[NB][8], m = 0.0f;
#pragma unroll
				for (int b = 0; b < NB; ++b)
				{
					const float4 u = *reinterpret_cast<const float4*>(src + 32 * b), v = *reinterpret_cast<const float4*>(src + 32 * b + 4);
					x[b][0] = u.x, x[b][1] = v.x, x[b][2] = u.y, x[b][3] = v.y;
					x[b][4] = u.z, x[b][5] = v.z, x[b][6] = u.w, x[b][7] = v.w;
#pragma unroll
					for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[b][j]));
				}
				float up;
				q_scale(p.qscale, column_max(m), back, up);
#pragma unroll
				for (int b = 0; b < NB; ++b)
				{
					u32x4 hi, lo;
#pragma unroll
					for (int j = 0; j < 4; ++j)
					{
						hi[j] = part_of(x[b][2 * j] * up, x[b][2 * j + 1] * up, false);
						lo[j] = part_of(x[b][2 * j] * up, x[b][2 * j + 1] * up, true);
					}
					qh[b] = as_f16x8(hi);
					ql[b] = as_f16x8(lo);
				}
			}

			f32x4 acc[NB][2] = {}, oh[NB][2] = {}, ol[NB][2] = {};
			float m_all = -INFINITY, l_all = 0.0f, m_off = -INFINITY, l = 0.0f;
			follow(now[PER - 1], ahead);
#pragma unroll
			for (int i = 0; i < PER; ++i) convert(now[i], regs[i], 0, i);
#pragma unroll
			for (int i = 0; i < PER; ++i) load(ahead[i], regs[i]);
			__syncthreads();
			for (int buf = 0; now[0].cls < kW; buf ^= 1)
			{
#pragma unroll
				for (int i = 0; i < PER; ++i) convert(ahead[i], regs[i], buf ^ 1, i);
				place then[PER];
				follow(ahead[PER - 1], then);
#pragma unroll
				for (int i = 0; i < PER; ++i) load(then[i], regs[i]);
				if (any)
				{
					auto op = [&](int slot, int v, int b, int t) { return *reinterpret_cast<const f16x8*>(&s_op[buf][slot][v][b][1024 * t + 16 * lane]); };
					float sc[PER][8];
#pragma unroll
					for (int x = 0; x < PER; ++x)
					{
						if (now[x].cls >= kW) continue;
						f32x4 sh[2] = {}, sl[2] = {};
#pragma unroll
						for (int b = 0; b < NB; ++b)
#pragma unroll
							for (int t = 0; t < 2; ++t)
							{
								const f16x8 a = op(x, 0, b, t);
								sh[t] = mfma16x16x32(a, qh[b], sh[t]);
								sl[t] = mfma16x16x32(a, ql[b], sl[t]);
							}
#pragma unroll
						for (int j = 0; j < 8; ++j) sc[x][j] = sh[j >> 2][j & 3] + sl[j >> 2][j & 3];
					}
#pragma unroll
					for (int x = 0; x < PER; ++x)
					{
						if (now[x].cls >= kW) continue;
						const int key0 = now[x].kg * kQ4Rows;
						if (key0 < full_from || key0 + kQ4Rows - 1 > full_to)
						{
							asm volatile("");
#pragma unroll
							for (int j = 0; j < 8; ++j)
							{
								const int key = key0 + 16 * (j >> 2) + 4 * g + (j & 3);
								if (key < first || key > last) sc[x][j] = -INFINITY;
							}
						}
						float m = sc[x][0];
#pragma unroll
						for (int j = 1; j < 8; ++j) m = fmaxf(m, sc[x][j]);
						m = column_max(m) * back;
						const bool up = m > m_off + kRaise;
						if (__any(up))
						{
							const float to = up ? m - kBelow : m_off;
							const float f = up ? fast_exp2(m_off - to) : 1.0f;
							if (!__all(m_off == -INFINITY)) // (else nothing has been added yet)
							{
								l *= f;
#pragma unroll
								for (int b = 0; b < NB; ++b) oh[b][0] *= f, oh[b][1] *= f, ol[b][0] *= f, ol[b][1] *= f;
							}
							m_off = to;
						}
						const float off = m_off == -INFINITY ? 0.0f : m_off;
#pragma unroll
						for (int j = 0; j < 8; ++j)
						{
							sc[x][j] = fast_exp2(fmaf(sc[x][j], back, -off));
							l += sc[x][j];
						}
						u32x4 hi, lo;
#pragma unroll
						for (int j = 0; j < 4; ++j)
						{
							hi[j] = part_of(sc[x][j], sc[x][4 + j], false);
							lo[j] = part_of(sc[x][j], sc[x][4 + j], true);
						}
						const f16x8 wh = as_f16x8(hi), wl = as_f16x8(lo);
#pragma unroll
						for (int b = 0; b < NB; ++b)
#pragma unroll
							for (int t = 0; t < 2; ++t)
							{
								const f16x8 a = op(x, 1, b, t);
								oh[b][t] = mfma16x16x32(a, wh, oh[b][t]);
								ol[b][t] = mfma16x16x32(a, wl, ol[b][t]);
							}
						if ((x + 1 < PER ? now[(x + 1) % PER].cls : ahead[0].cls) != now[x].cls) // the class is done: it joins those before it
						{
							joined y;
							y.m = m_all;
							float fa, fb;
							y.factors(m_off, fa, fb);
							l_all = fmaf(column_sum(l), fb, l_all * fa);
							m_all = y.m;
							m_off = -INFINITY;
							l = 0.0f;
#pragma unroll
							for (int b = 0; b < NB; ++b)
#pragma unroll
								for (int t = 0; t < 2; ++t)
#pragma unroll
									for (int j = 0; j < 4; ++j)
									{
										acc[b][t][j] = fmaf(oh[b][t][j] + ol[b][t][j], fb, acc[b][t][j] * fa);
										oh[b][t][j] = ol[b][t][j] = 0.0f;
									}
						}
					}
				}
#pragma unroll
				for (int i = 0; i < PER; ++i) now[i] = ahead[i], ahead[i] = then[i];
				__syncthreads();
			}
			if (!real) return;
#pragma unroll
			for (int b = 0; b < NB; ++b)
#pragma unroll
				for (int t = 0; t < 2; ++t)
					write_pair<HD>(p, tok, kvh, h, group, split, 32 * b + 16 * t + 4 * g,
					               float4{acc[b][t][0], acc[b][t][1], acc[b][t][2], acc[b][t][3]}, m_all, l_all);
		}

		template <int NB>
		void launch_nb(const decode_params& p, int n_tok, int group, int n_cu, hipStream_t stream)
		{
			// Up to 8 pairs a wavefront takes them all; up to 16 two tiles of 8, from four
			// blocks on a work-group each (two tiles' registers leave one wavefront per SIMD
			// there: 4 tokens of 32 over 8 x 128 at 8k keys 21.1 us alone and 15.5 with three
			// streams, two work-groups 18.0 and 10.9; of 8 x 64 at 20k 15.0 and 7.6, two
			// work-groups 15.6 and 8.1). More pairs: a work-group per tile while all of them
			// are resident at once, else the kernel for many, which makes every value once
			// (alone / three streams, many -> a work-group per tile: 16 tokens of 4 over 1 x
			// 256 at 1k keys, 72 work-groups, 26.0 / 8.9 -> 11.5 / 7.1; 6 of 32 over 8 x 128
			// at 2k, 408, 13.3 / 7.1 -> 10.5 / 6.6; past them 16 of 4 over 1 x 256 at 8k, 504
			// at one wavefront per SIMD, 30 / 11.5 -> 24 / 17.8; 5 of 32 over 8 x 128 at 9k,
			// 864, 22.0 / 10.3 -> 18.8 / 11.8). Its registers do not fit at 16 blocks.
			const int pairs = n_tok * group, tiles = (pairs + 7) / 8;
			const bool tiled = pairs <= 8 || (NB > 3 && pairs <= 16) || NB > 8 ||
			                   (pairs > 16 && static_cast<long long>(p.n_split) * p.n_kv * tiles <= q4_per_simd(NB) * n_cu);
			const dim3 threads(64 * kW);
			if constexpr (NB <= 8)
				if (pairs > 16 && !tiled)
					decode_q4_multi_kernel<NB><<<dim3(p.n_split, p.n_kv, (pairs + 16 * kW - 1) / (16 * kW)), threads, 0, stream>>>(p, group);
			if constexpr (NB <= 3)
				if (pairs > 8 && pairs <= 16)
					decode_q4_kernel<NB, 2, false><<<dim3(p.n_split, p.n_kv, 1), threads, 0, stream>>>(p, group);
			if constexpr (NB <= 8)
				if (n_tok == 1 && pairs <= 8 && p.n_split > 1 && p.n_split <= kFuseSplits && p.counts)
				{
					decode_q4_kernel<NB, 1, true><<<dim3(p.n_split, p.n_kv, 1), threads, 0, stream>>>(p, group);
					return;
				}
			if (tiled)
				decode_q4_kernel<NB, 1, false><<<dim3(p.n_split, p.n_kv, tiles), threads, 0, stream>>>(p, group);
			if (p.n_split > 1)
				merge_q4_kernel<<<dim3(p.n_head, n_tok), kMergeThreads, 0, stream>>>(p, NB * kQ4Block, group);
		}
	}

	bool launch_decode_q4(const decode_params& p, int n_tok, int head_dim, int group, int n_cu, hipStream_t stream)
	{
		switch (head_dim)
		{
		case 32: launch_nb<1>(p, n_tok, group, n_cu, stream); return true;
		case 64: launch_nb<2>(p, n_tok, group, n_cu, stream); return true;
		case 96: launch_nb<3>(p, n_tok, group, n_cu, stream); return true;
		case 128: launch_nb<4>(p, n_tok, group, n_cu, stream); return true;
		case 192: launch_nb<6>(p, n_tok, group, n_cu, stream); return true;
		case 256: launch_nb<8>(p, n_tok, group, n_cu, stream); return true;
		case 512: launch_nb<16>(p, n_tok, group, n_cu, stream); return true;
		default: return false;
		}
	}
}
