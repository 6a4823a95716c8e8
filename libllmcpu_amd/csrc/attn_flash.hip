// Attention of many query rows over whole sequences on the matrix cores: packed
// prompts (BF16 or F32 q, k, v in device memory, several sequences end to end)
// and batches over the 4-bit cache (kv_q4.h).
//
// The rows of a KV head are (token, query head) pairs, token by token, so the
// heads that share its keys share every load. A work-group of RG x KG wavefronts
// owns RG row groups of TR rows of one sequence and walks their keys in steps,
// every KG-th step a key group's. A step's K, and V transposed, go to LDS once
// for all row groups, and each wavefront computes for its TR rows
//   S^T = K Q^T        (a lane holds several keys' scores of one row)
//   P = 2^(S - offset) (running offset and sum per row; see kRaise)
//   O^T += V^T P^T     (the lane's own weights are the operand: a lane's eight k
//                       slots of a product are taken to be the keys it holds)
// The key groups of a row meet in LDS at the end. Where few rows have many keys,
// several work-groups share a tile's steps, and a second launch merges what they
// wrote (plan). TR is 32 (32 x 32 products) up to head_dim 128, and 16 (16 x 16
// products, half the rows' O and Q) at 256, so that two wavefronts' registers fit
// on a SIMD: one's products run beside the other's softmax and conversions.
// One pass over the keys; only steps that cross a row's span are masked.
//
// Precision. BF16: the operands are exact, P is rounded to BF16 (2^-8 of a
// weight at most; the output is rounded to BF16 as well). F32 and the 4-bit
// cache, whose outputs are F32: Q, P and F32's K and V are fp16 hi + lo (22 bits),
// brought into fp16's range by powers of two (per row of Q, per step for K,
// running for V), the product of two lo parts left out: 3 products for F32, 2
// over the 4-bit cache, whose values are fp16 themselves. Scores, sums and
// outputs are fp32.
//
// Bound: the matrix cores' products beside the softmax's and the conversions'
// VALU work, which two wavefronts per SIMD overlap in part. Useful flops (masked
// ones not counted), where a large BF16 product reaches 1235 TFLOP/s: 8192 tokens
// of 32 over 8 x 64 in BF16 870, eight prompts of 1 to 2048 of 32 over 8 x 128 740,
// 512 tokens over 4096 keys in 4 bits (two products for one) 520 with three
// streams. Tried without gain: two sets of tiles and one barrier a step (2-8 %
// slower up to head_dim 128, 2 % faster at 256), wave priorities around the
// products or the softmax, 16 rows and four wavefronts per SIMD.
//
// Elements that are infinite or NaN: a key's reach only the rows that attend it.
// Scores of masked keys are replaced, but 0 x inf in P V is not, and inf has no
// lo part: a work-group that meets such an element in a masked step (F32: in any
// step) computes its rows anew in fp32 on the vector ALUs, each over its own
// span.
#include "kernels.h"
#include "kv_q4.h"

#include <algorithm>
#include <type_traits>

namespace nnchip
{
	namespace
	{
		constexpr int kBf16 = 0, kF32 = 1, kQ4 = 2;
		// Weights are 2^(score - offset); the offset is raised, to kBelow under the
		// largest score so far, when a score passes it by more than kRaise: weights
		// stay in fp16's range, and rescaling O is rare.
		constexpr float kRaise = 14.0f, kBelow = 6.0f;

		constexpr int kBufferFlags = 0x00020000; // buffer descriptor word 3: raw 32-bit data

		// Keys of a step: as many as leave two wavefronts' registers on a SIMD.
		constexpr int flash_step(int mode, int hd) { return hd <= (mode == kF32 ? 96 : mode == kQ4 ? 128 : 256) ? 64 : 32; }

		template <int MODE_, int HD_, int TR_, int RG_, int KG_>
		struct shape
		{
			static constexpr int MODE = MODE_, HD = HD_, TR = TR_, RG = RG_, KG = KG_;
			static constexpr int WAVES = RG * KG, ROWS = TR * RG;
			static constexpr int KS = flash_step(MODE, HD); // keys of a step
			// Halves per K row, per V^T row: an odd number of 16-byte pieces, or whole
			// rows with their pieces permuted (k_piece, v_piece).
			static constexpr int KP = TR == 16 ? HD : HD + 8, VP = TR == 16 ? KS : KS + 8;
			static constexpr int PARTS = MODE == kF32 ? 2 : 1; // hi, lo
			static constexpr int K_HALVES = KS * KP, V_HALVES = HD * VP;
			static constexpr int TILE_BYTES = 2 * PARTS * (K_HALVES + V_HALVES); // of a key group
			static constexpr int MEET_BYTES = (KG - 1) * RG * (TR * HD + 128) * 4;
			static constexpr int BYTES = KG * TILE_BYTES > MEET_BYTES ? KG * TILE_BYTES : MEET_BYTES;
			static constexpr int THREADS = 64 * RG; // of a key group
			static constexpr int NK = KS * HD / 8 / THREADS; // 8-element pieces of K per thread
			static constexpr int NV = (HD / 2 * (KS / 8) + THREADS - 1) / THREADS; // (column pair, 8 keys) pieces of V per thread
			static constexpr int NR = (KS / 32 * (HD / 32) + RG - 1) / RG; // records per wavefront
			static constexpr int NS = KS / TR, NO = HD / TR, EL = TR * TR / 64; // score tiles, output tiles, registers of one
			static constexpr int QD = 512 / TR, NQ = HD / QD; // columns of a product, products over head_dim
		static_assert(NK * THREADS * 8 == KS * HD && BYTES <= 160 << 10, "shape");
		};

		// Where 8-element piece x of row r of K (of V^T) lies in the row. A 16-byte LDS
		// read goes out in groups of 16 lanes, {0-3, 12-15, 20-27} and {4-11, 16-19,
		// 28-31} of each half wavefront, and two lanes of a group on the same banks
		// take twice as long. In a 32-row product's operand 20-27 are rows 20-27 of one
		// piece, and rows an odd number of pieces long keep them apart; in a 16-row one
		// they are rows 4-11 of the next piece, and those rows ran into one another (1024
		// tokens of 8 over 4 x 256, a window of 1024 over 4 bits: 39 % of the LDS cycles).
		// There a row's pieces are permuted by an exclusive or with a number of the row's
		// that, over rows 4-11, takes x and x ^ 1 equally often.
		template <class G>
		__device__ __forceinline__ int k_piece(int r, int x)
		{
			return G::TR == 16 ? x ^ (r & 15) : x;
		}
		template <class G>
		__device__ __forceinline__ int v_piece(int r, int x)
		{
			if (G::TR != 16) return x;
			if (G::KS == 64) return x ^ ((r >> 1) & 7);
			const int y = (r >> 2) & 3; // (0, 2, 3, 1: rows 4-11 have 2 and 3)
			return x ^ ((y >> 1) | (((y ^ (y >> 1)) & 1) << 1));
		}

		// What a step's loads leave in registers until LDS is free.
		template <class G, bool Q4>
		struct step_regs
		{
			u32x4 k[G::NK * G::PARTS];
			uint32_t v[G::NV][8 * G::PARTS];
		};
		template <class G>
		struct step_regs<G, true> // (4-bit: the wavefront's records)
		{
			u32x4 code[G::NR];
			u32x2 ksz[G::NR];
			u32x4 vs[G::NR], vz[G::NR];
		};

		__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

		// The largest of x over the wavefront.
		__device__ __forceinline__ uint32_t wave_umax(uint32_t x)
		{
			x = umax(x, __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, false));
			x = umax(x, __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, false));
			x = umax(x, __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, false));
			x = umax(x, __builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, false));
			const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
			x = umax(r[0], r[1]);
			const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
			return umax(s[0], s[1]);
		}

		// The power of two that brings a largest magnitude (its bits) under 2^15; 0
		// for zero.
		__device__ __forceinline__ int up_to_2_15(uint32_t bits)
		{
			return bits == 0 ? 0 : 14 - ilogbf(__uint_as_float(bits));
		}

		// Two values as fp16 hi and lo pairs, both rounded to nearest: a lo part is
		// at most 2^-11 of its value and of either sign, so leaving out the products
		// of two lo parts (2^-22 at most) adds no bias.
		__device__ __forceinline__ void split_f16x2(float a, float b, uint32_t& hi, uint32_t& lo)
		{
			const f16x2 h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
			hi = as_u32(h);
			lo = pack_f16x2(a - static_cast<float>(h.x), b - static_cast<float>(h.y));
		}
		// The same for weights, hi cut instead of rounded (one instruction for both):
		// their lo parts meet V's lo parts only, which have either sign.
		__device__ __forceinline__ void split_weights(float a, float b, uint32_t& hi, uint32_t& lo)
		{
			const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
			hi = __builtin_bit_cast(uint32_t, h);
			lo = pack_f16x2(a - static_cast<float>(h[0]), b - static_cast<float>(h[1]));
		}

		// A row's attention in fp32 on the vector ALUs by one wavefront, every
		// operand straight from memory: 64 keys at a time, a lane per key for the
		// scores and per column for the outputs. part: where the row's partial goes
		// (head_dim sums, offset, weights' sum), or null: to out.
		template <int MODE>
		__device__ void vector_row(const flash_params& p, size_t row_at, int tok, int head, int kvh, int first, int last,
		                           int lane, float* part)
		{
			auto el = [](const void* b, size_t i)
			{
				if constexpr (MODE == kBf16) return bf16_bits_to_f32(static_cast<const uint16_t*>(b)[i]);
				else return static_cast<const float*>(b)[i];
			};
			const int hd = p.head_dim;
			const size_t qi = (row_at + tok) * p.q_stride + static_cast<size_t>(head) * hd, col = static_cast<size_t>(kvh) * hd;
			float o[kFlashMaxDim / 64] = {};
			float m = -INFINITY, l = 0.0f;
			for (int k0 = first; k0 <= last; k0 += 64)
			{
				float s = -INFINITY;
				if (k0 + lane <= last)
				{
					const size_t ki = (row_at + k0 + lane) * p.k_stride + col;
					s = 0.0f;
					for (int d = 0; d < hd; ++d) s = fmaf(el(p.q, qi + d), el(p.k, ki + d), s);
					s *= p.scale * kLog2e;
				}
				float now = s;
				for (int x = 1; x < 64; x *= 2) now = fmaxf(now, __shfl_xor(now, x));
				now = fmaxf(now, m);
				const float f = now == m ? 1.0f : fast_exp2(m - now), at = now == -INFINITY ? 0.0f : now;
				m = now;
				const float w = k0 + lane <= last ? fast_exp2(s - at) : 0.0f;
				l = l * f + w;
				for (int c = 0; c < kFlashMaxDim / 64; ++c) o[c] *= f;
				for (int j = 0; j < 64 && k0 + j <= last; ++j)
				{
					const float wj = __shfl(w, j);
					const size_t vi = (row_at + k0 + j) * p.v_stride + col;
					for (int c = 0; c < kFlashMaxDim / 64; ++c)
						if (64 * c + lane < hd) o[c] = fmaf(wj, el(p.v, vi + 64 * c + lane), o[c]);
				}
			}
			for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x);
			if (part && lane == 0) *reinterpret_cast<float2*>(part + hd) = make_float2(m, l);
			const float inv = part ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
			const size_t oi = (row_at + tok) * p.out_stride + static_cast<size_t>(head) * hd;
			for (int c = 0; c < kFlashMaxDim / 64; ++c)
			{
				const int d = 64 * c + lane;
				if (d >= hd) continue;
				if (part) part[d] = o[c];
				else if constexpr (MODE == kBf16) static_cast<uint16_t*>(p.out)[oi + d] = static_cast<uint16_t>(cvt_pk_bf16(o[c] * inv, 0.0f));
				else static_cast<float*>(p.out)[oi + d] = o[c] * inv;
			}
		}

		__device__ __forceinline__ f32x4 mfma(const bf16x8& a, const bf16x8& b, const f32x4& c) { return mfma16x16x32(a, b, c); }
		__device__ __forceinline__ f32x4 mfma(const f16x8& a, const f16x8& b, const f32x4& c) { return mfma16x16x32(a, b, c); }
		__device__ __forceinline__ f32x16 mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) { return mfma32x32x16(a, b, c); }
		__device__ __forceinline__ f32x16 mfma(const f16x8& a, const f16x8& b, const f32x16& c) { return mfma32x32x16(a, b, c); }

		// Over the lanes that hold the same row.
		template <int TR>
		__device__ __forceinline__ float row_max(float x)
		{
			if constexpr (TR == 16)
			{
				const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
				x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
			}
			return max_with_other_half(x);
		}
		template <int TR>
		__device__ __forceinline__ float row_sum(float x)
		{
			return add_with_other_half(TR == 16 ? add_with_other_row(x) : x);
		}

		template <class G, int NSEQ>
		__global__ __launch_bounds__(64 * G::WAVES, 2) void flash_kernel(const flash_params p, const flash_seqs<NSEQ> seqs)
		{
			constexpr int MODE = G::MODE, HD = G::HD, TR = G::TR, KS = G::KS, NS = G::NS, NO = G::NO, EL = G::EL;
			constexpr bool SPLIT = MODE != kBf16; // Q and P as hi + lo
			typedef std::conditional_t<MODE == kBf16, bf16x8, f16x8> op8;
			typedef std::conditional_t<TR == 32, f32x16, f32x4> acc_t;
			typedef step_regs<G, MODE == kQ4> regs_t;
			__shared__ __align__(16) unsigned char smem[G::BYTES];
			__shared__ uint32_t s_max[2][G::WAVES];
			__shared__ uint32_t s_bad;

			const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
			const int rg = wave % G::RG, kg = wave / G::RG; // row group, key group
			const int kt_id = threadIdx.x - 64 * G::RG * kg; // thread of the key group
			const int col = lane % TR, sub = lane / TR; // the lane's row of the row group, its share of a row's keys
			uint16_t* const sk = reinterpret_cast<uint16_t*>(smem + kg * G::TILE_BYTES);
			uint16_t* const sv = sk + G::PARTS * G::K_HALVES;
			if constexpr (MODE != kQ4)
			{
				if (threadIdx.x == 0) s_bad = 0;
				__syncthreads();
			}

			const int hd = p.head_dim, group = p.n_head / p.n_kv;
			const int kvh = static_cast<int>(blockIdx.x % p.n_kv), tile = static_cast<int>(blockIdx.x / p.n_kv);

			// The sequence the tile belongs to: the last one whose tiles begin at or
			// before it (every listed sequence has tiles).
			int s_idx = 0;
#pragma unroll
			for (int c = 0; c < (NSEQ + 63) / 64; ++c)
			{
				const int i = 64 * c + lane;
				s_idx += __popcll(__ballot(i < seqs.n && seqs.tile[i < NSEQ ? i : 0] <= tile));
			}
			s_idx = __builtin_amdgcn_readfirstlane(s_idx - 1);
			const int len = seqs.len[s_idx];
			const size_t row_at = static_cast<size_t>(seqs.start[s_idx]); // of the sequence's first token
			const long long n_rows = static_cast<long long>(len) * group;
			// (the last rows of a causal sequence have the most keys: they go first)
			const int n_blk = static_cast<int>((n_rows + G::ROWS - 1) / G::ROWS);
			const int n_split = seqs.split[s_idx], sp = (tile - seqs.tile[s_idx]) % n_split;
			const long long r0 = static_cast<long long>(n_blk - 1 - (tile - seqs.tile[s_idx]) / n_split) * G::ROWS;
			const int pos0 = MODE == kQ4 ? p.pos0 : 0, n_keys = MODE == kQ4 ? p.n_seq : len;

			auto token_of = [&](long long r) { return static_cast<int>((r < n_rows ? r : n_rows - 1) / group); };
			auto span_of = [&](long long r, int& a, int& b) { attn_span(p.causal, p.window, pos0 + token_of(r), n_keys, a, b); };

			// The lane's row, and the keys of the work-group's and the wavefront's rows.
			const long long w0 = r0 + TR * rg, row = w0 + col;
			const bool real = row < n_rows;
			const int tok = token_of(row), head = kvh * group + (real ? static_cast<int>(row % group) : 0);
			int first, last;
			attn_span(p.causal, p.window, pos0 + tok, n_keys, first, last);
			int kmin, kmax, full_from, full_to, unused;
			span_of(r0, kmin, unused);
			span_of(r0 + G::ROWS - 1, unused, kmax);
			span_of(w0, unused, full_to); // every row of the wavefront sees full_from .. full_to
			span_of(w0 + TR - 1, full_from, unused);
			// The work-group's steps: its share of those from kmin's on.
			const int k_first = kmin / KS * KS;
			const int all_steps = kmax < k_first ? 0 : (kmax - k_first) / KS + 1;
			const int s_from = static_cast<int>(static_cast<long long>(all_steps) * sp / n_split);
			const int s_to = static_cast<int>(static_cast<long long>(all_steps) * (sp + 1) / n_split);
			const int k_from = k_first + s_from * KS, k_end = k_first + s_to * KS; // (a key group may step past k_end: masked)
			last = last < k_end - 1 ? last : k_end - 1;
			full_to = full_to < k_end - 1 ? full_to : k_end - 1;

			// ---- Q ----
			constexpr int NQ = G::NQ;
			op8 qh[NQ];
			f16x8 ql[SPLIT ? NQ : 1];
			// (S * sc in log2 units; the scale's sign goes into Q, so that a masked
			// score stays the least whatever the scale)
			float sc = fmaxf(fabsf(p.scale) * kLog2e, 1.17549435e-38f);
			if constexpr (!SPLIT)
			{
				const uint16_t* q = static_cast<const uint16_t*>(p.q) + (row_at + tok) * p.q_stride + static_cast<size_t>(head) * hd;
				const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
				for (int ks = 0; ks < NQ; ++ks)
				{
					const int d = G::QD * ks + 8 * sub;
					u32x4 w = {0, 0, 0, 0};
					if (d < hd) w = *reinterpret_cast<const u32x4*>(q + d) ^ u32x4{flip, flip, flip, flip};
					qh[ks] = as_bf16x8(w);
				}
			}
			else
			{
				const float* q = static_cast<const float*>(p.q) + (row_at + tok) * p.q_stride + static_cast<size_t>(head) * hd;
				float x[NQ][8];
				float m = 0.0f;
#pragma unroll
				for (int ks = 0; ks < NQ; ++ks)
				{
					const int d = G::QD * ks + 8 * sub;
					float4 u = {0, 0, 0, 0}, v = {0, 0, 0, 0};
					if (d < hd) u = *reinterpret_cast<const float4*>(q + d), v = *reinterpret_cast<const float4*>(q + d + 4);
					if constexpr (MODE == kQ4) // (the k slot order of the 4-bit values)
						x[ks][0] = u.x, x[ks][1] = v.x, x[ks][2] = u.y, x[ks][3] = v.y, x[ks][4] = u.z, x[ks][5] = v.z, x[ks][6] = u.w,
						x[ks][7] = v.w;
					else
						x[ks][0] = u.x, x[ks][1] = u.y, x[ks][2] = u.z, x[ks][3] = u.w, x[ks][4] = v.x, x[ks][5] = v.y, x[ks][6] = v.z,
						x[ks][7] = v.w;
#pragma unroll
					for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[ks][j]));
				}
				m = row_max<TR>(m);
				// (0, infinity and NaN: as they are)
				const int e = m > 0.0f && m < INFINITY ? up_to_2_15(__float_as_uint(m)) : 0;
				const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
				sc = fmaxf(ldexpf(sc, -e), 1.17549435e-38f);
#pragma unroll
				for (int ks = 0; ks < NQ; ++ks)
				{
					u32x4 h, l;
#pragma unroll
					for (int j = 0; j < 4; ++j)
					{
						uint32_t a, b;
						split_f16x2(sign * ldexpf(x[ks][2 * j], e), sign * ldexpf(x[ks][2 * j + 1], e), a, b);
						h[j] = a;
						l[j] = b;
					}
					qh[ks] = as_f16x8(h);
					ql[ks] = as_f16x8(l);
				}
			}

			// ---- the loads of a step ----
			// Through buffer descriptors that end with the sequence's last row: keys
			// past it read as zeros, and a thread's offsets are the same in every
			// step (columns past head_dim: an offset past any descriptor).
			constexpr int ESIZE = MODE == kBf16 ? 2 : 4;
			const int blocks = hd / kQ4Block; // 4-bit: records of a KV head and group
			// V^T's rows hold 32 keys as four pieces of eight k slots: keys 4 x + j and
			// 16 + 4 x + j alternate in piece x, which are keys whose weights one lane
			// holds, in either product's layout.
			constexpr uint32_t kNowhere = 0x80000000u;
			uint32_t k_off[G::NK], v_off[G::NV];
			if constexpr (MODE != kQ4)
			{
#pragma unroll
				for (int n = 0; n < G::NK; ++n)
				{
					const int c = kt_id + G::THREADS * n, d = 8 * (c % (HD / 8));
					k_off[n] = d < hd ? static_cast<uint32_t>((c / (HD / 8)) * p.k_stride + d) * ESIZE : kNowhere;
				}
#pragma unroll
				for (int n = 0; n < G::NV; ++n)
				{
					const int c = kt_id + G::THREADS * n, set = c / (HD / 2), d = 2 * (c % (HD / 2));
					const int key = 32 * (set >> 2) + 4 * (set & 3);
					v_off[n] = set < KS / 8 && d < hd ? static_cast<uint32_t>(key * p.v_stride + d) * ESIZE : kNowhere;
				}
			}
			// Rows k0 .. of a tensor (at most KS of them, as far as the sequence goes; past
			// the work-group's last key none: zeros).
			auto rows_from = [&](const void* base, size_t stride, int k0)
			{
				const int n = k0 > kmax || k0 >= k_end ? 0 : n_keys - k0 < KS ? n_keys - k0 : KS;
				const char* at = static_cast<const char*>(base) + ((row_at + k0) * stride + static_cast<size_t>(kvh) * hd) * ESIZE;
				return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(at), 0, n ? static_cast<int>(((n - 1) * stride + hd) * ESIZE) : 0, kBufferFlags);
			};
			auto load_step = [&](int k0, regs_t& g)
			{
				if constexpr (MODE == kQ4)
				{
					const int groups = p.rows / kQ4Rows;
#pragma unroll
					for (int n = 0; n < G::NR; ++n)
					{
						const int rec = rg * G::NR + n, b = rec % (HD / 32), gi = rec / (HD / 32);
						g.code[n] = u32x4{0, 0, 0, 0};
						g.ksz[n] = u32x2{0, 0};
						g.vs[n] = g.vz[n] = u32x4{0, 0, 0, 0};
						if (gi >= KS / 32 || b >= blocks || k0 + 32 * gi > kmax || k0 >= k_end) continue;
						const unsigned char* at = static_cast<const unsigned char*>(p.k) +
						                          (static_cast<size_t>((k0 / kQ4Rows + gi) % groups) * (p.n_kv * blocks) + kvh * blocks + b) * kQ4Record;
						g.code[n] = *reinterpret_cast<const u32x4*>(at + 16 * lane);
						g.ksz[n] = *reinterpret_cast<const u32x2*>(at + kQ4KScales + 8 * (lane & 15));
						g.vs[n] = *reinterpret_cast<const u32x4*>(at + kQ4VScales + 32 * (lane >> 4));
						g.vz[n] = *reinterpret_cast<const u32x4*>(at + kQ4VScales + 32 * (lane >> 4) + 16);
					}
				}
				else
				{
					const auto rk = rows_from(p.k, p.k_stride, k0), rv = rows_from(p.v, p.v_stride, k0);
#pragma unroll
					for (int n = 0; n < G::NK; ++n)
#pragma unroll
						for (int x = 0; x < G::PARTS; ++x)
							g.k[G::PARTS * n + x] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off[n] + 16 * x, 0, 0));
					const uint32_t row_bytes = static_cast<uint32_t>(p.v_stride * ESIZE);
#pragma unroll
					for (int n = 0; n < G::NV; ++n)
#pragma unroll
						for (int u = 0; u < 8; ++u)
						{
							// (in the checked offset: a scalar one would be taken off the bound)
							const uint32_t at = v_off[n] + ((u >> 1) + 16 * (u & 1)) * row_bytes;
							if constexpr (MODE == kBf16)
								g.v[n][u] = __builtin_amdgcn_raw_buffer_load_b32(rv, at, 0, 0);
							else
							{
								const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rv, at, 0, 0));
								g.v[n][2 * u] = w.x;
								g.v[n][2 * u + 1] = w.y;
							}
						}
				}
			};

			// The registers' K rows and V^T rows into LDS (F32: times 2^ek, 2^ev).
			auto store_step = [&](const regs_t& g, int ek, int ev)
			{
				if constexpr (MODE == kQ4)
				{
					const q4_masks masks;
#pragma unroll
					for (int n = 0; n < G::NR; ++n)
					{
						const int rec = rg * G::NR + n, b = rec % (HD / 32), gi = rec / (HD / 32);
						if (gi >= KS / 32) continue;
						const int i = lane & 15, q = lane >> 4;
#pragma unroll
						for (int t = 0; t < 2; ++t)
						{
							const f16x8 x = q4_k(t ? g.code[n].y : g.code[n].x, t ? g.ksz[n].y : g.ksz[n].x, masks);
							const int kr = 32 * gi + 16 * t + i, vr = 32 * b + 16 * t + i;
							*reinterpret_cast<f16x8*>(sk + kr * G::KP + 8 * k_piece<G>(kr, 4 * b + q)) = x;
							// (quarter q of the rows is V^T's piece q)
							const f16x8 y = q4_v(t ? g.code[n].w : g.code[n].z, g.vs[n], g.vz[n], masks);
							*reinterpret_cast<f16x8*>(sv + vr * G::VP + 8 * v_piece<G>(vr, 4 * gi + q)) = y;
						}
					}
				}
				else if constexpr (MODE == kBf16)
				{
#pragma unroll
					for (int n = 0; n < G::NK; ++n)
					{
						const int c = kt_id + G::THREADS * n;
						*reinterpret_cast<u32x4*>(sk + c / (HD / 8) * G::KP + 8 * k_piece<G>(c / (HD / 8), c % (HD / 8))) = g.k[n];
					}
#pragma unroll
					for (int n = 0; n < G::NV; ++n)
					{
						const int c = kt_id + G::THREADS * n, set = c / (HD / 2), d = 2 * (c % (HD / 2));
						if (set >= KS / 8) continue;
						u32x4 a, b; // columns d and d + 1
#pragma unroll
						for (int j = 0; j < 4; ++j)
						{
							a[j] = __builtin_amdgcn_perm(g.v[n][2 * j + 1], g.v[n][2 * j], 0x05040100u);
							b[j] = __builtin_amdgcn_perm(g.v[n][2 * j + 1], g.v[n][2 * j], 0x07060302u);
						}
						*reinterpret_cast<u32x4*>(sv + d * G::VP + 8 * v_piece<G>(d, set)) = a;
						*reinterpret_cast<u32x4*>(sv + (d + 1) * G::VP + 8 * v_piece<G>(d + 1, set)) = b;
					}
				}
				else
				{
#pragma unroll
					for (int n = 0; n < G::NK; ++n)
					{
						const int c = kt_id + G::THREADS * n;
						u32x4 h, l;
#pragma unroll
						for (int j = 0; j < 4; ++j)
						{
							const u32x4 w = g.k[2 * n + (j >> 1)];
							uint32_t a, b;
							split_f16x2(ldexpf(__uint_as_float(w[2 * (j & 1)]), ek), ldexpf(__uint_as_float(w[2 * (j & 1) + 1]), ek), a, b);
							h[j] = a;
							l[j] = b;
						}
						uint16_t* at = sk + c / (HD / 8) * G::KP + 8 * k_piece<G>(c / (HD / 8), c % (HD / 8));
						*reinterpret_cast<u32x4*>(at) = h;
						*reinterpret_cast<u32x4*>(at + G::K_HALVES) = l;
					}
#pragma unroll
					for (int n = 0; n < G::NV; ++n)
					{
						const int c = kt_id + G::THREADS * n, set = c / (HD / 2), d = 2 * (c % (HD / 2));
						if (set >= KS / 8) continue;
#pragma unroll
						for (int col = 0; col < 2; ++col)
						{
							u32x4 h, l;
#pragma unroll
							for (int j = 0; j < 4; ++j)
							{
								uint32_t a, b;
								split_f16x2(ldexpf(__uint_as_float(g.v[n][4 * j + col]), ev), ldexpf(__uint_as_float(g.v[n][4 * j + 2 + col]), ev), a, b);
								h[j] = a;
								l[j] = b;
							}
							uint16_t* at = sv + (d + col) * G::VP + 8 * v_piece<G>(d + col, set);
							*reinterpret_cast<u32x4*>(at) = h;
							*reinterpret_cast<u32x4*>(at + G::V_HALVES) = l;
						}
					}
				}
			};

			// ---- the walk ----
			const int k_lane = col * G::KP + 8 * k_piece<G>(col, sub), v_lane = col * G::VP + 8 * v_piece<G>(col, sub);
			acc_t o[NO] = {};
			float off = -INFINITY, l = 0.0f;
			// F32: V goes to LDS times 2^ev, O is in units of 2^-ev_o (1000: nothing yet).
			int ev = 1000, ev_o = 1000;
			// Raises the offset for a largest score m (in log2 units), and takes O to ev's
			// units.
			auto raise = [&](float m)
			{
				const bool up = m > off + kRaise;
				if (__any(up) || (MODE == kF32 && ev_o != ev))
				{
					const float now = up ? m - kBelow : off;
					float f = up ? fast_exp2(off - now) : 1.0f; // (equal ones: -inf - -inf is NaN)
					off = now;
					l *= f;
					if constexpr (MODE == kF32)
					{
						if (ev_o != 1000) f = ldexpf(f, ev - ev_o);
						ev_o = ev;
					}
#pragma unroll
					for (int dt = 0; dt < NO; ++dt) o[dt] *= f;
				}
			};

			regs_t regs;
			if (s_from < s_to) load_step(k_from + kg * KS, regs);
			for (int step = s_from + kg; step - kg < s_to; step += G::KG) // (as often for every key group)
			{
				const int k0 = k_first + step * KS;
				// Largest magnitudes (F32), or whether V holds an infinite or NaN element
				// (BF16, masked steps).
				int ek = 0;
				if constexpr (MODE == kF32)
				{
					uint32_t mk = 0, mv = 0;
#pragma unroll
					for (int n = 0; n < 2 * G::NK; ++n)
#pragma unroll
						for (int j = 0; j < 4; ++j) mk = umax(mk, regs.k[n][j] & 0x7fffffffu);
#pragma unroll
					for (int n = 0; n < G::NV; ++n)
#pragma unroll
						for (int j = 0; j < 16; ++j) mv = umax(mv, regs.v[n][j] & 0x7fffffffu);
					mk = wave_umax(mk);
					mv = wave_umax(mv);
					if (lane == 0) s_max[0][wave] = mk, s_max[1][wave] = mv;
				}
				else if constexpr (MODE == kBf16)
				{
					int a, b;
					span_of(r0, unused, b);
					span_of(r0 + G::ROWS - 1, a, unused);
					if (k0 < a || k0 + KS - 1 > b) // some row of the work-group does not see them all
					{
						bool bad = false;
#pragma unroll
						for (int n = 0; n < G::NV; ++n)
#pragma unroll
							for (int u = 0; u < 8; ++u)
								bad |= (regs.v[n][u] & 0x7f80u) == 0x7f80u || (regs.v[n][u] & 0x7f800000u) == 0x7f800000u;
						if (__any(bad)) s_bad = 1;
					}
				}
				__syncthreads(); // every wavefront is done with the step before
				if constexpr (MODE == kF32)
				{
					uint32_t mk = 0, mv = 0;
#pragma unroll
					for (int w = 0; w < G::RG; ++w) mk = umax(mk, s_max[0][kg * G::RG + w]), mv = umax(mv, s_max[1][kg * G::RG + w]);
					mk = __builtin_amdgcn_readfirstlane(mk);
					mv = __builtin_amdgcn_readfirstlane(mv);
					if (mk >= 0x7f800000u || mv >= 0x7f800000u)
						s_bad = 1; // (what this step computes is not used)
					else
					{
						ek = up_to_2_15(mk);
						const int want = mv == 0 ? ev : up_to_2_15(mv);
						if (want < ev) ev = want; // (V grows: O follows, in raise)
					}
				}
				// (a key group past the last step stores zeros, and all its keys are masked)
				store_step(regs, ek, ev);
				if (step + G::KG - kg < s_to) load_step(k0 + G::KG * KS, regs);
				__syncthreads();

				acc_t s[NS] = {};
#pragma unroll
				for (int t = 0; t < NS; ++t)
#pragma unroll
					for (int ks = 0; ks < NQ; ++ks)
					{
						// (4 ks + sub, permuted by col: bits 2 and 3 of the piece's number from ks)
						const uint16_t* at = TR == 16 ? sk + (k_lane ^ (32 * (ks & 3))) + TR * t * G::KP + 128 * (ks >> 2)
						                              : sk + k_lane + TR * t * G::KP + G::QD * ks;
						const op8 a = *reinterpret_cast<const op8*>(at);
						s[t] = mfma(a, qh[ks], s[t]);
						if constexpr (SPLIT) s[t] = mfma(a, ql[ks], s[t]);
						if constexpr (MODE == kF32) s[t] = mfma(*reinterpret_cast<const op8*>(at + G::K_HALVES), qh[ks], s[t]);
					}
				float f = sc;
				if constexpr (MODE == kF32) f = fminf(fmaxf(ldexpf(sc, -ek), 1.17549435e-38f), 1e36f);
				if (k0 < full_from || k0 + KS - 1 > full_to)
#pragma unroll
					for (int t = 0; t < NS; ++t)
#pragma unroll
						for (int i = 0; i < EL; ++i)
						{
							const int key = k0 + TR * t + 8 * (i >> 2) + 4 * sub + (i & 3);
							if (key < first || key > last) s[t][i] = -INFINITY;
						}
				float m = s[0][0];
#pragma unroll
				for (int t = 0; t < NS; ++t)
#pragma unroll
					for (int i = 0; i < EL; ++i) m = fmaxf(m, s[t][i]);
				raise(row_max<TR>(m) * f);
				const float at = off == -INFINITY ? 0.0f : off;
#pragma unroll
				for (int t = 0; t < NS; ++t)
#pragma unroll
					for (int i = 0; i < EL; ++i)
					{
						s[t][i] = fast_exp2(fmaf(s[t][i], f, -at));
						l += s[t][i];
					}
				// (a product's 64 * 8 / TR keys: half a 32-key tile's pieces, or all four)
#pragma unroll
				for (int x = 0; x < KS * TR / 512; ++x)
				{
					u32x4 wh, wl;
#pragma unroll
					for (int j = 0; j < 4; ++j)
					{
						float a, b;
						if constexpr (TR == 32)
							a = s[x >> 1][4 * (x & 1) + j], b = s[x >> 1][8 + 4 * (x & 1) + j];
						else
							a = s[2 * x][j], b = s[2 * x + 1][j];
						if constexpr (SPLIT)
						{
							uint32_t y, z;
							split_weights(a, b, y, z);
							wh[j] = y;
							wl[j] = z;
						}
						else
							wh[j] = cvt_pk_bf16(a, b);
					}
					const op8 ph = __builtin_bit_cast(op8, wh);
#pragma unroll
					for (int dt = 0; dt < NO; ++dt)
					{
						const uint16_t* v = sv + (TR == 16 ? v_lane ^ (32 * x) : v_lane + 16 * x) + TR * dt * G::VP;
						const op8 a = *reinterpret_cast<const op8*>(v);
						o[dt] = mfma(a, ph, o[dt]);
						if constexpr (SPLIT) o[dt] = mfma(a, __builtin_bit_cast(op8, wl), o[dt]);
						if constexpr (MODE == kF32) o[dt] = mfma(*reinterpret_cast<const op8*>(v + G::V_HALVES), ph, o[dt]);
					}
				}
			}

			auto part_of_row = [&](long long r)
			{ return p.part + (seqs.part[s_idx] + (static_cast<size_t>(r) * p.n_kv + kvh) * n_split + sp) * (hd + 4); };
			l = row_sum<TR>(l);
			if constexpr (MODE == kF32)
				if (ev_o != 1000)
#pragma unroll
					for (int dt = 0; dt < NO; ++dt)
#pragma unroll
						for (int i = 0; i < EL; ++i) o[dt][i] = ldexpf(o[dt][i], -ev_o);
			if (G::KG > 1 || MODE != kQ4) __syncthreads();
			if constexpr (MODE != kQ4)
				if (s_bad)
				{
					for (int r = wave; r < G::ROWS && r0 + r < n_rows; r += G::WAVES)
					{
						const long long x = r0 + r;
						int a, b;
						span_of(x, a, b);
						vector_row<MODE>(p, row_at, token_of(x), kvh * group + static_cast<int>(x % group), kvh, a > k_from ? a : k_from,
						                 b < k_end - 1 ? b : k_end - 1, lane, n_split > 1 ? part_of_row(x) : nullptr);
					}
					return;
				}

			// ---- the key groups of a row meet, in order ----
			if constexpr (G::KG > 1)
			{
				constexpr int Q = TR * HD / 256; // float4s of a lane
				float4* const part = reinterpret_cast<float4*>(smem);
				float2* const ml = reinterpret_cast<float2*>(smem + static_cast<size_t>(G::KG - 1) * G::RG * TR * HD * 4);
				if (kg > 0)
				{
					const int w = (kg - 1) * G::RG + rg;
#pragma unroll
					for (int q = 0; q < Q; ++q)
						part[(w * Q + q) * 64 + lane] = float4{o[q / (EL / 4)][4 * (q % (EL / 4))], o[q / (EL / 4)][4 * (q % (EL / 4)) + 1],
						                                       o[q / (EL / 4)][4 * (q % (EL / 4)) + 2], o[q / (EL / 4)][4 * (q % (EL / 4)) + 3]};
					ml[w * 64 + lane] = make_float2(off, l);
				}
				__syncthreads();
				if (kg > 0) return;
#pragma unroll
				for (int g = 1; g < G::KG; ++g)
				{
					const int w = (g - 1) * G::RG + rg;
					const float2 y = ml[w * 64 + lane];
					const float now = fmaxf(off, y.x), to = now == -INFINITY ? 0.0f : now;
					const float fa = fast_exp2(off - to), fb = fast_exp2(y.x - to);
					off = now;
					l = l * fa + y.y * fb;
#pragma unroll
					for (int q = 0; q < Q; ++q)
					{
						const float4 z = part[(w * Q + q) * 64 + lane];
						auto& t = o[q / (EL / 4)];
						const int e = 4 * (q % (EL / 4));
						t[e] = fmaf(z.x, fb, t[e] * fa);
						t[e + 1] = fmaf(z.y, fb, t[e + 1] * fa);
						t[e + 2] = fmaf(z.z, fb, t[e + 2] * fa);
						t[e + 3] = fmaf(z.w, fb, t[e + 3] * fa);
					}
				}
			}

			// ---- out ----
			if (!real) return;
			if (n_split > 1)
			{
				float* const part = part_of_row(row);
#pragma unroll
				for (int dt = 0; dt < NO; ++dt)
#pragma unroll
					for (int c = 0; c < EL / 4; ++c)
					{
						const int d = TR * dt + 8 * c + 4 * sub;
						if (d < hd) *reinterpret_cast<float4*>(part + d) = float4{o[dt][4 * c], o[dt][4 * c + 1], o[dt][4 * c + 2], o[dt][4 * c + 3]};
					}
				if (sub == 0) *reinterpret_cast<float2*>(part + hd) = make_float2(off, l);
				return;
			}
			const float inv = l == 0.0f ? 0.0f : 1.0f / l; // (a row that sees nothing: zeros)
			const size_t oi = (row_at + tok) * p.out_stride + static_cast<size_t>(head) * hd;
#pragma unroll
			for (int dt = 0; dt < NO; ++dt)
#pragma unroll
				for (int c = 0; c < EL / 4; ++c)
				{
					const int d = TR * dt + 8 * c + 4 * sub;
					if (d >= hd) continue;
					float y[4];
#pragma unroll
					for (int j = 0; j < 4; ++j)
					{
						y[j] = o[dt][4 * c + j] * inv;
						if constexpr (MODE == kQ4) y[j] = gated(y[j], p.gate, oi + d + j);
					}
					if constexpr (MODE == kBf16)
						*reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.out) + oi + d) = u32x2{cvt_pk_bf16(y[0], y[1]), cvt_pk_bf16(y[2], y[3])};
					else
						*reinterpret_cast<float4*>(static_cast<float*>(p.out) + oi + d) = float4{y[0], y[1], y[2], y[3]};
				}
		}

		// The partials of rows whose keys several work-groups shared, joined in key
		// order. A float4 column of a row per thread.
		template <int MODE, int NSEQ>
		__global__ __launch_bounds__(256) void flash_merge_kernel(const flash_params p, const flash_seqs<NSEQ> seqs)
		{
			const int hd = p.head_dim, group = p.n_head / p.n_kv, cols = hd / 4, rows_here = 256 / cols;
			const int c = threadIdx.x % cols, lane = threadIdx.x & 63;
			int s_idx = 0;
#pragma unroll
			for (int x = 0; x < (NSEQ + 63) / 64; ++x)
			{
				const int i = 64 * x + lane;
				s_idx += __popcll(__ballot(i < seqs.n && seqs.tile[i < NSEQ ? i : 0] <= static_cast<int>(blockIdx.x)));
			}
			s_idx = __builtin_amdgcn_readfirstlane(s_idx - 1);
			const long long x = static_cast<long long>(blockIdx.x - seqs.tile[s_idx]) * rows_here + threadIdx.x / cols;
			if (threadIdx.x / cols >= rows_here || x >= static_cast<long long>(seqs.len[s_idx]) * p.n_head) return;
			const int n_split = seqs.split[s_idx], kvh = static_cast<int>(x % p.n_kv);
			const long long row = x / p.n_kv;
			const int tok = static_cast<int>(row / group), head = kvh * group + static_cast<int>(row % group);
			const float* part = p.part + (seqs.part[s_idx] + static_cast<size_t>(x) * n_split) * (hd + 4);
			float m = -INFINITY;
			for (int i = 0; i < n_split; ++i) m = fmaxf(m, part[static_cast<size_t>(i) * (hd + 4) + hd]);
			const float off = m == -INFINITY ? 0.0f : m;
			float4 o = {0, 0, 0, 0};
			float l = 0.0f;
			for (int i = 0; i < n_split; ++i, part += hd + 4)
			{
				const float2 ml = *reinterpret_cast<const float2*>(part + hd);
				const float4 v = *reinterpret_cast<const float4*>(part + 4 * c);
				const float f = fast_exp2(ml.x - off);
				o = float4{fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w)};
				l = fmaf(ml.y, f, l);
			}
			const float inv = l == 0.0f ? 0.0f : 1.0f / l;
			float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
			const size_t at = (static_cast<size_t>(seqs.start[s_idx]) + tok) * p.out_stride + static_cast<size_t>(head) * hd + 4 * c;
			if constexpr (MODE == kQ4)
				for (int j = 0; j < 4; ++j) y[j] = gated(y[j], p.gate, at + j);
			if constexpr (MODE == kBf16)
				*reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.out) + at) = u32x2{cvt_pk_bf16(y[0], y[1]), cvt_pk_bf16(y[2], y[3])};
			else
				*reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = float4{y[0], y[1], y[2], y[3]};
		}

		// The compiled head_dim that takes head_dim's place, and the rows of a tile.
		int flash_dim(int hd) { return hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : 256; }
		int flash_rows(int hd, int key_groups) { return flash_dim(hd) == 256 && key_groups == 2 ? 64 : 128; }

		// Fills in the tiles and launches; then, where keys are shared, the merge.
		template <class G, int NSEQ>
		bool launch_shape(const flash_params& p, flash_seqs<NSEQ>& s, hipStream_t stream)
		{
			long long tiles = 0;
			for (int i = 0; i < s.n; ++i)
			{
				s.tile[i] = static_cast<int>(tiles);
				tiles += (static_cast<long long>(s.len[i]) * (p.n_head / p.n_kv) + G::ROWS - 1) / G::ROWS * s.split[i];
				if (tiles * p.n_kv * (64 * G::WAVES) > 0xffffffffll) return false;
			}
			if (!tiles) return true;
			flash_kernel<G, NSEQ><<<dim3(static_cast<unsigned>(tiles * p.n_kv)), 64 * G::WAVES, 0, stream>>>(p, s);
			flash_seqs<NSEQ> m{};
			long long groups = 0;
			const int rows_here = 256 / (p.head_dim / 4);
			for (int i = 0; i < s.n; ++i)
			{
				if (s.split[i] == 1) continue;
				m.start[m.n] = s.start[i];
				m.len[m.n] = s.len[i];
				m.split[m.n] = s.split[i];
				m.part[m.n] = s.part[i];
				m.tile[m.n] = static_cast<int>(groups); // (partials of at most kFlashScratch bytes: few)
				groups += (static_cast<long long>(s.len[i]) * p.n_head + rows_here - 1) / rows_here;
				++m.n;
			}
			if (m.n) flash_merge_kernel<G::MODE, NSEQ><<<dim3(static_cast<unsigned>(groups)), 256, 0, stream>>>(p, m);
			return true;
		}

		// Keys that the tile of token t0 .. reads (rows of a tile: `tokens` tokens).
		long long tile_keys(const flash_params& p, bool q4, int len, int t0, int tokens)
		{
			const int pos0 = q4 ? p.pos0 : 0, n_keys = q4 ? p.n_seq : len, t1 = std::min(t0 + tokens, len) - 1;
			int a, b, unused;
			attn_span(p.causal, p.window, pos0 + t0, n_keys, a, unused);
			attn_span(p.causal, p.window, pos0 + t1, n_keys, unused, b);
			return std::max(0, b - a + 1);
		}

		// Key groups and splits of a launch.
		//
		// One key group while there is a work-group for every CU; below that two, so
		// that a CU's one work-group still has two wavefronts per SIMD (us alone /
		// with three streams in flight, one -> two: 512 tokens of 32 over 8 x 128 at
		// 4k keys over 4 bits, 128 work-groups, 137 / 65 -> 108 / 61; 1024 of 8
		// over 4 x 256, a window of 1024, 64 work-groups, 72 / 25 -> 48 / 25;
		// eight prompts of 1 to 2048 tokens, 1752 work-groups, 113 / 113 -> 152 /
		// 148). Four key groups of half the rows gain more alone (78 and 38) and lose
		// as much in flight (73 and 37). F32 at head_dim 256 converts K and V for half
		// as many rows with two, and keeps one down to a quarter of the CUs (twelve
		// texts of 5 to 1500 tokens of 3 x 256, 121 work-groups: 77 / 33 -> 63 / 44).
		//
		// A sequence's keys are shared out where its longest tile has at least 2.3
		// times the steps (64 keys) that each CU has on average, counted as 12 at least
		// (6 where the partials are small): a launch lasts as long as its longest work-group.
		// (us alone / three streams, not shared -> shared: 20 tokens of 4 over 1 x 256
		// at 8k keys 265 / 90 -> 37 / 14; 40 of 32 over 8 x 128 at 6k 154 / 52 -> 39 /
		// 18; 900 of 8 over 4 x 256 at 5k 203 / 89 -> 116 / 95.) Its partials cost
		// memory traffic and a launch: from twice the average on, or down to 6 steps
		// for all, what a lone stream gained others in flight lost (512 tokens at 4k
		// keys, above, 108 / 61 -> 80 / 72; the window of 1024 48 / 25 -> 42 / 32; one
		// BF16 prompt of 1500 tokens of 4 over 1 x 256 51 / 18 -> 39 / 27). At most
		// `limit` bytes of partials, the longest sequences first (they come in that
		// order).
		constexpr double kShare = 2.3, kShareSteps = 12.0, kShareFewSteps = 6.0;
		constexpr size_t kShareSmall = size_t{8} << 20;
		template <int NSEQ>
		size_t plan(const flash_params& p, flash_seqs<NSEQ>& s, int mode, int n_cu, size_t limit)
		{
			const int group = p.n_head / p.n_kv, hd = flash_dim(p.head_dim);
			long long tiles = 0;
			for (int i = 0; i < s.n; ++i) tiles += (static_cast<long long>(s.len[i]) * group + 127) / 128;
			s.key_groups = tiles * p.n_kv > (mode == kF32 && hd == 256 ? n_cu / 4 : n_cu) ? 1 : 2;
			const int rows = flash_rows(hd, s.key_groups), tokens = std::max(1, rows / group);
			auto steps_of = [&](int i, bool longest)
			{
				const int len = s.len[i], end = std::max(0, len - tokens);
				const long long a = tile_keys(p, mode == kQ4, len, 0, tokens), b = tile_keys(p, mode == kQ4, len, end, tokens),
				                mid = tile_keys(p, mode == kQ4, len, end / 2, tokens);
				return static_cast<double>(longest ? std::max({a, b, mid}) : (a + b + 2 * mid) / 4) / 64;
			};
			double work = 0;
			for (int i = 0; i < s.n; ++i)
				work += steps_of(i, false) * static_cast<double>((static_cast<long long>(s.len[i]) * group + rows - 1) / rows) * p.n_kv;
			size_t used = 0;
			const size_t row_bytes = static_cast<size_t>(p.head_dim + 4) * sizeof(float);
			for (int i = 0; i < s.n; ++i)
			{
				s.split[i] = 1;
				s.part[i] = 0;
				const double steps = steps_of(i, true);
				const size_t one = static_cast<size_t>(s.len[i]) * p.n_head * row_bytes;
				const bool small = one * (steps / kShareFewSteps) <= kShareSmall;
				const double share = std::max(small ? kShareFewSteps : kShareSteps, work / n_cu);
				if (steps < kShare * share) continue;
				const long long fit = static_cast<long long>((limit - used) / one), want = static_cast<long long>(steps / share + 0.5);
				const int n = static_cast<int>(std::min<long long>({fit, want, 64}));
				if (n < 2) continue;
				s.split[i] = n;
				s.part[i] = static_cast<int>(used / row_bytes);
				used += one * n;
			}
			return used;
		}

		template <int MODE, int HD, int NSEQ>
		bool launch_dim(const flash_params& p, flash_seqs<NSEQ>& s, hipStream_t stream)
		{
			const bool one = s.key_groups == 1;
			if constexpr (HD == 256)
				return one ? launch_shape<shape<MODE, HD, 16, 8, 1>>(p, s, stream) : launch_shape<shape<MODE, HD, 16, 4, 2>>(p, s, stream);
			else
				return one ? launch_shape<shape<MODE, HD, 32, 4, 1>>(p, s, stream) : launch_shape<shape<MODE, HD, 32, 4, 2>>(p, s, stream);
		}
		template <int MODE, int NSEQ>
		bool launch_mode(const flash_params& p, flash_seqs<NSEQ>& s, hipStream_t stream)
		{
			switch (flash_dim(p.head_dim))
			{
			case 64: return launch_dim<MODE, 64>(p, s, stream);
			case 96: return launch_dim<MODE, 96>(p, s, stream);
			case 128: return launch_dim<MODE, 128>(p, s, stream);
			default: return launch_dim<MODE, 256>(p, s, stream);
			}
		}
	}

	size_t plan_packed(const flash_params& p, flash_seqs<kFlashSeqs>& s, bool bf16, int n_cu, size_t limit)
	{
		return plan(p, s, bf16 ? kBf16 : kF32, n_cu, limit);
	}
	bool launch_packed(const flash_params& p, flash_seqs<kFlashSeqs>& s, bool bf16, hipStream_t stream)
	{
		return bf16 ? launch_mode<kBf16>(p, s, stream) : launch_mode<kF32>(p, s, stream);
	}
	size_t plan_flash_q4(const flash_params& p, flash_seqs<1>& s, int n_tok, int n_cu, size_t limit)
	{
		s.n = 1;
		s.start[0] = 0;
		s.len[0] = n_tok;
		return plan(p, s, kQ4, n_cu, limit);
	}
	bool launch_flash_q4(const flash_params& p, flash_seqs<1>& s, hipStream_t stream) { return launch_mode<kQ4>(p, s, stream); }
}
