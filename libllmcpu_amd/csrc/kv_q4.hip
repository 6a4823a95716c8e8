// Writing the 4-bit cache (kv_q4.h has the format and the layout): rows
// quantised from F32 or taken in the interchange form, and their values or raw
// blocks read back.
#include "kernels.h"
#include "kv_q4.h"

namespace nnchip
{
	namespace
	{
		constexpr int kWaves = 4; // wavefronts per work-group, a record each

		// Half a block of one row: 16 codes, and the block's s and z.
		struct half_block
		{
			uint32_t code[2]; // columns 8 n .. 8 n + 7 of the half in nibbles, n = 0, 1
			uint32_t sz; // s in the low half, z in the high one
		};

		__device__ __forceinline__ float finite(float x)
		{
			return x == x ? fminf(fmaxf(x, -kQ4Max), kQ4Max) : 0.0f;
		}

		// Lanes l and l + 32 hold the two halves of a block.
		__device__ __forceinline__ half_block quantise(const float* src, bool real)
		{
			float x[16];
#pragma unroll
			for (int j = 0; j < 4; ++j)
			{
				const float4 v = real ? reinterpret_cast<const float4*>(src)[j] : float4{0, 0, 0, 0};
				x[4 * j] = finite(v.x);
				x[4 * j + 1] = finite(v.y);
				x[4 * j + 2] = finite(v.z);
				x[4 * j + 3] = finite(v.w);
			}
			float lo = x[0], hi = x[0];
#pragma unroll
			for (int j = 1; j < 16; ++j)
			{
				lo = fminf(lo, x[j]);
				hi = fmaxf(hi, x[j]);
			}
			lo = -max_with_other_half(-lo);
			hi = max_with_other_half(hi);
			// The product rounded to fp32 before it is rounded to fp16: the compiler
			// would make one instruction of both, which rounds once.
			float step = (hi - lo) * (1.0f / 15.0f);
			asm("" : "+v"(step));
			const _Float16 s = static_cast<_Float16>(step), z = static_cast<_Float16>(lo);
			const float sf = static_cast<float>(s), zf = static_cast<float>(z);
			half_block b{};
			// (the quotient itself, not a product with 1 / s: a code is defined by it;
			// s by a product with 1 / 15, as nnc's 4-bit weights form theirs)
#pragma unroll
			for (int j = 0; j < 16; ++j)
			{
				const float c = sf > 0.0f ? fminf(fmaxf(rintf((x[j] - zf) / sf), 0.0f), 15.0f) : 0.0f;
				b.code[j / 8] |= static_cast<uint32_t>(c) << (4 * (j % 8));
			}
			b.sz = as_u32(f16x2{s, z});
			return b;
		}

		// The same from the interchange form: elements i and i + 16 in byte i.
		__device__ __forceinline__ half_block raw_half(const unsigned char* src, int half, bool real)
		{
			half_block b{};
			if (!real) return b;
			const uint32_t* w = reinterpret_cast<const uint32_t*>(src); // (kQ4RawBlock is a multiple of 4)
			b.sz = w[0];
#pragma unroll
			for (int n = 0; n < 2; ++n)
#pragma unroll
				for (int j = 0; j < 8; ++j)
				{
					const int i = 8 * n + j;
					b.code[n] |= ((w[1 + i / 4] >> (8 * (i % 4) + 4 * half)) & 15u) << (4 * j);
				}
			return b;
		}

		// Rows pos0 .. pos0 + n_tok - 1 into records, a wavefront per (row group,
		// block): lane l quantises half l / 32 of row l % 32. A row of the group
		// holds at most one position of the batch (n_tok <= rows); where the batch
		// fills the ring and begins inside a group, that group holds its first
		// and its last positions. K's words belong to one row each; V's hold eight
		// rows, so a group of which only some rows are written keeps the others'
		// nibbles. One wavefront writes a record, so nothing else does meanwhile.
		// Bound: HBM (4 bytes an element read, 0.625 written: 4096 rows of 1024, 38.8 MB
		// in 11.3 us, 3.4 TB/s, the read of their values 9); one row: a load, the
		// quotients and a store, one after the other (6 us; with the old nibbles loaded
		// ahead of the quotients 0.5 more).
		template <bool RAW>
		__global__ __launch_bounds__(64 * kWaves) void append_q4_kernel(unsigned char* recs, const void* k_rows,
		                                                                const void* v_rows, int rows, int kv_dim, int pos0,
		                                                                int n_tok, int n_groups)
		{
			__shared__ uint32_t s_code[kWaves][32][5]; // a row's 32 V codes (and a word against bank conflicts)
			__shared__ uint32_t s_sz[kWaves][32];
			const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
			const int blocks = kv_dim / kQ4Block, row_groups = rows / kQ4Rows;
			const long long item = static_cast<long long>(blockIdx.x) * kWaves + wave;
			const bool live = item < static_cast<long long>(n_groups) * blocks;
			const int gi = live ? static_cast<int>(item / blocks) : 0, blk = live ? static_cast<int>(item % blocks) : 0;
			const int pos_group = pos0 / kQ4Rows + gi; // (fewer than row_groups after the first)
			unsigned char* rec = recs + (static_cast<size_t>(pos_group % row_groups) * blocks + blk) * kQ4Record;

			const int row = lane & 31, half = lane >> 5;
			// The batch's token in this row: 64 bits, since the position behind a
			// ring's wrap may pass the largest int.
			long long t = static_cast<long long>(pos_group) * kQ4Rows + row - pos0;
			if (t < 0) t += rows;
			const bool real = live && t < n_tok;
			half_block k, v;
			if constexpr (RAW)
			{
				const size_t at = (static_cast<size_t>(real ? t : 0) * blocks + blk) * kQ4RawBlock;
				k = raw_half(static_cast<const unsigned char*>(k_rows) + at, half, real);
				v = raw_half(static_cast<const unsigned char*>(v_rows) + at, half, real);
			}
			else
			{
				const size_t at = static_cast<size_t>(real ? t : 0) * kv_dim + blk * kQ4Block + 16 * half;
				k = quantise(static_cast<const float*>(k_rows) + at, real);
				v = quantise(static_cast<const float*>(v_rows) + at, real);
			}
			if (real)
			{
#pragma unroll
				for (int n = 0; n < 2; ++n) // quarter 2 half + n of the columns
					*reinterpret_cast<uint32_t*>(rec + 16 * (16 * (2 * half + n) + (row & 15)) + 4 * (row >> 4)) = k.code[n];
				if (half == 0)
					*reinterpret_cast<uint32_t*>(rec + kQ4KScales + 8 * (row & 15) + 4 * (row >> 4)) = k.sz;
			}
			s_code[wave][row][2 * half] = v.code[0];
			s_code[wave][row][2 * half + 1] = v.code[1];
			if (half == 0) s_sz[wave][row] = v.sz;
			const uint32_t written = static_cast<uint32_t>(__ballot(real)); // bit: row (lanes 0 .. 31)
			wave_sync();
			if (!live || written == 0) return; // (whole wavefronts; no barrier follows)

			// V: lane (g, i) makes the words of columns i and 16 + i for its eight rows.
			const int g = lane >> 4, i = lane & 15;
			uint32_t keep = 0; // nibbles of rows not in the batch
#pragma unroll
			for (int n = 0; n < 8; ++n)
				if (!((written >> (4 * g + (n & 3) + 16 * (n >> 2))) & 1)) keep |= 15u << (4 * n);
			u32x2* vw = reinterpret_cast<u32x2*>(rec + 16 * lane + 8);
			u32x2 w = {0, 0};
			if (keep != 0) w = *vw & u32x2{keep, keep};
#pragma unroll
			for (int n = 0; n < 8; ++n)
			{
				const int r = 4 * g + (n & 3) + 16 * (n >> 2);
				if (!((written >> r) & 1)) continue;
				w.x |= ((s_code[wave][r][i >> 3] >> (4 * (i & 7))) & 15u) << (4 * n);
				w.y |= ((s_code[wave][r][2 + (i >> 3)] >> (4 * (i & 7))) & 15u) << (4 * n);
			}
			if (keep != 0xffffffffu) *vw = w;
			if (lane < 32 && (written >> lane) & 1) // row `lane`: its s and z, a half each
			{
				const int rg = (lane >> 2) & 3, r = lane & 3, hi = lane >> 4;
				uint16_t* sv = reinterpret_cast<uint16_t*>(rec + kQ4VScales + 32 * rg);
				sv[2 * r + hi] = static_cast<uint16_t>(s_sz[wave][lane] & 0xffffu);
				sv[8 + 2 * r + hi] = static_cast<uint16_t>(s_sz[wave][lane] >> 16);
			}
		}

		// Rows row0 .. row0 + n_rows - 1: their values in F32, or (RAW) their
		// blocks in the interchange form. A wavefront per record.
		template <bool RAW>
		__global__ __launch_bounds__(64 * kWaves) void read_q4_kernel(const unsigned char* recs, void* k_out, void* v_out,
		                                                              int kv_dim, int row0, int n_rows, int n_groups)
		{
			__shared__ uint32_t s_code[kWaves][32][5];
			const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
			const int blocks = kv_dim / kQ4Block;
			const long long item = static_cast<long long>(blockIdx.x) * kWaves + wave;
			if (item >= static_cast<long long>(n_groups) * blocks) return; // (whole wavefronts; no barrier follows)
			const int group = row0 / kQ4Rows + static_cast<int>(item / blocks), blk = static_cast<int>(item % blocks);
			const unsigned char* rec = recs + (static_cast<size_t>(group) * blocks + blk) * kQ4Record;
			const int g = lane >> 4, i = lane & 15;
			const u32x4 w = *reinterpret_cast<const u32x4*>(rec + 16 * lane);
			const u32x2 ksz = *reinterpret_cast<const u32x2*>(rec + kQ4KScales + 8 * i);
			const u32x4 vs = *reinterpret_cast<const u32x4*>(rec + kQ4VScales + 32 * g);
			const u32x4 vz = *reinterpret_cast<const u32x4*>(rec + kQ4VScales + 32 * g + 16);
			const int first = group * kQ4Rows - row0; // the group's first row, in the output
			const q4_masks masks;
			if constexpr (!RAW)
			{
				if (k_out)
#pragma unroll
					for (int t = 0; t < 2; ++t)
					{
						const int r = first + 16 * t + i;
						const f16x8 x = q4_k(t ? w.y : w.x, t ? ksz.y : ksz.x, masks);
						if (r < 0 || r >= n_rows) continue;
						float4* dst = reinterpret_cast<float4*>(static_cast<float*>(k_out) + static_cast<size_t>(r) * kv_dim +
						                                        blk * kQ4Block + 8 * g);
						// (register j holds nibbles j and j + 4)
						dst[0] = float4{static_cast<float>(x[0]), static_cast<float>(x[2]), static_cast<float>(x[4]), static_cast<float>(x[6])};
						dst[1] = float4{static_cast<float>(x[1]), static_cast<float>(x[3]), static_cast<float>(x[5]), static_cast<float>(x[7])};
					}
				if (v_out)
#pragma unroll
					for (int t = 0; t < 2; ++t)
					{
						const f16x8 x = q4_v(t ? w.w : w.z, vs, vz, masks);
						float* dst = static_cast<float*>(v_out) + blk * kQ4Block + 16 * t + i;
#pragma unroll
						for (int n = 0; n < 8; ++n)
						{
							const int r = first + 4 * g + (n & 3) + 16 * (n >> 2);
							if (r >= 0 && r < n_rows) dst[static_cast<size_t>(r) * kv_dim] = static_cast<float>(x[2 * (n & 3) + (n >> 2)]);
						}
					}
			}
			else
			{
				// K's words hold a row's columns already; V's go through LDS.
				auto put = [&](void* out, int row, uint32_t sz)
				{
					// lanes of (row, 4 words): each row's codes as s_code[row][0 .. 3]
					const int r = first + row;
					if (!out || r < 0 || r >= n_rows) return;
					uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(out) +
					                                            (static_cast<size_t>(r) * blocks + blk) * kQ4RawBlock);
					dst[0] = sz;
#pragma unroll
					for (int b = 0; b < 4; ++b) // bytes 4 b .. 4 b + 3: elements of both halves
					{
						uint32_t o = 0;
#pragma unroll
						for (int j = 0; j < 4; ++j)
						{
							const int e = 4 * b + j;
							const uint32_t lo = (s_code[wave][row][e >> 3] >> (4 * (e & 7))) & 15u;
							const uint32_t hi = (s_code[wave][row][2 + (e >> 3)] >> (4 * (e & 7))) & 15u;
							o |= (lo | (hi << 4)) << (8 * j);
						}
						dst[1 + b] = o;
					}
				};
				s_code[wave][i][g] = w.x;
				s_code[wave][16 + i][g] = w.y;
				wave_sync();
				if (lane < 32)
				{
					const uint32_t sz = reinterpret_cast<const uint32_t*>(rec + kQ4KScales)[2 * (lane & 15) + (lane >> 4)];
					put(k_out, lane, sz);
				}
				wave_sync();
				for (int j = lane; j < 32 * 5; j += 64) s_code[wave][j / 5][j % 5] = 0;
				wave_sync();
#pragma unroll
				for (int n = 0; n < 8; ++n)
				{
					const int r = 4 * g + (n & 3) + 16 * (n >> 2);
					atomicOr(&s_code[wave][r][i >> 3], ((w.z >> (4 * n)) & 15u) << (4 * (i & 7)));
					atomicOr(&s_code[wave][r][2 + (i >> 3)], ((w.w >> (4 * n)) & 15u) << (4 * (i & 7)));
				}
				wave_sync();
				if (lane < 32)
				{
					const uint16_t* sv = reinterpret_cast<const uint16_t*>(rec + kQ4VScales + 32 * ((lane >> 2) & 3));
					const int at = 2 * (lane & 3) + (lane >> 4);
					put(v_out, lane, sv[at] | (static_cast<uint32_t>(sv[8 + at]) << 16));
				}
			}
		}

		// Values of a BF16 or F32 buffer's rows, F32.
		__global__ __launch_bounds__(256) void read_rows_kernel(const void* K, const void* V, float* k_out, float* v_out,
		                                                       size_t first, size_t n, bool bf16)
		{
			for (size_t i = blockIdx.x * static_cast<size_t>(256) + threadIdx.x; i < n; i += static_cast<size_t>(gridDim.x) * 256)
			{
				if (k_out)
					k_out[i] = bf16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(K)[first + i]) : static_cast<const float*>(K)[first + i];
				if (v_out)
					v_out[i] = bf16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(V)[first + i]) : static_cast<const float*>(V)[first + i];
			}
		}

		unsigned work_groups(int n_groups, int kv_dim)
		{
			return static_cast<unsigned>((static_cast<long long>(n_groups) * (kv_dim / kQ4Block) + kWaves - 1) / kWaves);
		}
	}

	void launch_append_q4(void* recs, const void* k_rows, const void* v_rows, int rows, int kv_dim, int pos0, int n_tok,
	                      bool raw, hipStream_t stream)
	{
		const int touched = static_cast<int>((static_cast<long long>(pos0) + n_tok - 1) / kQ4Rows - pos0 / kQ4Rows + 1);
		const int n_groups = touched < rows / kQ4Rows ? touched : rows / kQ4Rows;
		const dim3 grid(work_groups(n_groups, kv_dim));
		if (raw)
			append_q4_kernel<true><<<grid, 64 * kWaves, 0, stream>>>(static_cast<unsigned char*>(recs), k_rows, v_rows, rows,
			                                                        kv_dim, pos0, n_tok, n_groups);
		else
			append_q4_kernel<false><<<grid, 64 * kWaves, 0, stream>>>(static_cast<unsigned char*>(recs), k_rows, v_rows, rows,
			                                                         kv_dim, pos0, n_tok, n_groups);
	}

	void launch_read_q4(const void* recs, void* k_out, void* v_out, int kv_dim, int row0, int n_rows, bool raw,
	                    hipStream_t stream)
	{
		const int n_groups = (row0 + n_rows - 1) / kQ4Rows - row0 / kQ4Rows + 1;
		const dim3 grid(work_groups(n_groups, kv_dim));
		if (raw)
			read_q4_kernel<true><<<grid, 64 * kWaves, 0, stream>>>(static_cast<const unsigned char*>(recs), k_out, v_out, kv_dim,
			                                                      row0, n_rows, n_groups);
		else
			read_q4_kernel<false><<<grid, 64 * kWaves, 0, stream>>>(static_cast<const unsigned char*>(recs), k_out, v_out, kv_dim,
			                                                       row0, n_rows, n_groups);
	}

	void launch_read_rows(const void* K, const void* V, float* k_out, float* v_out, size_t first, size_t n, bool bf16,
	                      hipStream_t stream)
	{
		const size_t wg = (n + 255) / 256;
		read_rows_kernel<<<dim3(static_cast<unsigned>(wg < 4096 ? wg : 4096)), 256, 0, stream>>>(K, V, k_out, v_out, first, n, bf16);
	}
}
