// The 4-bit K/V cache: its block format, where a block's codes lie in device
// memory, and the device helpers of the kernels that write and read it.
//
// Format. A block is 32 consecutive elements of a row (nnc's own 4-bit block,
// reference nn_ops.h:138-142, along the head instead of a weight row). With lo
// and hi its least and largest element,
//   s = f16((hi - lo) r), r = 1 / 15 in fp32,  z = f16(lo),
//   c = rint((x - z) / s) within 0 .. 15 (0 where s is 0),
// and the element stands for f16(c s + z), rounded once: one fused multiply-add
// in fp16, which is what the attention kernels feed to the matrix cores, so
// they lose nothing against the format's own definition. s and z are fp16 and
// not BF16 as in the weights for that reason, and because a step of f16(lo) is
// then a 136th of s at most for a block whose elements lie on both sides of 0.
// Elements are brought within +-kQ4Max and NaN is taken as 0 first: every
// value of the cache is finite, so a masked row can never reach an output
// (0 x inf is NaN). 5 bits an element.
//
// Layout. Rows go in groups of 32 and columns in blocks of 32; a (group,
// block) pair is one record of kQ4Record bytes, records in [group][block] order.
// A record is what the 64 lanes of one wavefront read for 32 keys, in the
// operand order of v_mfma_f32_16x16x32_f16, so no lane moves anything to
// another:
//   byte 16 l, l = 16 g + i the lane (g = 0 .. 3, i = 0 .. 15):
//     words 0, 1: K of rows i and 16 + i, columns 8 g + n in nibble n (the A
//       operand of S^T = K Q^T: row i, k slots of quarter g);
//     words 2, 3: V of columns i and 16 + i, rows 4 g + r in nibble r and
//       16 + 4 g + r in nibble 4 + r, r = 0 .. 3 (the A operand of
//       O^T = V^T P^T, whose k slots are the rows whose weights lane l holds
//       after the score products);
//   byte 1024 + 8 i: (s, z) of K's rows i and 16 + i, a word each;
//   byte 1152 + 32 g: V's s of rows 4 g + r (low half) and 16 + 4 g + r (high
//     half) in word r, then z likewise.
// Nibbles n and n + 4 of a word become one register of two fp16, so k slot
// 2 r of a quarter is nibble r and slot 2 r + 1 nibble 4 + r.
#pragma once

#include "device_common.h"

namespace nnchip
{
	constexpr int kQ4Rows = 32, kQ4Block = 32; // rows of a group, columns of a block
	constexpr int kQ4Record = 1280; // bytes of a (group, block) pair, K and V
	constexpr int kQ4KScales = 1024, kQ4VScales = 1152; // byte offsets in a record
	// z + 15 s <= kQ4Max (1 + 2^-10) with s and z rounded up by half a step
	// each, which still rounds to a finite fp16 (the largest is 65504).
	constexpr float kQ4Max = 65280.0f;
	// A row of the interchange form (nnc_hip_kv_append, nnc_hip_kv_read): per
	// block s, z, then 16 bytes of codes, elements i and i + 16 in byte i.
	constexpr int kQ4RawBlock = 20;

	__device__ __forceinline__ f16x2 as_f16x2(uint32_t w) { return __builtin_bit_cast(f16x2, w); }
	__device__ __forceinline__ uint32_t as_u32(f16x2 h) { return __builtin_bit_cast(uint32_t, h); }

	// The eight codes of a word as fp16 whole numbers, nibbles r and r + 4 in
	// c[r]. A nibble ORed into the mantissa of 1024 is 1024 + c (in bits 0 .. 3)
	// or 1024 + 16 c (bits 4 .. 7), and both subtractions are exact: 13
	// operations for eight codes with the fused multiply-adds that follow (a
	// shift, four and-ors, four to remove the 1024, four to scale), where a
	// conversion per code takes 24.
	// (The and and the or are one instruction if neither constant is a literal:
	// q4_masks holds them in registers.)
	struct q4_masks
	{
		uint32_t low = 0x000f000fu, high = 0x00f000f0u, k1024 = 0x64006400u;
		__device__ __forceinline__ q4_masks() { asm("" : "+s"(low), "+s"(high), "+v"(k1024)); }
	};
	__device__ __forceinline__ void q4_codes(uint32_t w, const q4_masks& k, f16x2 c[4])
	{
		const uint32_t h = w >> 8;
		const f16x2 m1024 = {static_cast<_Float16>(-1024.0f), static_cast<_Float16>(-1024.0f)};
		const f16x2 m64 = {static_cast<_Float16>(-64.0f), static_cast<_Float16>(-64.0f)};
		const f16x2 s16 = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
		c[0] = as_f16x2((w & k.low) | k.k1024) + m1024;
		c[1] = __builtin_elementwise_fma(as_f16x2((w & k.high) | k.k1024), s16, m64);
		c[2] = as_f16x2((h & k.low) | k.k1024) + m1024;
		c[3] = __builtin_elementwise_fma(as_f16x2((h & k.high) | k.k1024), s16, m64);
	}

	// A K word's values: sz holds the row's (s, z).
	__device__ __forceinline__ f16x8 q4_k(uint32_t w, uint32_t sz, const q4_masks& k)
	{
		f16x2 c[4];
		q4_codes(w, k, c);
		const f16x2 h = as_f16x2(sz);
		const f16x2 s = {h.x, h.x}, z = {h.y, h.y};
		u32x4 r;
#pragma unroll
		for (int j = 0; j < 4; ++j) r[j] = as_u32(__builtin_elementwise_fma(c[j], s, z));
		return as_f16x8(r);
	}

	// A V word's values: s and z of its eight rows.
	__device__ __forceinline__ f16x8 q4_v(uint32_t w, const u32x4& s, const u32x4& z, const q4_masks& k)
	{
		f16x2 c[4];
		q4_codes(w, k, c);
		u32x4 r;
#pragma unroll
		for (int j = 0; j < 4; ++j) r[j] = as_u32(__builtin_elementwise_fma(c[j], as_f16x2(s[j]), as_f16x2(z[j])));
		return as_f16x8(r);
	}

	// The nibble order above: nibble n of a word is column (or row slot) n, and
	// register r of its values holds n = r and n = r + 4.
}
