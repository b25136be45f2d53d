// The 4-bit key-value cache: where its bytes lie, and how a row of 16-bit numbers becomes codes and back.
//
// A row (one token, one kv head; hd numbers x of the model's 16-bit type) is held as
//   low  = min x                       a value of the row, so 16 bits hold it exactly
//   s    = (max x - low) / 15          in fp32, then rounded UP to 16 bits: rounded to the nearest, 15 s could end short of the largest value
//                                      (the number below where low + 15 s would round to an infinity)
//   code = rint((x - low) / s)         0..15 (all 0 where s is 0); differences and quotients in fp32, ties to the even code
// and stands for low + s * code: no value of a row is off by more than s / 2.  A row with an infinity or NaN in it, or whose range is no
// finite fp32 number, has s = low = NaN and reads back as NaN: codes themselves are always finite, so what a product of codes has to keep
// out of masked places is the two numbers of a row alone.
//
// Sixteen tokens of one kv head are a group of 16 (hd + 8) bytes, and a block of block_size tokens is block_size / 16 of them in a row:
// [num_blocks][KV][block_size / 16][group].  A group is one contiguous piece whatever the block size, so a tile of keys is fetched by as
// many bulk copies as it has blocks:
//   key codes   [16][hd / 2]   the rows in the order 0 4 1 5 2 6 3 7 8 12 9 13 10 14 11 15: rows as an mma.m16n8k16 A operand then leave keys
//                              (t, t + 4), (t + 8, t + 12) with thread t of a quad, which are four rows of the values' bank pattern below
//   value codes [16][hd / 2]   in token order; for hd = 128 the two 32-byte halves of tokens 2, 3, 6, 7, 10, 11, 14, 15 are exchanged,
//                              so that four neighbouring rows read 8 bytes a lane touch every bank once
//   (s, low) of the keys [16], (s, low) of the values [16]   two 16-bit numbers each
// A 32-bit word has eight codes, d = 8 j .. 8 j + 7 of word j: nibble p is d = 8 j + 2 p and nibble p + 4 is d = 8 j + 2 p + 1, so that
// (w >> 4 p) & 0x000f000f is the pair (2 p, 2 p + 1) in the two halves of a register.
#pragma once
#include "common.cuh"

namespace kge {
namespace kv4 {

__host__ __device__ constexpr int group_bytes(int hd) { return 16 * (hd + 8); }
__host__ __device__ constexpr int key_row(int token) { return (token & 8) | ((token & 3) << 1) | ((token >> 2) & 1); }      // place of a token's key codes
__host__ __device__ constexpr int key_token(int row) { return (row & 8) | ((row & 1) << 2) | ((row >> 1) & 3); }            // and back
// word of a value row that holds dimensions 8 j .. 8 j + 7
__host__ __device__ constexpr int value_word(int hd, int token, int j) { return hd == 128 ? j ^ ((token & 2) << 2) : j; }

}  // namespace kv4
}  // namespace kge
