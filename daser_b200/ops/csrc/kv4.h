// Host-visible parameter block of the 4-bit paged pool (mirrored with ctypes in daser_b200/ops/_lib.py).
#pragma once
#include <stdint.h>

#include "kv_paged.h"

// A page of DASER_KV4_TOKENS tokens of one KV head is one record of DASER_KV4_RECORD bytes:
//   [0, 1024)     K codes   [token][64]: two dims a byte, the even dim in the low half
//   [1024, 2048)  V codes   [token / 8][group][token % 8][8]
//   [2048, 2176)  K scales  [token][group]
//   [2176, 2304)  V scales  [token / 8][group][token % 8]
// (group: 16 consecutive dims).  A page is one contiguous run, so that a reader fetches it with a single
// bulk copy; K rows are dim-contiguous because scores contract over dims, V is grouped by tokens because
// the output contracts over tokens.  Every (token, K|V) row is made of bytes of its own, so that tokens can be
// written by different threads, or steps, without a read-modify-write.
#define DASER_KV4_TOKENS 16
#define DASER_KV4_DIM 128
#define DASER_KV4_RECORD 2304
#define DASER_KV4_V 1024
#define DASER_KV4_KS 2048
#define DASER_KV4_VS 2176

// Record (layer, block, head_local) of rank r starts at records[r] + layer * stride_layer + block * stride_block +
// head_local * stride_head (strides in bytes, multiples of 16; bases 16-byte aligned).
typedef struct {
  uint8_t* records[DASER_MAX_RANKS];
  int64_t stride_layer;
  int64_t stride_block;
  int64_t stride_head;
  int32_t num_layers;
  int32_t num_blocks;       // blocks per layer in every rank's pool (bounds check)
  int32_t n_ranks;          // tensor-parallel degree
  int32_t heads_per_rank;   // KV heads each rank keeps (1 when n_ranks > num_kv_heads)
} DaserKV4Pool;
