// Kernel arguments of the calls on a cache of latent vectors (latent.h, latent_append.h).
#pragma once
#include "decode_fp8.h"
#include "latent_plan.h"
#include "rotary.h"

namespace fa {

constexpr int kLatentKeys = 64;  // keys of a tile: two runs of 32, each in one page

struct LatentArgs {
  DecodeArgs d;  // the partition (Hkv = rt = 1, tiles of 32 keys), lengths, page table, windows, workspace, o, lse
  int rt;        // row blocks of a batch row
  bool near;     // where they run (latent_place)
  const uint16_t* cache;  // (num_pages, page_size, L + R)
  const void *q, *qr;     // bf16; element strides of (row, head, query)
  long long qsb, qsh, qst, rsb, rsh, rst;
};

struct LatentAppendArgs {
  const void *latent, *rope;  // (B, T, L), (B, T, R) bf16; element strides of (row, token)
  long long lsb, lst, rsb, rst;
  uint16_t* cache;            // (num_pages, page_size, L + R)
  const int *page_table, *kv_lens, *new_lens;
  int page_size, max_pages, num_pages, B, T, L, R;
  const double* freq;         // null: not turned
  int n, interleaved;
  float scale;
  int units;                  // 16-element units of a token
  int kv_blocks;              // workgroups of this part
  RotaryArgs q;
};

}  // namespace fa
