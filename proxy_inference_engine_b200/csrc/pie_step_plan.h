// A ragged step's plan: one buffer of 32-bit words on the device, laid out by what its dimensions are (pie_ragged.cu writes it, pie_chunk_attn.cuh and
// the callers read it).  Nothing here is part of the public ABI but the words' order, which pie_step_plan_offsets tells.
#pragma once
#include "pie_internal.h"

namespace pie {

constexpr int kStepPage = 64;          // tokens of a page
constexpr int kStepMaxRequests = 4096; // the scans of a step's lengths are held in shared memory
constexpr int kStepMaxCtas = 192;      // CTAs that the attention's work is dealt out to, at most
constexpr int kStepTile = 128;         // rows of a query tile, keys of a key tile
constexpr int kStepPieceWords = 12;
constexpr int kStepRoom = 1024;        // what is added to a number of keys in 32 bits (a tile, an item's cost) is less

// One CTA's share of an item of attention: some of the key tiles of up to two query tiles of one key / value head of one request.  A query tile's rows are
// its tokens' query heads of that key / value head, token by token.
struct StepPiece {
  int row0, pos0, tokens;   // first row of the step, its position, live tokens
  int request, kv_head;
  int k0, k1;               // key tiles [k0, k1); none: nothing to do
  int first_cta, pieces;    // the CTA of the item's first piece, and how many CTAs share it
  int pages[2];             // of key tile k0
  int pad;
};
static_assert(sizeof(StepPiece) == 4 * kStepPieceWords, "read as three 16-byte words");

struct StepLayout {
  // offsets in words
  long long row_starts, contexts, sequences, positions, slots, block_table, logit_starts, logit_rows, draft_tokens, status, ranges, pieces, words;
  long long items;          // most items of attention
  int tile_tokens;          // tokens of a query tile
};

// Hq / Hkv <= 128
inline StepLayout step_layout(const pie_step_dims& d) {
  StepLayout l;
  long long at = 0;
  auto take = [&](long long n) { const long long p = at; at += (n + 3) / 4 * 4; return p; };   // (16-byte boundaries)
  l.row_starts = take(d.requests + 1LL);
  l.contexts = take(d.requests);
  l.sequences = take(d.rows);
  l.positions = take(d.rows);
  l.slots = take(d.rows);
  l.block_table = take((long long)d.requests * d.blocks);
  l.logit_starts = take(d.requests + 1LL);
  l.logit_rows = take(d.logit_rows);
  l.draft_tokens = take(d.logit_rows);
  l.status = take(kStepMaxCtas);
  l.ranges = take(2 * kStepMaxCtas);
  l.tile_tokens = kStepTile / (d.Hq / d.Hkv);
  l.items = (long long)d.Hkv * (d.rows / (2 * l.tile_tokens) + d.requests);
  l.pieces = take((l.items + kStepMaxCtas) * kStepPieceWords);
  l.words = at;
  return l;
}

int step_dims_status(const pie_step_dims* d);   // what is wrong with them, PIE_OK otherwise

}  // namespace pie
