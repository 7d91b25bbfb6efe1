// C entry points to the order of the many-row attention kernel's units, for
// tests without a GPU.
#include "kv_tile_order.h"

using shield::kv::TileOrder;

extern "C" {

TileOrder *order_new(int32_t nb, int32_t wide, int32_t clean, uint32_t ring) {
    auto *o = new TileOrder;
    o->set(nb, wide != 0, clean, ring);
    return o;
}
void order_delete(TileOrder *o) { delete o; }
int32_t order_ahead(const TileOrder *o) { return o->ahead; }
int32_t order_lead(const TileOrder *o) { return o->lead; }
int32_t order_two(const TileOrder *o) { return o->two(); }
uint32_t order_key_slot(const TileOrder *o, int32_t b) { return o->key_slot(b); }
uint32_t order_value_slot(const TileOrder *o, int32_t b) { return o->value_slot(b); }
int32_t order_blocks_of(const TileOrder *o, int32_t tile) { return o->blocks_of(tile); }
int32_t order_first_block(const TileOrder *o, int32_t tile) { return o->first_block(tile); }
int32_t order_block_step(const TileOrder *o) { return o->block_step(); }
int32_t order_looker(const TileOrder *o, int32_t tile) { return o->looker(tile); }
int32_t order_says_values_here(const TileOrder *o) { return o->says_values_here(); }
int32_t order_frees_queries(const TileOrder *o, int32_t tile) { return o->frees_queries(tile); }
int32_t values_here() { return shield::kv::VALUES_HERE; }
int32_t queries_free() { return shield::kv::QUERIES_FREE; }

}  // extern "C"
