// kvcache_tiles.h -- launching the attention kernel for many query rows.
#ifndef KVCACHE_TILES_H
#define KVCACHE_TILES_H

#include "kvcache_device.h"

// 16-bit types; `groups` workgroups: one for each item and KV head of its block (of kHeadBlock, or all of them if they are fewer).  `a.items` are tile items.
__attribute__((visibility("hidden"))) int kvm_launch_tiles(const kvc::AttnArgs &a, int dtype, int source, uint32_t groups,
                                                           hipStream_t stream);

#endif  // KVCACHE_TILES_H
