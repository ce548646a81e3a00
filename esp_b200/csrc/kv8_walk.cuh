// The way of the row threads of attn_prefill_kv8.cu through a block's items, and where they meet.  What they compute is passed in, so that
// the way can also be gone on the CPU, with waits that run out.
//
// The row threads are two groups.  Of an item of two tiles each group has one, and the threads of a row meet within their group; of
// an item of one tile both have a share, and the threads of a row meet across the groups.  Waits are bounded, but a meeting is a named
// barrier and has no limit: whoever may be waited for has to come to it, also when a wait of its own has run out.
//   * Who fails in an item comes to that item's meeting all the same and says so, and all that it meets leave with it.
//   * In an item of two tiles that is its own group alone.  The other group may have come through, and would wait for it at the next
//     item of one tile: so whoever leaves an item of two tiles comes to that meeting, too, where the other group learns of it.
#pragma once

#ifdef __CUDACC__
#define KV8_WALK_FN __device__ __forceinline__
#else
#define KV8_WALK_FN inline
#endif

// ``open(round)``: makes the block's item of that round the current one; false: there is none.  ``two_tiles()``: of the current
// item.  ``work()``: false where a wait has run out.  ``meet(across, ok)``: whether all that meet are ok.  ``finish()``: what follows
// the meeting.  Returns false to threads that have left early.
template <typename Open, typename TwoTiles, typename Work, typename Meet, typename Finish>
KV8_WALK_FN bool kv8_walk_items(const Open& open, const TwoTiles& two_tiles, const Work& work, const Meet& meet, const Finish& finish) {
    for (int round = 0; open(round); round++) {
        const bool ok = work();
        if (meet(!two_tiles(), ok)) {
            finish();
            continue;
        }
        if (two_tiles()) {
            while (open(++round)) {
                if (two_tiles()) continue;
                meet(true, false);
                break;
            }
        }
        return false;
    }
    return true;
}
