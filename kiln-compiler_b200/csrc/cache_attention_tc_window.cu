// Attention of drafted tokens over a paged K/V cache, to a sliding window and a few first tokens: the tiles of 128 query rows.  (A file of its own because files are
// compiled side by side.)
#define KB200_WINDOW
#include "cache_attention_tc.cu"
