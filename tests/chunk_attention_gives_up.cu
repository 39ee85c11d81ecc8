// Attention of new tokens on tcgen05 whose tile CT_STRAY of values (a flag of the compiler) is waited for in vain, for a short while.
#define TC_WAIT_LIMIT (1u << 14)
#define TC_DRAIN_LIMIT (1u << 14)
#include "attention_chunks_tc.cu"
