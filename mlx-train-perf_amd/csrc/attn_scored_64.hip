// The kernels of attn_scored.hpp for head_dim 64.
#define MTP_SCORED_DH 64
#include "attn_scored.hpp"
