// The kernels of attn_scored.hpp for head_dim 96.
#define MTP_SCORED_DH 96
#include "attn_scored.hpp"
