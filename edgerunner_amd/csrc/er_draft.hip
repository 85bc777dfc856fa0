// er_draft.hip -- what a step needs that drafts tokens, streams without end or
// answers under rules: attention over the 8-bit cache under masks (er_kv8_attn.hip
// once more), acceptance of drafts, rules on logits and the choice.  A code
// object of its own, compiled beside er_kv8.hip's.
#define ER_KV8_MASKED
#include "er_kv8.hip"
#include "er_draft.h"
#include "er_kv8_few.hip"
#include "er_accept.hip"
#include "er_choose.hip"
