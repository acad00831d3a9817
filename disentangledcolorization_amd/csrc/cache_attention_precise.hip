// cache_attention_precise.hip - the forms of many and large rows of cache_attention.hip with weights of fp32 precision (REST), in a translation unit of their own:
// the two are the longest steps of a build, and compile side by side.
#define DISCO_CACHE_PRECISE
#include "cache_attention.hip"
