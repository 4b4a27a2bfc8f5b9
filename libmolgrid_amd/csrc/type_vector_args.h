// Arguments of the learned type vectors' launches, as the entry points fill them in.  Plain data: what
// the kernels compute with is in element_types.h.
#ifndef LIBMOLGRID_AMD_TYPE_VECTOR_ARGS_H_
#define LIBMOLGRID_AMD_TYPE_VECTOR_ARGS_H_

#include <stdint.h>

namespace mg {

// The tokens of a call: type indices and the table whose rows they name.
struct TokenArg {
  const void* index;  // ntokens indices of kind MG_INDEX_*
  int ntokens, nrows, channels;
  int dtype;  // MG_FLOAT32, ...: of the table and the type vectors
  int index_kind;
};

// A layer norm: rows of `channels` elements.
struct NormArg {
  int nrows, channels;
  int dtype, param_dtype;
  const void* weight;  // channels elements, or nullptr for ones
  float eps;
};

// Which elements a call drops.  Element e of the flattened array takes half e % 8 (low half of a
// word first) of the words of counter (e / 8, offset) under key seed, and is kept where that half
// is at least `limit`; `factor` multiplies what is kept.  16 bits an element: one counter serves
// eight of them, so that the generator (about 60 vector instructions a wave and counter, counted in
// the encoder) stays behind the memory that dropout runs beside.
struct DropArg {
  uint32_t limit;         // round(65536 p): 0 keeps everything, 65536 nothing
  float factor;           // 65536 / (65536 - limit), 0 when nothing is kept
  uint64_t seed, offset;
  const uint64_t* state;  // device: two numbers that are added to them, or nullptr
};

// Which rows of a table tokens name: by bits (of up to 32 rows, in `count` words that are ORed
// together), or by where the sorted tokens of a row begin and end.
struct NamedRows {
  const uint32_t* words;
  int count;
  const int32_t* start;   // or nullptr
};

}  // namespace mg

#endif
