// How the dX product of distill.hip cuts a range of the vocabulary into splits: integer arithmetic alone, which the device
// evaluates (one k a lane) and a host compiler can check.
#pragma once
#ifdef __HIP__
#define DX_FN __host__ __device__ __forceinline__
#else
#define DX_FN inline
#endif

namespace cvae {

constexpr int DT_DX_BLOCKS = 256, DT_DX_MOST = 1024;

// k splits of `stages` stages for each of `tiles` tiles: `k - longer` of `size` stages, then `longer` of more.  `d`: a tile of dW
// in stages, `dwtiles` of them; `spare`: use the CUs that dW's last round leaves.  No tiles (no live row): nothing is spared.
struct DxSplit {
  int size, longer, cost;
};
DX_FN DxSplit dx_split(int k, int tiles, int stages, int d, int dwtiles, bool spare) {
  const int items = tiles * k, rounds = (dwtiles + DT_DX_BLOCKS - 1) / DT_DX_BLOCKS;
  int spared = 0;
  if (spare && tiles > 0 && items <= DT_DX_BLOCKS) {
    spared = (rounds * DT_DX_BLOCKS - dwtiles) / tiles;
    spared = spared < k ? spared : k;
  }
  int more = 0;
  if (spared > 0) {
    more = (stages - 4 * k) / spared;
    more = more < d ? more : d;
    more = more > 0 ? more : 0;
  }
  DxSplit r;
  r.size = more > 0 ? (stages - spared * more) / k : (stages + k - 1) / k;
  r.longer = more > 0 ? spared : 0;
  r.cost = 0x7fffffff;
  if (k == 1 || (items <= DT_DX_MOST && k * 4 <= stages)) {
    const int c = ((items + DT_DX_BLOCKS - 1) / DT_DX_BLOCKS) * (r.size + 14);
    r.cost = (c < 0x1ffffff ? c : 0x1ffffff) * 64 + (k - 1);
  }
  return r;
}

// partial tiles that any number of live rows can ask for: one split of every tile, or more of fewer
DX_FN int dx_partial_tiles(int tiles, int stages) {
  const int k = stages / 4 < 1 ? 1 : (stages / 4 > 64 ? 64 : stages / 4);
  const long many = (long)tiles * k < DT_DX_MOST ? (long)tiles * k : DT_DX_MOST;
  return tiles > many ? tiles : (int)many;
}

struct Splits {
  int n, even, size, most;                                        // splits; the first `even` of `size` stages, the others of `most`
  DX_FN int begin(int s) const { return s <= even ? s * size : even * size + (s - even) * most; }
};
DX_FN Splits dx_splits_of(int k, int size, int longer, int stages) {
  Splits r;
  r.n = k;
  r.size = size;
  r.even = k - longer;
  r.most = longer ? (stages - r.even * size + longer - 1) / longer : 0;
  return r;
}

}  // namespace cvae
