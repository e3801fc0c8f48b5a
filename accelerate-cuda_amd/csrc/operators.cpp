// Operators on segments of rows: the products, the router, the combination and the 4-bit numbers of a layer of experts
// (operators/op_*.h), reached through acc_op_create and acc_exec_product_*, acc_exec_route*, acc_exec_combine*, acc_exec_micro_*.
//
// They are instances as the skeletons are: a few lines of definitions in front of an embedded header, compiled for the
// device's ISA by hiprtc through the kernel cache.  An instance is made for a kind and an element type; its variants (tile
// shapes, which way an operand lies, alignment) are compiled when a call first needs them.
#include <algorithm>
#include <cstring>
#include <exception>
#include <map>
#include <new>

#include "acc_internal.hpp"
#include "operators/op_args.h"

using acc::fail;

// no exception leaves an entry point: what is thrown below them is a failure to allocate host memory
#define ACC_OP_CATCH(who)                                                             \
  catch (const std::bad_alloc &) { return fail(ACC_ERR_OOM, "%s: out of host memory", who); } \
  catch (const std::exception &e) { return fail(ACC_ERR_INVALID, "%s: %s", who, e.what()); }

namespace {

struct OpVariant {
  std::shared_ptr<acc::CompileJob> job;
  hipModule_t module = nullptr;
  hipFunction_t fn = nullptr, fn2 = nullptr, fn3 = nullptr;
};

// what an instance was asked for
struct OpSpec {
  int kind = 0;
  int type = 0;                 // 0 float, 1 half, 2 bfloat16
  int choose = 0;
  bool normalise = true;
  int gate = 0;
  int group = 0;
  int groups = 1, keep = 1;
  float scale = 1.0f;
  int tile = -1;                // knob product.tile: the products' tile shape, for measurement
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

const char *const kKindName[] = {"product", "route", "combine", "micro", "", "recur", "grouped", "score"};
int type_bytes(int type) { return type == 0 ? 4 : 2; }

// ---- the variants of each kind ------------------------------------------------------

// product: tile shapes, in waves of 64 lanes.  Which a call takes is said at rows_tile and outer_tile.
struct ProductTile { int bm, bn, wm, wn; };
const ProductTile kProductTiles[] = {{32, 64, 2, 2}, {64, 64, 2, 2}, {64, 128, 2, 2}, {128, 128, 2, 2}, {256, 256, 2, 4}, {16, 32, 1, 4}, {16, 64, 1, 4}};
constexpr int kProductTileCount = 7, kLow = 0, kSquare = 1, kWide = 2, kMiddle = 3, kLarge = 4, kSkinny = 5;      // the last two: op_skinny.h
struct ProductVariant {
  int tile = 0;
  bool outer = false, b_fast = true, aligned = true;
  bool fours = true;            // 4 bits, in the form for a few rows: scales are whole words of four
  bool tiny = false;            // not aligned: a row is shorter than 16 bytes; 4 bits: it has fewer than four scales
  int index = 0;                // outer: whose rows an index names: 1 b's, 2 a's
  bool places = false;          // ... which a kernel in front has looked up
  uint32_t key() const { return (uint32_t)tile | (outer ? 16u : 0u) | (b_fast ? 32u : 0u) | (aligned ? 64u : 0u) | (uint32_t)index << 7 | (tiny ? 512u : 0u) | (places ? 2048u : 0u); }
};

std::string product_source(const OpSpec &sp, const ProductVariant &v)
{
  const ProductTile &t = kProductTiles[v.tile];
  char text[512];
  if (v.tile >= kSkinny) {
    std::snprintf(text, sizeof(text),
                  "#define OP_ELT %d\n#define OP_TYPE %d\n#define OP_BM %d\n#define OP_FN %d\n#include \"acc_hip_device.h\"\n#include \"op_skinny.h\"\n",
                  sp.type, sp.kind == ACC_OP_MICRO ? 3 : sp.type, t.bm, t.bn / 16);
    return text;
  }
  std::snprintf(text, sizeof(text),
                "#define OP_ELT %d\n#define OP_TYPE %d\n#define OP_BM %d\n#define OP_BN %d\n#define OP_WM %d\n#define OP_WN %d\n#define OP_OUTER %d\n"
                "#define OP_A_FAST %d\n#define OP_B_FAST %d\n#define OP_ALIGNED %d\n#define OP_INDEX %d\n#define OP_PLACES %d\n#define OP_TINY %d\n#include \"acc_hip_device.h\"\n#include \"op_product.h\"\n",
                sp.type, sp.kind == ACC_OP_MICRO ? 3 : sp.type, t.bm, t.bn, t.wm, t.wn, v.outer ? 1 : 0, v.outer ? 0 : 1, v.outer ? 0 : v.b_fast ? 1 : 0, v.aligned ? 1 : 0, v.index, v.places ? 1 : 0,
                v.tiny ? 1 : 0);
  return text;
}

constexpr int kRouteThreads = 1024, kRouteFewThreads = 256, kRouteTallThreads = 256, kRouteMaxExperts = 2048;
// route: how a token's logits are shared out
struct RouteVariant {
  int lanes = 1, per = 8, vec = 1, sels = 1;
  bool few = false;             // tokens that four waves take at once
  bool tall = false;            // a lane a token, or `halves` of them
  int halves = 1;
  int threads() const { return few ? kRouteFewThreads : kRouteThreads; }
  uint32_t key() const { return (uint32_t)lanes | (few ? 128u : 0u) | (uint32_t)per << 8 | (uint32_t)vec << 16 | (uint32_t)sels << 24 | (tall ? (halves == 1 ? 1u : halves == 2 ? 2u : 3u) << 30 : 0u); }
};

constexpr int64_t kRouteAlone = 8192;                // up to as many logits go to one workgroup, see route_block

// The form with a lane a token, or two or four that share its logits, is for up to eight choices and rows of 16 bytes or more.  us,
// bfloat16, eight chosen unless said.
// How many lanes: one for up to 64 experts, two for up to 128, four for more: with one, two, four, 65536 tokens of 64: 17, 20, 27; 4096
// of 128: 17, 14, 14; 16384 of 512: 51, 35, 28; Float32, whose keys are twice as long, up to 32: 65536 of 128: 57, 48, 53.
// From how many tokens on, the other form's time last:
//   up to 64 experts enough for a wave of 64 a SIMD: 65536 of 64: 17 and 25; 16384: 13 and 12
//   up to 256 from the second workgroup on: 65 tokens of 128: 10.3 and 13.0, of 256: 11.9 and 14.4; 4096 of 128: 12.0 and 14.8; two
//     chosen of 65 to 128: 9.8 to 10.7 and 9.9 to 11.1
//   up to 512, which the other form has eight a lane of: 65: 15.7 and 15.9, four chosen 14.3 and 13.4, one 13.5 and 11.5, one of 501
//     15.2 and 12.2; 4096, four chosen: 21.5 and 20.7; 6000: 22.0 and 23.4
//   up to 1024, sixteen a lane: 65 of 576: 19.0 and 35.8, one chosen 15.8 and 15.5; of 1024: 23.7 and 37.9, 19.8 and 17.7
//   beyond, in rows of whole chunks: 65 of 2048: 39.8 and 28.3; 4096: 67.9 and 58.5; 6000: 67.8 and 65.3, four chosen 63.3 and 61.0; 8192:
//     67.3 and 70.0; of 1104: 65: 27.3 and 23.6, 6000: 44.4 and 49.1; in other rows 65 of 2047: 44.8 and 40.9, one chosen 38.0 and 39.3;
//     of 1500, four: 32.1 and 33.6
//   Float32: 65536 of 128: 48 and 56; 16384 of 128: 27 and 20, of 512: 63 and 65
RouteVariant route_variant(const OpSpec &sp, int experts, bool aligned, int64_t tokens)
{
  RouteVariant v;
  const int epc = 16 / type_bytes(sp.type);
  while (v.lanes < 64 && v.lanes * v.per < experts) v.lanes *= 2;
  while (v.lanes * v.per < experts) v.per *= 2;
  v.vec = aligned && experts % epc == 0 ? epc : 1;
  v.sels = (sp.choose + v.lanes - 1) / v.lanes;
  // (8 tokens of 64: 5.1 us on the device, 5.6 with sixteen waves and the choices read back from memory)
  v.few = tokens > 0 && tokens * v.lanes <= kRouteFewThreads && tokens * experts <= kRouteAlone;
  const bool early = (experts > 64 && experts <= 256) || (experts > 512 && (experts <= 1024 || v.vec == 1));
  const int64_t from = sp.type == 0 ? (experts >= 256 ? 16384 : 65536) : early ? 65 : experts > 256 ? 5000 : 32768;      // (65: more than one workgroup)
  v.tall = experts >= epc && sp.choose <= 8 && tokens >= from && tokens * experts > kRouteAlone;
  if (v.tall) v.halves = experts <= (sp.type == 0 ? 32 : 64) ? 1 : experts <= 128 ? 2 : 4;
  return v;
}

std::string route_source(const OpSpec &sp, const RouteVariant &v)
{
  char text[512];
  std::snprintf(text, sizeof(text),
                "#define OP_ELT %d\n#define OP_LANES %d\n#define OP_PER %d\n#define OP_VEC %d\n#define OP_SELS %d\n#define OP_THREADS %d\n#define OP_TALL %d\n#define OP_HALVES %d\n#define OP_CHOOSE %d\n"
                "#include \"acc_hip_device.h\"\n#include \"op_route.h\"\n",
                sp.type, v.lanes, v.per, v.vec, v.sels, v.threads(), v.tall ? 1 : 0, v.halves, sp.choose);
  return text;
}

// Tokens of a workgroup: what its waves take at once or up to 64, and more where that were more than 256 workgroups, each of
// which reads the counts of all.  A single one places its slots itself, a launch less: 128 tokens of 16 experts take 6 us, in two
// 9; 256 of 64 16 and 9.
int route_block(const RouteVariant &v, int64_t tokens, int64_t experts)
{
  if (tokens * experts <= kRouteAlone) return (int)std::max<int64_t>(1, tokens);
  return (int)std::max<int64_t>(std::min(64, kRouteThreads / v.lanes), ceil_div(tokens, 256));
}

constexpr int kCombineSlots = 4;
// rows 0 anywhere, 1 aligned, 2 of fewer than eight elements
std::string combine_source(const OpSpec &sp, int rows)
{
  char text[256];
  std::snprintf(text, sizeof(text), "#define OP_ELT %d\n#define OP_ALIGNED %d\n#define OP_TINY %d\n#define OP_SLOTS %d\n#include \"acc_hip_device.h\"\n#include \"op_combine.h\"\n",
                sp.type, rows == 1 ? 1 : 0, rows == 2 ? 1 : 0, kCombineSlots);
  return text;
}

std::string pack_source(const OpSpec &sp)
{
  char text[128];
  std::snprintf(text, sizeof(text), "#define OP_ELT %d\n#include \"acc_hip_device.h\"\n#include \"op_pack.h\"\n", sp.type);
  return text;
}

std::string micro_source(const OpSpec &sp, bool aligned)
{
  char text[256];
  std::snprintf(text, sizeof(text), "#define OP_ELT %d\n#define OP_ALIGNED %d\n#include \"acc_hip_device.h\"\n#include \"op_micro.h\"\n", sp.type, aligned ? 1 : 0);
  return text;
}

// score: how a token's logits are shared out
struct ScoreVariant {
  int lanes = 4, per = 64;
  bool few = false;             // one workgroup, which places the slots, too
  int threads() const { return few ? kRouteFewThreads : 512; }
  int place_threads() const { return few ? kRouteFewThreads : kRouteThreads; }
  uint32_t key() const { return (uint32_t)lanes | (uint32_t)per << 8 | (few ? 1u << 16 : 0u); }
};
constexpr int kScoreSlice = 32;
// logits of a lane: a group, or a part of one
int64_t score_slice(const OpSpec &sp, int64_t experts, int lanes) { return ceil_div(experts / sp.groups, lanes / sp.groups); }
std::string score_source(const OpSpec &sp, const ScoreVariant &v)
{
  char text[512];
  std::snprintf(text, sizeof(text),
                "#define OP_ELT %d\n#define OP_LANES %d\n#define OP_PER %d\n#define OP_CHOOSE %d\n#define OP_ROW %d\n#define OP_FEW %d\n#define OP_THREADS %d\n"
                "#include \"acc_hip_device.h\"\n#include \"op_score.h\"\n",
                sp.type, v.lanes, v.per, sp.choose, 32, v.few ? 1 : 0, v.place_threads());
  return text;
}
ScoreVariant score_variant(const OpSpec &sp, int64_t experts, int64_t tokens)
{
  ScoreVariant v;
  v.few = tokens * experts <= kRouteAlone;
  v.lanes = std::max(v.lanes, sp.groups);
  // (32 logits a lane where that makes four waves a SIMD, fewer otherwise: what counts is how soon a token is done)
  while (v.lanes < 64 && (score_slice(sp, experts, v.lanes) > kScoreSlice || (tokens * v.lanes < 64 * 4096 && score_slice(sp, experts, v.lanes) > 8))) v.lanes *= 2;
  v.per = 8;
  while (v.per < score_slice(sp, experts, v.lanes)) v.per *= 2;
  return v;
}

// recur: a workgroup's tile is eight waves' rows of 64 words of channels.  Rows of a wave, which are held in registers: the
// gradient has twice as many arrays
struct RecurVariant {
  bool back = false, step = false;
  bool thin = false;            // rows of up to 64 channels of 16 bits: one a lane (and a row of one has no word of two)
  int rows = 32;                // of a wave: 8, 16 or (forward) 32
  int channels(int type) const { return thin ? 64 : 64 * (4 / type_bytes(type)); }
  uint32_t key() const { return (back ? 1u : 0u) | (step ? 2u : 0u) | (thin ? 4u : 0u) | (uint32_t)rows << 4; }
};
constexpr int kRecurWaves = 8;

// Rows of a wave.  512 tiles are on the device at once, two a compute unit; a tile takes about as long as its rows and sixteen more
// (what it waits for), eight where it has a compute unit for itself, and a state takes a fifth of a row to go on to the next tile of a
// long sequence.  us, with 8, 16 and 32 rows a wave: forward, bfloat16, 32768 x 2048: 156, 103, 89; 4096 x 2048: 25, 18, 19; 2048 x 2048:
// 15, 12, 17; 512 x 1024: 8, 10, 14; half, one sequence, 65536 x 64: 56, 33, 25; 16384 x 128: 23, 17, 18; Float32 9001 x 1001: 38, 36, 39; gradient,
// bfloat16, 32768 x 2048: 205, 170; 1024 x 1024: 12, 14.
int recur_rows(bool back, int64_t rows, int64_t strips)
{
  int best = 0;
  int64_t least = 0;
  for (int r : {32, 16, 8}) {
    if (back && r == 32) continue;
    const int64_t tiles = ceil_div(rows, (int64_t)kRecurWaves * r), groups = tiles * strips, cost = 5 * (groups <= 256 ? r + 8 : ceil_div(groups, 512) * (r + 16)) + tiles;
    if (best == 0 || cost < least) {
      best = r;
      least = cost;
    }
  }
  return best;
}
std::string recur_source(const OpSpec &sp, const RecurVariant &v)
{
  char text[256];
  std::snprintf(text, sizeof(text), "#define OP_ELT %d\n#define OP_GATE %d\n#define OP_BACK %d\n#define OP_STEP %d\n#define OP_THIN %d\n#define OP_R %d\n#include \"acc_hip_device.h\"\n#include \"op_recur.h\"\n",
                sp.type, sp.gate, v.back ? 1 : 0, v.step ? 1 : 0, v.thin ? 1 : 0, v.rows);
  return text;
}

// grouped: rows and columns of a tile, in sixteens, and the steps that are asked for ahead
struct GroupedVariant {
  int bm = 16, fn = 1;
  bool zeros = false;
  int wide = 16;                // ... waves of that form
  bool few = false;             // ... and each has a few steps
  bool sixteen = false;         // tiles of sixteen rows, whose places are known when the kernel is compiled
  bool stream = false;          // rows in LDS, waves that go over columns (else they read rows and codes for every tile)
  bool tall = false;            // tiles of 64 rows by 256 columns
  bool elements = false;
  int waves() const { return tall ? 4 : stream || fn == 1 ? wide : 4; }
  int ahead(const OpSpec &sp) const
  {
    // (their scales and zeros are a load of 64 lanes)
    if (stream) return few || sp.group == 32 || (sp.group == 64 && sp.type == 0) ? 2 : 4;
    return elements || bm > 32 || (bm > 16 && sp.type == 0) ? 1 : bm > 16 || fn > 1 || sp.type == 0 ? 2 : 4;
  }
  uint32_t key() const { return (uint32_t)(bm / 16) | (uint32_t)fn << 4 | (elements ? 256u : 0u) | (stream ? 512u : 0u) | (zeros ? 1024u : 0u) | (wide == 8 ? 2048u : 0u) | (sixteen ? 4096u : 0u) | (few ? 8192u : 0u) | (tall ? 16384u : 0u); }
};
std::string grouped_source(const OpSpec &sp, const GroupedVariant &v)
{
  char text[512];
  std::snprintf(text, sizeof(text),
                "#define OP_ELT %d\n#define OP_TYPE %d\n#define OP_BM %d\n#define OP_FN %d\n#define OP_GROUP %d\n#define OP_AHEAD %d\n#define OP_STREAM %d\n#define OP_WIDE %d\n#define OP_WAVES %d\n#define OP_ZEROS %d\n#define OP_HEIGHT %d\n#define OP_ELEMENTS %d\n#include \"acc_hip_device.h\"\n#include \"op_grouped.h\"\n",
                sp.type, sp.type == 1 ? 1 : 2, v.bm, v.fn, v.elements ? 4 : std::min(4, sp.group / 32), v.ahead(sp), v.stream ? 1 : 0, v.tall ? 1 : 0, v.waves(), v.zeros ? 1 : 0, v.sixteen ? 16 : 0, v.elements ? 1 : 0);
  return text;
}

std::vector<std::string> op_options()
{
  // (sums of products may be contracted: nothing here has to round as a scalar expression of the array language does; packed
  // Float32 arithmetic is off as for the skeletons)
  return {"-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"};
}

// whether products of this form come in that tile
bool has_tile(const OpSpec &sp, const ProductVariant &v, int t)
{
  const bool wide = sp.kind == ACC_OP_MICRO, word = !wide && sp.type == 0;
  if (t >= kSkinny) return !v.outer && v.aligned && v.fours && v.b_fast && (t == kSkinny || (!wide && !word));
  if (t == kLarge) return v.aligned && !word;
  if (t == kMiddle) return v.outer || !word;
  if (t == kWide) return !v.outer && !word;
  return t == kSquare ? v.outer || word : !v.outer;
}

// every translation unit an instance may need: the build check compiles them all
std::vector<std::string> all_sources(const OpSpec &sp)
{
  std::vector<std::string> out;
  if (sp.kind == ACC_OP_PRODUCT) {
    if (sp.type != 0) out.push_back(pack_source(sp));
    for (int t = 0; t < kProductTileCount; ++t)
      for (int form = 0; form < 15; ++form) {
        ProductVariant v;
        v.tile = t;
        v.outer = form >= 6;
        v.b_fast = !v.outer && (form & 1) == 0;
        v.aligned = v.outer ? form % 3 == 0 : form < 2;
        v.tiny = v.outer ? form % 3 == 2 : form >= 4;
        v.index = v.outer ? (form - 6) / 3 : 0;
        if (!has_tile(sp, v, t)) continue;
        v.places = v.index != 0 && !v.tiny;
        out.push_back(product_source(sp, v));
        if (!v.places || t == kLarge) continue;
        v.places = false;
        out.push_back(product_source(sp, v));
      }
  } else if (sp.kind == ACC_OP_ROUTE) {
    for (int experts : {1, 8, 16, 32, 64, 128, 256, 512, 1024, 2048}) if (experts >= sp.choose)
      for (bool aligned : {true, false})
        for (int64_t tokens : {int64_t(0), int64_t(1), int64_t(1) << 20}) out.push_back(route_source(sp, route_variant(sp, experts, aligned, tokens)));
  } else if (sp.kind == ACC_OP_COMBINE) {
    for (int rows : {0, 1, 2}) out.push_back(combine_source(sp, rows));
  } else if (sp.kind == ACC_OP_SCORE) {
    for (int lanes : {4, 8, 16, 32, 64})
      for (int per : {8, 16, 32, 64})
        for (bool few : {true, false}) {
          if (per > kScoreSlice) continue;
          ScoreVariant v;
          v.lanes = lanes;
          v.per = per;
          v.few = few;
          if ((per <= 32 || lanes < 64) && lanes >= sp.groups) out.push_back(score_source(sp, v));
        }
  } else if (sp.kind == ACC_OP_GROUPED) {
    for (int bm : {16, 32, 64})
      for (int form = 0; form < 12; ++form) {
        GroupedVariant v;
        v.bm = bm;
        v.zeros = form & 1;
        v.stream = form >= 4;
        if (!v.stream) v.fn = 1 + form / 2;
        if (!v.stream && bm > 32 && v.fn == 1) continue;
        v.wide = form & 2 || !v.stream ? 8 : 16;
        v.sixteen = form >= 8;
        for (bool few : {false, true}) {
          v.few = few;
          if (!(few && !v.stream) && !(v.stream && bm > 32) && !(v.sixteen && bm > 16)) out.push_back(grouped_source(sp, v));
        }
      }
    GroupedVariant v;
    v.tall = true;
    for (bool zeros : {false, true}) {
      v.zeros = zeros;
      out.push_back(grouped_source(sp, v));
    }
    v = {};
    v.elements = true;
    out.push_back(grouped_source(sp, v));
  } else if (sp.kind == ACC_OP_RECUR) {
    for (int form = 0; form < 6; ++form)
      for (int rows : {8, 16, 32}) {
        RecurVariant v;
        v.step = form >= 4;
        v.thin = form & 1;
        v.back = form & 2 && !v.step;
        if (!v.step) v.rows = rows;
        if (!(v.thin && sp.type == 0) && !(v.back && rows == 32)) out.push_back(recur_source(sp, v));
      }
  } else {
    for (bool aligned : {true, false}) out.push_back(micro_source(sp, aligned));
    for (int t = 0; t < kProductTileCount; ++t)
      for (int form = 0; form < 4; ++form) {
        ProductVariant v;
        v.tile = t;
        v.aligned = form < 2;
        v.tiny = form % 2 == 1;
        if (!has_tile(sp, v, t)) continue;
        out.push_back(product_source(sp, v));
      }
  }
  std::sort(out.begin(), out.end());
  out.erase(std::unique(out.begin(), out.end()), out.end());
  return out;
}

int make_spec(const acc_op_desc *d, OpSpec *sp)
{
  if (!d) return fail(ACC_ERR_INVALID, "acc_op_create: NULL description");
  if (d->kind < 0 || d->kind >= ACC_OP_KIND_COUNT || !*kKindName[d->kind]) return fail(ACC_ERR_INVALID, "acc_op_create: unknown kind %d", d->kind);
  const std::string t = d->elt_type ? d->elt_type : "";
  if (t == "float") sp->type = 0;
  else if (t == "half") sp->type = 1;
  else if (t == "bfloat16") sp->type = 2;
  else return fail(ACC_ERR_INVALID, "acc_op_create: element type '%s' (float, half and bfloat16 are served)", t.c_str());
  sp->kind = d->kind;
  sp->choose = d->choose;
  sp->normalise = d->normalise != 0;
  if (d->kind == ACC_OP_SCORE) {
    if (d->choose < 1 || d->choose > 32) return fail(ACC_ERR_INVALID, "acc_op_create: a router by scores chooses 1 to 32 experts, not %d", d->choose);
    if (d->groups < 1 || d->groups > 64 || (d->groups & (d->groups - 1)) != 0) return fail(ACC_ERR_INVALID, "acc_op_create: %d groups (a power of two up to 64)", d->groups);
    if (d->keep < 1 || d->keep > d->groups) return fail(ACC_ERR_INVALID, "acc_op_create: %d of %d groups are kept", d->keep, d->groups);
    if (!(d->scale - d->scale == 0.0f)) return fail(ACC_ERR_INVALID, "acc_op_create: a scale that is not finite");
    sp->groups = d->groups;
    sp->keep = d->keep;
    sp->scale = d->scale;
  }
  if (d->kind == ACC_OP_GROUPED) {
    if (d->group < 32 || (d->group & (d->group - 1)) != 0) return fail(ACC_ERR_INVALID, "acc_op_create: a group of %d neighbours (a power of two, 32 or more)", d->group);
    sp->group = d->group;
  }
  if (d->kind == ACC_OP_RECUR) {
    if (d->gate != ACC_GATE_GIVEN && d->gate != ACC_GATE_SIGMOID) return fail(ACC_ERR_INVALID, "acc_op_create: unknown gate %d", d->gate);
    sp->gate = d->gate;
  }
  if (d->kind == ACC_OP_ROUTE && (d->choose < 1 || d->choose > 64)) return fail(ACC_ERR_INVALID, "acc_op_create: a router chooses 1 to 64 experts, not %d", d->choose);
  return ACC_OK;
}

// ---- arrays ---------------------------------------------------------------------------

// the bytes that an array spans, and where they start
struct Span { uint64_t from = 0, to = 0; };
Span span_of(const acc_strided &a, int bytes)
{
  Span s;
  uint64_t last = 0;
  for (int d = 0; d < a.rank; ++d) {
    if (a.shape[d] == 0) return s;
    last += (uint64_t)(a.shape[d] - 1) * (uint64_t)a.stride[d];
  }
  s.from = a.ptr;
  s.to = a.ptr + (last + 1) * (uint64_t)bytes;
  return s;
}

bool is_empty(const acc_strided &a)
{
  for (int d = 0; d < a.rank; ++d)
    if (a.shape[d] == 0) return true;
  return false;
}

int check(const char *who, const char *what, const acc_strided *a, int rank)
{
  if (!a) return fail(ACC_ERR_INVALID, "%s: %s missing", who, what);
  if (a->rank != rank) return fail(ACC_ERR_INVALID, "%s: %s has rank %d, expected %d", who, what, a->rank, rank);
  for (int d = 0; d < rank; ++d) {
    if (a->shape[d] < 0 || a->shape[d] > 0x7fffffff) return fail(ACC_ERR_INVALID, "%s: %s has an extent of %lld", who, what, (long long)a->shape[d]);
    if (a->stride[d] < 0) return fail(ACC_ERR_INVALID, "%s: %s has a negative stride", who, what);
  }
  if (!a->ptr && !is_empty(*a)) return fail(ACC_ERR_INVALID, "%s: %s is NULL", who, what);
  return ACC_OK;
}

// dimension d moves by one element (or does not move at all)
bool unit(const acc_strided &a, int d) { return a.shape[d] <= 1 || a.stride[d] == 1; }

int check_unit(const char *who, const char *what, const acc_strided *a, int rank)
{
  ACC_TRY(check(who, what, a, rank));
  if (!unit(*a, rank - 1)) return fail(ACC_ERR_INVALID, "%s: the innermost dimension of %s is not contiguous", who, what);
  return ACC_OK;
}

// rows of a result must not lie on one another
int check_result(const char *who, const char *what, const acc_strided *a, int rank)
{
  ACC_TRY(check_unit(who, what, a, rank));
  int64_t least = a->shape[rank - 1];
  for (int d = rank - 2; d >= 0; --d) {
    if (a->shape[d] > 1 && a->stride[d] < least) return fail(ACC_ERR_INVALID, "%s: rows of %s overlap", who, what);
    least = std::max(least, a->stride[d] * std::max<int64_t>(1, a->shape[d]));
  }
  return ACC_OK;
}

int check_shape(const char *who, const char *what, const acc_strided &a, std::initializer_list<int64_t> shape)
{
  int d = 0;
  for (int64_t s : shape) {
    if (a.shape[d] != s) return fail(ACC_ERR_INVALID, "%s: dimension %d of %s is %lld, expected %lld", who, d, what, (long long)a.shape[d], (long long)s);
    ++d;
  }
  return ACC_OK;
}

// The products' kernels count rows, columns and elements of a sum in 32 bits, and a tile, or the step of a sum asked for ahead, reaches
// up to 1024 of them beyond the last.
constexpr int64_t kLongest = 0x7fffffff - 4095;
int check_extents(const char *who, std::initializer_list<int64_t> extents)
{
  for (int64_t n : extents)
    if (n > kLongest) return fail(ACC_ERR_INVALID, "%s: an extent of %lld (at most %lld)", who, (long long)n, (long long)kLongest);
  return ACC_OK;
}

struct Named { const acc_strided *a; int bytes; const char *what; };
// whether two arrays of rows are different columns of one: rows as far apart, whose stretches lie beside each other
bool beside(const Named &a, const Named &b)
{
  if (a.a->rank != 2 || b.a->rank != 2 || !unit(*a.a, 1) || !unit(*b.a, 1)) return false;
  const int64_t pitch = a.a->stride[0] * a.bytes, a_row = a.a->shape[1] * a.bytes, b_row = b.a->shape[1] * b.bytes;
  if (pitch <= 0 || pitch != b.a->stride[0] * b.bytes) return false;
  // (how far a's stretch begins behind b's, of whichever rows)
  const uint64_t p = (uint64_t)pitch;
  const int64_t at = (int64_t)(a.a->ptr >= b.a->ptr ? (a.a->ptr - b.a->ptr) % p : (p - (b.a->ptr - a.a->ptr) % p) % p);
  return at >= b_row && at + a_row <= pitch;
}
int check_apart(const char *who, const Named &out, std::initializer_list<Named> others)
{
  const Span o = span_of(*out.a, out.bytes);
  for (const Named &n : others) {
    if (!n.a) continue;
    const Span s = span_of(*n.a, n.bytes);
    if (s.from < o.to && o.from < s.to && !beside(out, n)) return fail(ACC_ERR_INVALID, "%s: %s shares memory with %s", who, out.what, n.what);
  }
  return ACC_OK;
}

// every row of an array starts on 16 bytes
bool aligned_rows(const acc_strided &a, int bytes, int inner)
{
  if (a.ptr & 15u) return false;
  for (int d = 0; d < a.rank; ++d)
    if (d != inner && a.shape[d] > 1 && (a.stride[d] * bytes) % 16 != 0) return false;
  return true;
}

template <typename T> T *device(const acc_strided *a) { return a ? reinterpret_cast<T *>(a->ptr) : nullptr; }

// tiles of `height` rows that cover the segments, whatever their lengths: every segment with a row (and the rows before the
// first and behind the last) may end amid a tile
int64_t tiles_at_most(int64_t rows, int64_t experts, int64_t height)
{
  const int64_t parts = std::min(rows, experts + 2);
  return (rows + parts * (height - 1)) / height;
}

// An index at is divided by `per` as (at * mul) >> (32 + shift), exact for 0 <= at < 2^31 (with l = ceil(log2 per), mul is
// 2^(31 + l) / per rounded up: its excess times at stays below 2^(31 + l)).
template <typename T> void set_divisor(int32_t per, T *a)
{
  if (per < 2) return;
  int l = 1;
  while ((int64_t(1) << l) < per) ++l;
  a->per_mul = static_cast<uint32_t>(((uint64_t(1) << (31 + l)) + (uint64_t)per - 1) / (uint64_t)per);
  a->per_shift = static_cast<uint32_t>(l - 1);
}

// Whether offsets of 32 bits (and buffers below 2 GB) do for an operand of the aligned form: rows of `row` bytes of which
// `tile` (all `rows` of them, with an index) are reached from one base; rows must not overlap, as a buffer that ends with the
// last row that counts would cut others short.
constexpr int kTallest = 256;
bool near_enough(const acc_strided &a, int rows_dim, int64_t row, int bytes, bool index)
{
  const int64_t stride = a.stride[rows_dim] * bytes, reached = index ? a.shape[rows_dim] : std::min<int64_t>(a.shape[rows_dim], kTallest);
  return (a.shape[rows_dim] <= 1 || stride >= row) && stride <= 0x7fffffff && reached * stride + row < 0x7fff0000;
}

// the knob's tile, where the form has it
int tile_of(const OpSpec &sp, const ProductVariant &v, int tile)
{
  return sp.tile >= 0 && sp.tile < kProductTileCount && has_tile(sp, v, sp.tile) ? sp.tile : tile;
}

// The tile shape for products of `rows` rows of `experts` segments, of sums of `steps` cache lines.  A larger tile reads less
// (an operand goes by once for every tile of the other's) and has more products for a load, a smaller one fills more compute
// units; what a segment leaves over is a tile of its own.  Measured in us, 16 segments unless said:
//   few rows (op_skinny.h): 16 rows, 8 of 1024 x 1024: 6.4 in columns of 32, 10 in tiles of 32 x 64; 64 rows, 32 of 4096 x 2048: 85 in
//     columns of 32, 94 in those of 64, 121 in tiles; 128 rows of 4096 x 4096: 122, 107 and 128; Float32, 16 rows of 2048 x 2048: 45,
//     52 in tiles.  4 bits only where the matrices are few: 32 rows of 4096 x 4096: 41 and 33 in tiles of 64 x 128
//   Float32, bound by the matrix cores, wants them full to the end: 8192 rows, 8 of 1024 x 1536: 207 in 32 x 64 or 64 x 64, 225 in
//     64 x 128, 270 in 128 x 128; 1024, 4 of 512 x 2048: 38, 37, 66, 124; 20000, 8 of 768 x 1024: 247, 233, 244, 244
//   256 x 256 from 128 rows a segment on: 2048 rows of 4096 x 4096: 137 in 128 x 128, 141 in 256 x 256; 4096: 227 and 147; 5120: 350
//     and 276.  Not for few tiles (8192 rows, 8 of 1024 x 1024, 128 tiles: 37 and 60) or short sums (16384, 8 of 2048 x 256: 36 and 41).
//     4 bits already from 48 rows on, and for any sum: 1024 rows of 4096 x 4096: 42 and 39; 22272, 4 of 1976 x 44: 48 and 44
//   128 x 128 from 64 rows on, 64 x 128 from 32, where there are 256 tiles: 1536 rows of 4096 x 2048: 104 in 64 x 128, 74 in
//     128 x 128; 768: 97 in 32 x 64, 70 in 64 x 128; 512: 67 and 70; but 1024 of 1000 x 1000, with 128 tiles of 64 x 128: 13 and 16
//   64 x 128 for long sums that 32 x 64 would not cut: 256 rows, 1 of 4096 x 4096: 28 in 32 x 64, 22 in pieces of 64 x 128
constexpr int64_t kCutBelow = 192;                   // workgroups, see rows_piece
int rows_tile(const OpSpec &sp, const ProductVariant &v, int64_t rows, int64_t experts, int64_t n, int64_t steps)
{
  const int64_t mean = ceil_div(rows, std::max<int64_t>(1, experts));
  const bool wide = sp.kind == ACC_OP_MICRO, word = !wide && sp.type == 0;
  const auto groups = [&](int t) {
    return std::max(ceil_div(rows, kProductTiles[t].bm), std::min(rows, experts)) * ceil_div(n, kProductTiles[t].bn);
  };
  if (v.aligned && v.fours && v.b_fast && mean <= 12) {
    if (word || std::min(rows, experts) * ceil_div(n, 64) < 192 || (!wide && steps <= 32)) return kSkinny;
    if (!wide) return kSkinny + 1;
  }
  if (word) return groups(kSquare) >= 1024 ? kSquare : kLow;
  if (v.aligned && n >= 256 && (wide || steps > 8) && groups(kLarge) >= 192 && mean > (wide ? 48 : 128)) return kLarge;
  if (groups(kMiddle) >= 256 && mean > 64) return kMiddle;
  if (groups(kWide) >= 256 && (wide || mean > 32)) return kWide;
  if (steps >= 48 && mean > 32 && groups(kLow) >= kCutBelow) return kWide;
  return kLow;
}

// Sums of `length` elements, in steps of `step`, in fewer workgroups than kCutBelow are cut into pieces of eight steps or more
// that make 512 of them, two a compute unit: elements of a piece, or 0 for one.  Another kernel adds the pieces up, 3 us.
// 64 rows, 4 matrices of 1024 x 4096 bfloat16: 13 us and 28 uncut; 8 Float32 rows of 611 x 3059: 20 and 48; 1094 half rows, 2 of
// 320 x 1005: 13 and 12.  (256 workgroups: 14, 22, 12; pieces of four steps: 13, 20, 13.)
int32_t rows_piece(const ProductVariant &v, int64_t groups, int64_t length, int64_t step)
{
  if (v.tile >= kSkinny || groups >= kCutBelow) return 0;
  const int64_t steps = ceil_div(length, step), each = std::max<int64_t>(8, ceil_div(steps * groups, 512));
  return each * 2 > steps ? 0 : (int32_t)(each * step);
}

// Outer: the tile shape.  A tile is worth its size where there are enough of them, cut as short as pays, to fill the
// compute units.  In us: 32000 rows, 16 bfloat16 results of 2048 x 2048: 249 in 256 x 256, 309 in 128 x 128, 465 in 64 x 64; 8192, 8 of
// 1024 x 1024: 52, 42 and 40; 1664, 13 of 800 x 2160: 29 in 128 x 128 and 36 in 64 x 64; 17385, 2 of 64 x 988: 29 and 25; 30000, 4 of
// 64 x 2048: 38 and 45.  Float32: 2240 rows, 15 of 3014 x 192: 85 and 48; 8192, 8 of 1024 x 1024, skewed: 235 and 147, of 1024 x 1536:
// 203 and 209.
int outer_tile(const OpSpec &sp, const ProductVariant &v, int64_t rows, int64_t experts, int64_t ni, int64_t nj)
{
  const auto groups = [&](int t, int64_t steps) {
    const int64_t tiles = ceil_div(ni, kProductTiles[t].bm) * ceil_div(nj, kProductTiles[t].bn), least = steps * 128 / type_bytes(sp.type);
    return tiles * std::max(experts, rows / least);
  };
  if (has_tile(sp, v, kLarge) && rows < (1 << 28) && ni >= 256 && nj >= 256 && groups(kLarge, 16) >= 256) return kLarge;
  return groups(kMiddle, 8) >= (sp.type == 0 ? 3000 : 512) ? kMiddle : kSquare;
}
// ... and the rows of a piece (0: segments are not cut), where whole segments make too few tiles to fill the compute units:
// 17110 Float32 rows, 13 results of 64 x 64: 17 us and 369 uncut; 30043, 3 of 64 x 768: 45 and 799.
int32_t outer_piece(const OpSpec &sp, const ProductVariant &v, int64_t rows, int64_t experts, int64_t tiles)
{
  const int64_t target = v.tile == kLarge ? 256 : v.tile == kMiddle ? 512 : 1024, step = 128 / type_bytes(sp.type);
  if (experts * tiles >= target) return 0;
  const int64_t least = (v.tile == kLarge ? 16 : 8) * step, most = std::max(least, ceil_div(rows * tiles, target - experts * tiles));
  // (segments of about the mean length in equal pieces, with a tenth to spare: 23602 rows, 11 of 431 x 576: 55 us, 65 otherwise)
  const int64_t mean = std::max<int64_t>(1, ceil_div(rows, experts)), each = ceil_div(mean, ceil_div(mean, most)), piece = ceil_div(std::max(least, std::min(most, each + each / 10)), step) * step;
  return experts * piece >= 2 * rows ? 0 : (int32_t)piece;
}

// grouped: LDS of the form with rows in it: `height` of them, their sums by groups, and the waves' results where they share columns
int64_t grouped_lds(const OpSpec &sp, int64_t height, int64_t steps, int64_t waves)
{
  const int64_t chunks = sp.group >= 128 ? 1 : 128 / sp.group;
  return steps * height * (256 * (sp.type == 0 ? 3 : 1) + chunks * (sp.type == 0 ? 8 : 4)) + waves * ceil_div(height, 16) * 1024;
}
constexpr int64_t kGroupedLds = 160 << 10;
// ... and of tiles of 64 rows by 256 columns: three steps of rows, scales and zeros, two of sums
int64_t grouped_tall_lds(const OpSpec &sp, bool zeros)
{
  const int64_t chunks = sp.group >= 128 ? 1 : 128 / sp.group;
  const int64_t rows = sp.type == 0 ? 32 : 64, parts = sp.type == 0 ? 3 : 1;
  return 3 * 16 * parts * rows * 16 + 3 * chunks * 272 * 4 * (zeros ? 2 : 1) + 2 * chunks * rows * 4 * (sp.type == 0 ? 2 : 1);
}
// ... and the tiles of 16 columns from which on rows in LDS are worth what it takes to put them there.  us, with and without, tiles: 1 row,
// 4096 x 4096, 256: 7.8 and 7.6; 16 rows: 14 and 10; 2 rows of 4096 x 11008, 256: 17 and 14; of 11008 x 4096, 688: 14 and 17; 1 row, 8192 x 8192,
// 512: 15 and 23; 64 rows, 16 half of 4096 x 2048, 4096: 24 and 33; 16, 8 of 4096 x 4096 in groups of 32: 26 and 36; Float32, 64, 16 of
// 1024 x 2048, 1024: 15 and 13
constexpr int64_t kGroupedStream = 384;
// Whether a call is for tiles of 64 rows (Float32: 32) by 256 columns that make numbers of the codes as they go: rows enough for them, and tiles
// enough (one that is 4096 long takes 50 us, in groups of 32 75, however few there are).  us, with and without, rows (a few more or less
// a segment), matrices, tiles: 320, 8 of 4096 x 4096, 128: 59 and 75; 200, 1 of 4096 x 4096, 64: 50 and 41; 300, 1, 80: 54 and 59, in groups of
// 32 81 and 70; 400, 1, 112: 52 and 69, in groups of 32 76 and 76; 2000, 1, 512: 85 and 278; 600, 4 of 1024 x 2048, 48: 29 and 24; 1200, 4, 80: 31
// and 39; 900, 4 of 2000 x 1000, 120: 22 and 27; 1000, 20 of 500 x 2000, 40: 37 and 24.  Float32: 130, 1 of 4096 x 4096, 80: 65 and 71, in groups
// of 32 91 and 93; 300, 1, 160: 66 and 113, 91 and 145; 300, 4 of 1024 x 2048, 48: 36 and 25; 600, 4, 80: 37 and 47, 49 and 57
bool grouped_tall(const OpSpec &sp, int64_t rows, int64_t experts, int64_t n, int64_t k, int64_t pitch, int64_t mean)
{
  const bool wide = sp.type == 0;
  const int64_t tiles = std::max(ceil_div(rows, wide ? 32 : 64), std::min(rows, experts)) * ceil_div(n, 256);
  return n >= 16 && k > 0 && pitch < (1 << 26) && mean > 32 && tiles >= (!wide && sp.group == 32 ? 96 : 72);
}
// the tile for `mean` rows a segment; *height: its rows.  (Where LDS holds fewer rows than a segment has, their codes are read again:
// 64 rows, 2 of 4096 x 4096: 28 us in tiles of 16, 31 without LDS.)
GroupedVariant grouped_variant(const OpSpec &sp, int64_t rows, int64_t experts, int64_t n, int64_t k, int64_t pitch, int64_t mean, int64_t *height)
{
  GroupedVariant v;
  const int64_t steps = ceil_div(k, 128);
  v.bm = mean > 32 ? 64 : mean > 16 ? 32 : 16;
  *height = v.bm;
  if (v.bm < 64 && n >= 16 && pitch < (1 << 27) && steps > 0) {
    int64_t h = v.bm;
    while (h > 1 && grouped_lds(sp, h, steps, 16) > kGroupedLds) h /= 2;
    const int64_t tiles = std::max(ceil_div(rows, h), std::min(rows, experts)) * ceil_div(n, 16);
    if (grouped_lds(sp, h, steps, 16) <= kGroupedLds && h * 4 >= mean && tiles >= kGroupedStream) {
      v.stream = true;
      v.bm = h > 16 ? 32 : 16;
      v.sixteen = h == 16;
      // (two workgroups a compute unit where there is room: one begins while the other is at its columns)
      v.wide = grouped_lds(sp, h, steps, 16) <= kGroupedLds / 2 ? 8 : 16;
      *height = h;
      return v;
    }
  }
  v.wide = 8;
  v.fn = v.bm > 32 || std::min(rows, experts) * ceil_div(n, 32) >= 512 ? 2 : 1;
  return v;
}

}  // namespace

struct acc_op_s {
  acc_context ctx = nullptr;
  OpSpec spec;
  std::mutex mu;
  std::map<uint32_t, OpVariant> variants;

  // the kernels of a variant: compiled, loaded, `names` looked up (fn, fn2, fn3 in that order)
  int variant(uint32_t key, const char *const *names, int n_names, std::string (*source)(const OpSpec &, uint32_t), const OpVariant **out);
};

namespace {

constexpr uint32_t kPack = 1u << 20;                 // (beside the products' keys)
std::string product_source_of(const OpSpec &sp, uint32_t key)
{
  if (key == kPack) return pack_source(sp);
  ProductVariant v;
  v.tile = (int)(key & 15u);
  v.outer = key & 16u;
  v.b_fast = key & 32u;
  v.aligned = key & 64u;
  v.index = (int)(key >> 7 & 3u);
  v.tiny = key & 512u;
  v.places = key & 2048u;
  return product_source(sp, v);
}
std::string route_source_of(const OpSpec &sp, uint32_t key)
{
  RouteVariant v;
  v.lanes = (int)(key & 127u);
  v.few = key & 128u;
  v.per = (int)(key >> 8 & 255u);
  v.vec = (int)(key >> 16 & 255u);
  v.sels = (int)(key >> 24 & 63u);
  v.tall = key >> 30;
  v.halves = key >> 30 == 3u ? 4 : key >> 30 == 2u ? 2 : 1;
  return route_source(sp, v);
}
std::string combine_source_of(const OpSpec &sp, uint32_t key) { return combine_source(sp, (int)(key & 3u)); }
constexpr uint32_t kMicroElements = 1024;            // (above the products' keys)
std::string micro_source_of(const OpSpec &sp, uint32_t key) { return (key & kMicroElements) ? micro_source(sp, key & 1u) : product_source_of(sp, key); }

std::string recur_source_of(const OpSpec &sp, uint32_t key)
{
  RecurVariant v;
  v.back = key & 1u;
  v.step = key & 2u;
  v.thin = key & 4u;
  v.rows = (int)(key >> 4);
  return recur_source(sp, v);
}

std::string grouped_source_of(const OpSpec &sp, uint32_t key)
{
  GroupedVariant v;
  v.bm = (int)(key & 15u) * 16;
  v.fn = (int)(key >> 4 & 15u);
  v.elements = key & 256u;
  v.stream = key & 512u;
  v.zeros = key & 1024u;
  v.wide = key & 2048u ? 8 : 16;
  v.sixteen = key & 4096u;
  v.few = key & 8192u;
  v.tall = key & 16384u;
  return grouped_source(sp, v);
}

std::string score_source_of(const OpSpec &sp, uint32_t key)
{
  ScoreVariant v;
  v.lanes = (int)(key & 127u);
  v.per = (int)(key >> 8 & 127u);
  v.few = key >> 16 & 1u;
  return score_source(sp, v);
}

const char *const kScoreNames[] = {"score", "route_place", "score_gradient"};
const char *const kGroupedNames[] = {"grouped"};
const char *const kGroupedElementNames[] = {"grouped_quantise", "grouped_values"};
const char *const kRecurNames[] = {"recur", "recur_clear"};
const char *const kRecurStepNames[] = {"recur_step"};
const char *const kProductNames[] = {"product", "product_join", "product_places"};
const char *const kPackNames[] = {"pack"};
const char *const kRouteNames[] = {"route", "route_place", "route_gradient"};
const char *const kCombineNames[] = {"combine", "combine_gradient"};
const char *const kMicroNames[] = {"micro_quantise", "micro_values"};

// one call's stream and its guard (a loop enqueued ahead, see acc_guard_create)
int begin(acc_op op, int kind, const char *who, acc_stream stream, const uint32_t **guard)
{
  if (!op) return fail(ACC_ERR_INVALID, "%s: NULL operator", who);
  if (op->spec.kind != kind) return fail(ACC_ERR_INVALID, "%s: the operator is a '%s'", who, kKindName[op->spec.kind]);
  *guard = reinterpret_cast<const uint32_t *>(op->ctx->guard_of(static_cast<hipStream_t>(stream)));
  return op->ctx->make_current();
}

// threads of a launch: their number has 32 bits, and HIP starts those of a larger one that are left over 2^32 without a word
constexpr int64_t kThreads = 0xffffffffll;

template <typename T>
int launch(acc_op op, const char *entry, hipFunction_t fn, int64_t grid, int block, size_t lds, acc_stream stream, const T &args)
{
  if (grid < 1 || grid > kThreads / block) return fail(ACC_ERR_INVALID, "%s: grid of %lld workgroups of %d", entry, (long long)grid, block);
  T copy = args;
  void *slots[] = {&copy};
  return acc::launch_operator(op->ctx, entry, fn, static_cast<unsigned>(grid), static_cast<unsigned>(block), static_cast<unsigned>(lds),
                              static_cast<hipStream_t>(stream), slots);
}

}  // namespace

int acc_op_s::variant(uint32_t key, const char *const *names, int n_names, std::string (*source)(const OpSpec &, uint32_t), const OpVariant **out)
{
  std::lock_guard<std::mutex> lock(mu);
  OpVariant &v = variants[key];              // (a map's elements stay where they are)
  if (!v.fn) {
    if (!v.job) {
      auto job = std::make_shared<acc::CompileJob>();
      job->target = ctx->arch;
      job->source = source(spec, key);
      job->options = op_options();
      v.job = job;
      job->run();
    }
    ACC_TRY(v.job->wait());
    ACC_TRY(ctx->make_current());
    hipModule_t module = nullptr;
    ACC_HIP_TRY(hipModuleLoadData(&module, v.job->code));
    hipFunction_t fn[3] = {nullptr, nullptr, nullptr};
    for (int k = 0; k < n_names; ++k) {
      const hipError_t e = hipModuleGetFunction(&fn[k], module, names[k]);
      if (e != hipSuccess) {
        (void)hipModuleUnload(module);
        return acc::fail_hip(e, names[k]);
      }
    }
    v.module = module;
    v.fn2 = fn[1];
    v.fn3 = fn[2];
    v.fn = fn[0];
  }
  *out = &v;
  return ACC_OK;
}

extern "C" {

int acc_op_create(acc_context ctx, const acc_op_desc *desc, acc_op *out)
try {
  if (!ctx || !out) return fail(ACC_ERR_INVALID, "acc_op_create: NULL argument");
  *out = nullptr;
  OpSpec sp;
  ACC_TRY(make_spec(desc, &sp));
  acc_op_s *op = new acc_op_s();
  op->ctx = ctx;
  op->spec = sp;
  op->spec.tile = ctx->tuning_now()->get("product.tile", -1);
  *out = op;
  return ACC_OK;
} ACC_OP_CATCH("acc_op_create")

int acc_op_destroy(acc_op op)
try {
  if (!op) return ACC_OK;
  (void)op->ctx->make_current();
  for (auto &kv : op->variants)
    if (kv.second.module) (void)hipModuleUnload(kv.second.module);
  delete op;
  return ACC_OK;
} ACC_OP_CATCH("acc_op_destroy")

int acc_op_compile_only(const char *target, const acc_op_desc *desc, int32_t *units, size_t *code_size)
try {
  if (!target || !units || !code_size) return fail(ACC_ERR_INVALID, "acc_op_compile_only: NULL argument");
  OpSpec sp;
  ACC_TRY(make_spec(desc, &sp));
  *units = 0;
  *code_size = 0;
  std::vector<std::shared_ptr<acc::CompileJob>> jobs;
  for (const std::string &text : all_sources(sp)) {
    auto job = std::make_shared<acc::CompileJob>();
    job->target = target;
    job->source = text;
    job->options = op_options();
    if (!acc::compile_submit(job)) job->run();
    jobs.push_back(job);
  }
  int rc = ACC_OK;
  for (auto &job : jobs) {
    const int one = job->wait();
    if (one != ACC_OK) rc = one;
    *code_size += job->size;
    ++*units;
  }
  return rc;
} ACC_OP_CATCH("acc_op_compile_only")

// ---- products -----------------------------------------------------------------------

// scratch memory; a graph's own where the call is being recorded into one
static int scratch_of(acc_op op, acc_stream stream, size_t bytes, acc::ScratchRef *out)
{
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(static_cast<hipStream_t>(stream), &capture) != hipSuccess) (void)hipGetLastError();
  return op->ctx->scratch_acquire(bytes, static_cast<hipStream_t>(stream), acc::SCRATCH_FOLD, out, capture != hipStreamCaptureStatusNone);
}

// scratch memory until the call's kernels are enqueued
struct ScratchHold {
  acc_context ctx = nullptr;
  hipStream_t stream = nullptr;
  acc::ScratchRef ref;
  int acquire(acc_op op, acc_stream s, size_t bytes)
  {
    ACC_TRY(scratch_of(op, s, bytes, &ref));
    ctx = op->ctx;
    stream = static_cast<hipStream_t>(s);
    return ACC_OK;
  }
  ~ScratchHold() { if (ctx) ctx->scratch_release(ref, stream); }
};

// Whether operands of 16 bits that the aligned form cannot take are worth a copy that it can (op_pack.h): `count` copies move
// `bytes` twice, at 4.8 TB/s and a launch each; what they save is, for every factor pair, 2.4 10^-15 s in gradients, 2.2 in
// products of two such operands, 0.4 of one.  In us, as they lie and with the copies: 5000 half rows, 1 of 5001 x 5001: 475 and
// 295; 4690 bfloat16 rows, 5 of 2021 x 3367: 184 and 157; 5760, 1 of 3557 x 1344, whose rows alone start anywhere: 88 and 92;
// gradients: 8487 rows, 44 of 960 x 2722: 221 and 166.
static bool worth_packing(const OpSpec &sp, const ProductVariant &v, double pairs, double bytes, int count)
{
  const double each = v.outer ? 2.4e-15 : count == 2 ? 2.2e-15 : 0.4e-15;
  return sp.type != 0 && !v.tiny && count > 0 && bytes < 2e9 && pairs * each > 1.25 * (2 * bytes / 4.8e12 + 6e-6 * count);
}

// `from` ([batches,] rows, cols; `cols` contiguous) as rows of `cols_out` elements, rows_out of them a batch, at `to`
static int pack(acc_op op, const char *who, const acc_strided &from, int cols_dim, int64_t rows_out, int64_t cols_out, uint64_t to, const uint32_t *guard, acc_stream stream, acc_strided *out)
{
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(kPack, kPackNames, 1, product_source_of, &var));
  const int rank = from.rank, rows_dim = cols_dim == rank - 1 ? rank - 2 : rank - 1;
  acc_pack_args a = {};
  a.in = device<const void>(&from);
  a.out = reinterpret_cast<void *>(to);
  a.batches = rank == 3 ? (uint32_t)from.shape[0] : 1u;
  a.batch_stride = rank == 3 ? from.stride[0] : 0;
  a.row_stride = from.stride[rows_dim];
  a.rows = (uint32_t)from.shape[rows_dim];
  a.rows_out = (uint32_t)rows_out;
  a.cols = (int32_t)from.shape[cols_dim];
  a.chunks = (uint32_t)(cols_out * type_bytes(op->spec.type) / 16);
  set_divisor((int32_t)a.chunks, &a);
  a.guard = guard;
  *out = from;
  out->ptr = to;
  out->shape[rows_dim] = rows_out;
  out->shape[cols_dim] = cols_out;
  out->stride[cols_dim] = 1;
  out->stride[rows_dim] = cols_out;
  if (rank == 3) out->stride[0] = rows_out * cols_out;
  return launch(op, who, var->fn, ceil_div((int64_t)a.batches * rows_out * a.chunks, 256), 256, 0, stream, a);
}

// the tiles of all rows, and their sums in pieces where they are too few
static int launch_rows(acc_op op, const char *who, const ProductVariant &v, const OpVariant *var, acc_product_args &a, acc_stream stream)
{
  const ProductTile &t = kProductTiles[v.tile];
  const int64_t step = 128 / (op->spec.kind == ACC_OP_MICRO ? 1 : type_bytes(op->spec.type));
  a.tiles_i = (int32_t)tiles_at_most(a.rows, a.experts, t.bm);
  a.tiles_j = (int32_t)ceil_div(a.nj, t.bn);
  const int64_t groups = std::max(ceil_div(a.rows, t.bm), std::min<int64_t>(a.rows, a.experts)) * a.tiles_j, grid = (int64_t)a.tiles_i * a.tiles_j;
  a.piece = rows_piece(v, groups, a.k, step);
  a.pieces = a.piece ? (int32_t)ceil_div(a.k, a.piece) : 1;
  if (!a.piece) return launch(op, who, var->fn, grid, 64 * t.wm * t.wn, 0, stream, a);
  acc::ScratchRef scratch;
  ACC_TRY(scratch_of(op, stream, (size_t)a.pieces * a.rows * a.nj * 4, &scratch));
  a.parts = static_cast<float *>(scratch.ptr);
  int rc = launch(op, who, var->fn, grid * a.pieces, 64 * t.wm * t.wn, 0, stream, a);
  if (rc == ACC_OK) rc = launch(op, who, var->fn2, ceil_div(a.rows * ceil_div(a.nj, 4), 256), 256, 0, stream, a);
  op->ctx->scratch_release(scratch, static_cast<hipStream_t>(stream));
  return rc;
}

int acc_exec_product_rows(acc_op op, const acc_strided *x, const acc_strided *w, const acc_strided *offsets, const acc_strided *index, int32_t per,
                          const acc_strided *out, acc_stream stream)
try {
  const char *who = "acc_exec_product_rows";
  acc_product_args a = {};
  ACC_TRY(begin(op, ACC_OP_PRODUCT, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "x", x, 2));
  ACC_TRY(check(who, "w", w, 3));
  ACC_TRY(check_unit(who, "offsets", offsets, 1));
  ACC_TRY(check_result(who, "the result", out, 2));
  if (index) ACC_TRY(check_unit(who, "index", index, 1));
  const int64_t experts = w->shape[0], n = w->shape[1], rows = out->shape[0];
  int64_t k = w->shape[2];
  if (!unit(*w, 2) && !unit(*w, 1)) return fail(ACC_ERR_INVALID, "%s: neither the second nor the third dimension of w is contiguous", who);
  if (per < 0) return fail(ACC_ERR_INVALID, "%s: a divisor of %d", who, per);
  ACC_TRY(check_shape(who, "offsets", *offsets, {experts + 1}));
  ACC_TRY(check_shape(who, "the result", *out, {rows, n}));
  if (index) ACC_TRY(check_shape(who, "index", *index, {rows}));
  ACC_TRY(check_shape(who, "x", *x, {index ? x->shape[0] : rows, k}));
  ACC_TRY(check_extents(who, {experts, n, k, rows, x->shape[0]}));
  const int bytes = type_bytes(op->spec.type), epc = 16 / bytes;
  ACC_TRY(check_apart(who, {out, bytes, "the result"}, {{x, bytes, "x"}, {w, bytes, "w"}, {offsets, 4, "offsets"}, {index, 4, "index"}}));
  if (rows == 0 || n == 0) return ACC_OK;

  ProductVariant v;
  // (where both are contiguous -- one column, or a sum of one -- either way of reading will do)
  v.b_fast = unit(*w, 2);
  const bool x_good = k % epc == 0 && aligned_rows(*x, bytes, 1) && near_enough(*x, 0, k * bytes, bytes, index != nullptr);
  const bool w_good = k % epc == 0 && aligned_rows(*w, bytes, v.b_fast ? 2 : 1) && (v.b_fast || n % epc == 0) &&
                      near_enough(*w, v.b_fast ? 1 : 2, (v.b_fast ? k : n) * bytes, bytes, false);
  v.aligned = x_good && w_good;
  v.tiny = !v.aligned && (k < epc || (!v.b_fast && n < epc));
  ScratchHold packed;
  acc_strided xp, wp;
  if (!v.aligned) {
    // (all rows of x are copied: an index may name any)
    const int64_t kp = ceil_div(k, epc) * epc, np = ceil_div(n, epc) * epc;
    const int64_t xb = x_good ? 0 : x->shape[0] * kp * bytes, wb = w_good ? 0 : experts * (v.b_fast ? n : np) * kp * bytes, front = (xb + 255) / 256 * 256;
    if (worth_packing(op->spec, v, (double)rows * (double)n * (double)k, (double)xb + (double)wb, (xb > 0) + (wb > 0))) {
      ACC_TRY(packed.acquire(op, stream, (size_t)(front + wb)));
      const uint64_t at = reinterpret_cast<uint64_t>(packed.ref.ptr);
      if (xb) {
        ACC_TRY(pack(op, who, *x, 1, x->shape[0], kp, at, a.guard, stream, &xp));
        x = &xp;
      }
      if (wb) {
        ACC_TRY(v.b_fast ? pack(op, who, *w, 2, n, kp, at + front, a.guard, stream, &wp) : pack(op, who, *w, 1, kp, np, at + front, a.guard, stream, &wp));
        w = &wp;
      }
      k = kp;
      v.aligned = true;
    }
  }
  v.tile = tile_of(op->spec, v, rows_tile(op->spec, v, rows, experts, n, ceil_div(k * bytes, 128)));
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kProductNames, v.tile >= kSkinny ? 1 : 2, product_source_of, &var));
  a.a = device<const void>(x);
  a.b = device<const void>(w);
  a.out = device<void>(out);
  a.offsets = device<const int32_t>(offsets);
  a.index_a = device<const int32_t>(index);
  a.a_stride = x->stride[0];
  a.b_stride = w->stride[v.b_fast ? 1 : 2];
  a.b_expert = w->stride[0];
  a.out_stride = out->stride[0];
  a.rows = rows;
  a.a_rows = (int32_t)x->shape[0];
  a.nj = (int32_t)n;
  a.k = (int32_t)k;
  a.experts = (int32_t)experts;
  set_divisor(per, &a);
  return launch_rows(op, who, v, var, a, stream);
} ACC_OP_CATCH("acc_exec_product_rows")

int acc_exec_product_outer(acc_op op, const acc_strided *x, const acc_strided *y, const acc_strided *offsets, const acc_strided *index, int32_t per,
                           const acc_strided *out, acc_stream stream)
try {
  const char *who = "acc_exec_product_outer";
  acc_product_args a = {};
  ACC_TRY(begin(op, ACC_OP_PRODUCT, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "a", x, 2));
  ACC_TRY(check_unit(who, "b", y, 2));
  ACC_TRY(check_unit(who, "offsets", offsets, 1));
  ACC_TRY(check(who, "the result", out, 3));
  if (index) ACC_TRY(check_unit(who, "index", index, 1));
  if (per < 0) return fail(ACC_ERR_INVALID, "%s: a divisor of %d", who, per);
  const int64_t experts = out->shape[0], rows = x->shape[0];
  ACC_TRY(check_shape(who, "offsets", *offsets, {experts + 1}));
  ACC_TRY(check_shape(who, "the result", *out, {experts, x->shape[1], y->shape[1]}));
  if (index) ACC_TRY(check_shape(who, "index", *index, {rows}));
  else ACC_TRY(check_shape(who, "b", *y, {rows, y->shape[1]}));
  // the result's rows may run along either dimension: the other way round the operands change places
  const bool turned = !unit(*out, 2);
  acc_strided o = *out;
  if (turned) {
    std::swap(o.shape[1], o.shape[2]);
    std::swap(o.stride[1], o.stride[2]);
  }
  ACC_TRY(check_result(who, "the result", &o, 3));
  ACC_TRY(check_extents(who, {experts, out->shape[1], out->shape[2], rows, y->shape[0]}));
  const int bytes = type_bytes(op->spec.type), epc = 16 / bytes;
  ACC_TRY(check_apart(who, {out, bytes, "the result"}, {{x, bytes, "a"}, {y, bytes, "b"}, {offsets, 4, "offsets"}, {index, 4, "index"}}));
  if (is_empty(o)) return ACC_OK;
  const acc_strided *p = turned ? y : x, *q = turned ? x : y;

  ProductVariant v;
  v.outer = true;
  v.b_fast = false;
  v.index = !index ? 0 : turned ? 2 : 1;
  const bool p_good = p->shape[1] % epc == 0 && aligned_rows(*p, bytes, 1) && near_enough(*p, 0, p->shape[1] * bytes, bytes, turned && index);
  const bool q_good = q->shape[1] % epc == 0 && aligned_rows(*q, bytes, 1) && near_enough(*q, 0, q->shape[1] * bytes, bytes, !turned && index);
  v.aligned = p_good && q_good;
  v.tiny = !v.aligned && (o.shape[1] < epc || o.shape[2] < epc);
  ScratchHold packed;
  acc_strided pp, qp;
  if (!v.aligned) {
    const int64_t ip = ceil_div(o.shape[1], epc) * epc, jp = ceil_div(o.shape[2], epc) * epc;
    const int64_t pb = p_good ? 0 : p->shape[0] * ip * bytes, qb = q_good ? 0 : q->shape[0] * jp * bytes, front = (pb + 255) / 256 * 256;
    if (worth_packing(op->spec, v, (double)rows * (double)ip * (double)jp, (double)pb + (double)qb, (pb > 0) + (qb > 0))) {
      ACC_TRY(packed.acquire(op, stream, (size_t)(front + qb)));
      const uint64_t at = reinterpret_cast<uint64_t>(packed.ref.ptr);
      if (pb) {
        ACC_TRY(pack(op, who, *p, 1, p->shape[0], ip, at, a.guard, stream, &pp));
        p = &pp;
      }
      if (qb) {
        ACC_TRY(pack(op, who, *q, 1, q->shape[0], jp, at + front, a.guard, stream, &qp));
        q = &qp;
      }
      v.aligned = true;
    }
  }
  v.tile = tile_of(op->spec, v, outer_tile(op->spec, v, rows, experts, o.shape[1], o.shape[2]));
  const OpVariant *var = nullptr;
  // (Where an index names rows, a kernel in front looks them up once for all tiles: a launch, 3 us, for 8192 rows of 8 segments
  // and 1024 x 1024 results 4 us less of 44, for 32768 and 4096 x 2048 in tiles of 128 x 128 328 of 976.  Tiles of 256 x 256 have no
  // registers for anything else.)
  v.places = v.index != 0 && !v.tiny && rows < (1 << 28) && (v.tile == kLarge || rows >= 4096);
  const bool places = v.places && rows > 0;
  ACC_TRY(op->variant(v.key(), kProductNames, v.places ? 3 : 2, product_source_of, &var));
  const ProductTile &t = kProductTiles[v.tile];
  a.a = device<const void>(p);
  a.b = device<const void>(q);
  a.out = device<void>(out);
  a.offsets = device<const int32_t>(offsets);
  (turned ? a.index_a : a.index_b) = device<const int32_t>(index);
  // (the kernel takes a stride as the length of a row that it may read; that of a single row says nothing)
  a.a_stride = p->shape[0] > 1 ? p->stride[0] : p->shape[1];
  a.b_stride = q->shape[0] > 1 ? q->stride[0] : q->shape[1];
  a.out_expert = o.stride[0];
  a.out_stride = o.stride[1];
  a.rows = rows;
  a.a_rows = (int32_t)p->shape[0];
  a.b_rows = (int32_t)q->shape[0];
  a.ni = (int32_t)o.shape[1];
  a.nj = (int32_t)o.shape[2];
  a.experts = (int32_t)experts;
  set_divisor(per, &a);
  a.tiles_i = (int32_t)ceil_div(o.shape[1], t.bm);
  a.tiles_j = (int32_t)ceil_div(o.shape[2], t.bn);
  a.piece = outer_piece(op->spec, v, rows, experts, (int64_t)a.tiles_i * a.tiles_j);
  const int64_t runs = a.piece ? tiles_at_most(rows, experts, a.piece) : experts;
  const size_t front = places ? ((size_t)rows * 4 + 255) / 256 * 256 : 0, bytes_of_parts = a.piece ? (size_t)runs * a.ni * a.nj * 4 : 0;
  acc::ScratchRef scratch;
  int rc = ACC_OK;
  if (front + bytes_of_parts) {
    ACC_TRY(scratch_of(op, stream, front + bytes_of_parts, &scratch));
    a.places = static_cast<uint32_t *>(scratch.ptr);
    a.parts = reinterpret_cast<float *>(static_cast<char *>(scratch.ptr) + front);
  }
  if (places) rc = launch(op, who, var->fn3, ceil_div(rows, 256), 256, 0, stream, a);
  if (rc == ACC_OK) rc = launch(op, who, var->fn, runs * a.tiles_i * a.tiles_j, 64 * t.wm * t.wn, 0, stream, a);
  if (rc == ACC_OK && a.piece) rc = launch(op, who, var->fn2, experts * ceil_div((int64_t)a.ni * ceil_div(a.nj, 4), 256), 256, 0, stream, a);
  if (front + bytes_of_parts) op->ctx->scratch_release(scratch, static_cast<hipStream_t>(stream));
  return rc;
} ACC_OP_CATCH("acc_exec_product_outer")

// ---- router ---------------------------------------------------------------------------

static size_t route_lds(const RouteVariant &v, int64_t experts, int64_t slots) { return ((size_t)(v.threads() / 64 + 2) * (size_t)experts + (size_t)slots) * 4; }

// what a router is given, and where its results go
static int check_routing(acc_op op, const char *who, const acc_strided *logits, const acc_strided *chosen, const acc_strided *weights, const acc_strided *offsets,
                         const acc_strided *order, const acc_strided *place)
{
  ACC_TRY(check_unit(who, "logits", logits, 2));
  ACC_TRY(check_result(who, "experts", chosen, 2));
  ACC_TRY(check_result(who, "weights", weights, 2));
  ACC_TRY(check_result(who, "offsets", offsets, 1));
  ACC_TRY(check_result(who, "order", order, 1));
  ACC_TRY(check_result(who, "place", place, 2));
  const int64_t tokens = logits->shape[0], experts = logits->shape[1], choose = op->spec.choose;
  if (experts < choose || experts > kRouteMaxExperts)
    return fail(ACC_ERR_INVALID, "%s: %lld experts (at least the %lld that are chosen, and at most %d)", who, (long long)experts, (long long)choose, kRouteMaxExperts);
  ACC_TRY(check_shape(who, "experts", *chosen, {tokens, choose}));
  ACC_TRY(check_shape(who, "weights", *weights, {tokens, choose}));
  ACC_TRY(check_shape(who, "place", *place, {tokens, choose}));
  ACC_TRY(check_shape(who, "offsets", *offsets, {experts + 1}));
  ACC_TRY(check_shape(who, "order", *order, {tokens * choose}));
  for (const acc_strided *t : {chosen, weights, place})
    if (tokens > 1 && t->stride[0] != choose) return fail(ACC_ERR_INVALID, "%s: experts, weights and place are dense arrays", who);
  const int bytes = type_bytes(op->spec.type);
  const Named all[] = {{chosen, 4, "experts"}, {weights, 4, "weights"}, {offsets, 4, "offsets"}, {order, 4, "order"}, {place, 4, "place"}};
  for (int k = 0; k < 5; ++k) {
    ACC_TRY(check_apart(who, all[k], {{logits, bytes, "logits"}}));
    for (int m = 0; m < k; ++m) ACC_TRY(check_apart(who, all[k], {all[m]}));
  }
  return ACC_OK;
}

int acc_exec_route(acc_op op, const acc_strided *logits, const acc_strided *chosen, const acc_strided *weights, const acc_strided *offsets,
                   const acc_strided *order, const acc_strided *place, acc_stream stream)
try {
  const char *who = "acc_exec_route";
  acc_route_args a = {};
  ACC_TRY(begin(op, ACC_OP_ROUTE, who, stream, &a.guard));
  ACC_TRY(check_routing(op, who, logits, chosen, weights, offsets, order, place));
  const int64_t tokens = logits->shape[0], experts = logits->shape[1], choose = op->spec.choose;
  const int bytes = type_bytes(op->spec.type);
  const RouteVariant v = route_variant(op->spec, (int)experts, aligned_rows(*logits, bytes, 1), tokens);
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kRouteNames, 3, route_source_of, &var));
  a.logits = device<const void>(logits);
  a.chosen = device<int32_t>(chosen);
  a.weights = device<float>(weights);
  a.offsets = device<int32_t>(offsets);
  a.order = device<int32_t>(order);
  a.place = device<int32_t>(place);
  a.tokens = tokens;
  a.logits_stride = logits->stride[0];
  a.experts = (int32_t)experts;
  a.choose = (int32_t)choose;
  a.normalise = op->spec.normalise ? 1 : 0;
  a.block = route_block(v, tokens, experts);
  a.blocks = (int32_t)std::max<int64_t>(1, ceil_div(tokens, a.block));
  acc::ScratchRef scratch;
  if (a.blocks > 1) {
    ACC_TRY(scratch_of(op, stream, (size_t)a.blocks * (size_t)experts * 4, &scratch));
    a.counts = static_cast<uint32_t *>(scratch.ptr);
  }
  int rc = v.tall ? launch(op, who, var->fn, a.blocks, kRouteTallThreads * v.halves, (size_t)experts * 4, stream, a)
                  : launch(op, who, var->fn, a.blocks, v.threads(), route_lds(v, experts, a.blocks == 1 ? tokens * choose : 0), stream, a);
  if (rc == ACC_OK && a.blocks > 1) rc = launch(op, who, var->fn2, a.blocks, kRouteThreads, route_lds(v, experts, 0), stream, a);
  if (a.blocks > 1) op->ctx->scratch_release(scratch, static_cast<hipStream_t>(stream));
  return rc;
} ACC_OP_CATCH("acc_exec_route")

int acc_exec_route_gradient(acc_op op, const acc_strided *logits, const acc_strided *chosen, const acc_strided *weights, const acc_strided *dweights,
                            const acc_strided *dlogits, acc_stream stream)
try {
  const char *who = "acc_exec_route_gradient";
  acc_route_args a = {};
  ACC_TRY(begin(op, ACC_OP_ROUTE, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "logits", logits, 2));
  ACC_TRY(check_unit(who, "experts", chosen, 2));
  ACC_TRY(check_unit(who, "weights", weights, 2));
  ACC_TRY(check_unit(who, "dweights", dweights, 2));
  ACC_TRY(check_result(who, "dlogits", dlogits, 2));
  const int64_t tokens = logits->shape[0], experts = logits->shape[1], choose = op->spec.choose;
  if (experts < choose || experts > kRouteMaxExperts)
    return fail(ACC_ERR_INVALID, "%s: %lld experts (at least the %lld that are chosen, and at most %d)", who, (long long)experts, (long long)choose, kRouteMaxExperts);
  ACC_TRY(check_shape(who, "experts", *chosen, {tokens, choose}));
  ACC_TRY(check_shape(who, "weights", *weights, {tokens, choose}));
  ACC_TRY(check_shape(who, "dweights", *dweights, {tokens, choose}));
  ACC_TRY(check_shape(who, "dlogits", *dlogits, {tokens, experts}));
  for (const acc_strided *t : {chosen, weights, dweights})
    if (tokens > 1 && t->stride[0] != choose) return fail(ACC_ERR_INVALID, "%s: experts, weights and dweights are dense arrays", who);
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {dlogits, bytes, "dlogits"}, {{logits, bytes, "logits"}, {chosen, 4, "experts"}, {weights, 4, "weights"}, {dweights, 4, "dweights"}}));
  if (tokens == 0) return ACC_OK;
  const RouteVariant v = route_variant(op->spec, (int)experts, aligned_rows(*logits, bytes, 1) && aligned_rows(*dlogits, bytes, 1), 0);
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kRouteNames, 3, route_source_of, &var));
  a.logits = device<const void>(logits);
  a.chosen = device<int32_t>(chosen);
  a.weights = device<float>(weights);
  a.dweights = device<const float>(dweights);
  a.dlogits = device<void>(dlogits);
  a.tokens = tokens;
  a.logits_stride = logits->stride[0];
  a.dlogits_stride = dlogits->stride[0];
  a.experts = (int32_t)experts;
  a.choose = (int32_t)choose;
  a.normalise = op->spec.normalise ? 1 : 0;
  const int64_t each = kRouteThreads / v.lanes, most = kThreads / kRouteThreads * each;
  for (int64_t first = 0; first < tokens; first += most) {
    acc_route_args part = a;
    part.tokens = std::min(most, tokens - first);
    part.logits = static_cast<const char *>(a.logits) + first * a.logits_stride * bytes;
    part.dlogits = static_cast<char *>(a.dlogits) + first * a.dlogits_stride * bytes;
    part.chosen = a.chosen + first * choose;
    part.weights = a.weights + first * choose;
    part.dweights = a.dweights + first * choose;
    ACC_TRY(launch(op, who, var->fn3, ceil_div(part.tokens, each), kRouteThreads, 0, stream, part));
  }
  return ACC_OK;
} ACC_OP_CATCH("acc_exec_route_gradient")

// ---- router by scores -------------------------------------------------------------------

static int check_score_experts(acc_op op, const char *who, int64_t experts)
{
  const OpSpec &sp = op->spec;
  if (experts > kRouteMaxExperts || experts % sp.groups != 0 || experts / sp.groups * sp.keep < sp.choose)
    return fail(ACC_ERR_INVALID, "%s: %lld experts (a multiple of %d, at most %d; %d are chosen of those of %d groups)", who, (long long)experts, sp.groups, kRouteMaxExperts, sp.choose, sp.keep);
  return ACC_OK;
}

int acc_exec_score(acc_op op, const acc_strided *logits, const acc_strided *bias, const acc_strided *chosen, const acc_strided *weights,
                   const acc_strided *offsets, const acc_strided *order, const acc_strided *place, acc_stream stream)
try {
  const char *who = "acc_exec_score";
  acc_route_args a = {};
  ACC_TRY(begin(op, ACC_OP_SCORE, who, stream, &a.guard));
  ACC_TRY(check_routing(op, who, logits, chosen, weights, offsets, order, place));
  const int64_t tokens = logits->shape[0], experts = logits->shape[1], choose = op->spec.choose;
  ACC_TRY(check_score_experts(op, who, experts));
  if (bias) {
    ACC_TRY(check_unit(who, "bias", bias, 1));
    ACC_TRY(check_shape(who, "bias", *bias, {experts}));
    for (const Named &n : {Named{chosen, 4, "experts"}, Named{weights, 4, "weights"}, Named{offsets, 4, "offsets"}, Named{order, 4, "order"}, Named{place, 4, "place"}})
      ACC_TRY(check_apart(who, n, {{bias, 4, "bias"}}));
  }
  const ScoreVariant v = score_variant(op->spec, experts, tokens);
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kScoreNames, 3, score_source_of, &var));
  a.logits = device<const void>(logits);
  a.bias = device<const float>(bias);
  a.chosen = device<int32_t>(chosen);
  a.weights = device<float>(weights);
  a.offsets = device<int32_t>(offsets);
  a.order = device<int32_t>(order);
  a.place = device<int32_t>(place);
  a.tokens = tokens;
  a.logits_stride = logits->stride[0];
  a.experts = (int32_t)experts;
  a.choose = (int32_t)choose;
  a.normalise = op->spec.normalise ? 1 : 0;
  a.groups = op->spec.groups;
  a.keep = op->spec.keep;
  a.scale = op->spec.scale;
  // (as the other router's: a single workgroup, or up to 256 of which each reads the counts of all)
  const int64_t at_once = v.threads() / v.lanes;
  a.block = v.few ? (int)std::max<int64_t>(1, tokens) : (int)std::max<int64_t>(at_once, ceil_div(ceil_div(tokens, 256), at_once) * at_once);
  a.blocks = (int32_t)std::max<int64_t>(1, ceil_div(tokens, a.block));
  const size_t groups = (size_t)at_once * (size_t)op->spec.groups * 8;
  if (v.few) return launch(op, who, var->fn, 1, v.threads(), (size_t)(6 * experts + tokens * choose) * 4 + groups, stream, a);
  ScratchHold counts;
  ACC_TRY(counts.acquire(op, stream, (size_t)a.blocks * (size_t)experts * 4));
  a.counts = static_cast<uint32_t *>(counts.ref.ptr);
  ACC_TRY(launch(op, who, var->fn, a.blocks, v.threads(), (size_t)experts * 4 + groups, stream, a));
  return launch(op, who, var->fn2, a.blocks, kRouteThreads, ((size_t)(kRouteThreads / 64 + 2) * (size_t)experts) * 4, stream, a);
} ACC_OP_CATCH("acc_exec_score")

int acc_exec_score_gradient(acc_op op, const acc_strided *logits, const acc_strided *chosen, const acc_strided *dweights, const acc_strided *dlogits, acc_stream stream)
try {
  const char *who = "acc_exec_score_gradient";
  acc_route_args a = {};
  ACC_TRY(begin(op, ACC_OP_SCORE, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "logits", logits, 2));
  ACC_TRY(check_unit(who, "experts", chosen, 2));
  ACC_TRY(check_unit(who, "dweights", dweights, 2));
  ACC_TRY(check_result(who, "dlogits", dlogits, 2));
  const int64_t tokens = logits->shape[0], experts = logits->shape[1], choose = op->spec.choose;
  ACC_TRY(check_score_experts(op, who, experts));
  ACC_TRY(check_shape(who, "experts", *chosen, {tokens, choose}));
  ACC_TRY(check_shape(who, "dweights", *dweights, {tokens, choose}));
  ACC_TRY(check_shape(who, "dlogits", *dlogits, {tokens, experts}));
  for (const acc_strided *t : {chosen, dweights})
    if (tokens > 1 && t->stride[0] != choose) return fail(ACC_ERR_INVALID, "%s: experts and dweights are dense arrays", who);
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {dlogits, bytes, "dlogits"}, {{logits, bytes, "logits"}, {chosen, 4, "experts"}, {dweights, 4, "dweights"}}));
  if (tokens == 0) return ACC_OK;
  ScoreVariant v;                                  // (any: the gradient is the same in all)
  v.lanes = 64;
  v.per = 8;
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kScoreNames, 3, score_source_of, &var));
  a.logits = device<const void>(logits);
  a.chosen = device<int32_t>(chosen);
  a.dweights = device<const float>(dweights);
  a.dlogits = device<void>(dlogits);
  a.logits_stride = logits->stride[0];
  a.dlogits_stride = dlogits->stride[0];
  a.experts = (int32_t)experts;
  a.choose = (int32_t)choose;
  a.normalise = op->spec.normalise ? 1 : 0;
  a.scale = op->spec.scale;
  const int64_t each = 256 / 32, most = kThreads / 256 * each;      // (tokens of a workgroup: 32 lanes each)
  for (int64_t first = 0; first < tokens; first += most) {
    acc_route_args part = a;
    part.tokens = std::min(most, tokens - first);
    part.logits = static_cast<const char *>(a.logits) + first * a.logits_stride * bytes;
    part.dlogits = static_cast<char *>(a.dlogits) + first * a.dlogits_stride * bytes;
    part.chosen = a.chosen + first * choose;
    part.dweights = a.dweights + first * choose;
    ACC_TRY(launch(op, who, var->fn3, ceil_div(part.tokens, each), 256, 0, stream, part));
  }
  return ACC_OK;
} ACC_OP_CATCH("acc_exec_score_gradient")

// ---- combination ----------------------------------------------------------------------

static int check_slots(const char *who, const acc_strided *place, const acc_strided *weights, int64_t tokens)
{
  ACC_TRY(check_unit(who, "place", place, 2));
  ACC_TRY(check_shape(who, "place", *place, {tokens, place->shape[1]}));
  if (tokens > 1 && place->stride[0] != place->shape[1]) return fail(ACC_ERR_INVALID, "%s: place is a dense array", who);
  if (!weights) return ACC_OK;
  ACC_TRY(check_unit(who, "weights", weights, 2));
  ACC_TRY(check_shape(who, "weights", *weights, {tokens, place->shape[1]}));
  if (tokens > 1 && weights->stride[0] != weights->shape[1]) return fail(ACC_ERR_INVALID, "%s: weights is a dense array", who);
  return ACC_OK;
}

int acc_exec_combine(acc_op op, const acc_strided *y, const acc_strided *place, const acc_strided *weights, const acc_strided *out, acc_stream stream)
try {
  const char *who = "acc_exec_combine";
  acc_combine_args a = {};
  ACC_TRY(begin(op, ACC_OP_COMBINE, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "y", y, 2));
  ACC_TRY(check_result(who, "the result", out, 2));
  const int64_t tokens = out->shape[0], width = out->shape[1];
  ACC_TRY(check_slots(who, place, weights, tokens));
  ACC_TRY(check_shape(who, "y", *y, {y->shape[0], width}));
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {out, bytes, "the result"}, {{y, bytes, "y"}, {place, 4, "place"}, {weights, 4, "weights"}}));
  if (is_empty(*out)) return ACC_OK;
  const bool aligned = width % 8 == 0 && aligned_rows(*y, bytes, 1) && aligned_rows(*out, bytes, 1);
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(aligned ? 1u : width < 8 ? 2u : 0u, kCombineNames, 2, combine_source_of, &var));
  a.y = device<const void>(y);
  a.out = device<void>(out);
  a.place = device<const int32_t>(place);
  a.weights = device<const float>(weights);
  a.tokens = tokens;
  a.y_rows = y->shape[0];
  a.y_stride = y->stride[0];
  a.out_stride = out->stride[0];
  a.choose = (int32_t)place->shape[1];
  a.width = (int32_t)width;
  const int64_t pieces = ceil_div(width, 8), most = std::max<int64_t>(1, 0x7fffff00 / pieces);
  set_divisor((int32_t)pieces, &a);
  for (int64_t first = 0; first < tokens; first += most) {           // (a lane's number has 31 bits)
    acc_combine_args part = a;
    part.tokens = std::min(most, tokens - first);
    part.out = static_cast<char *>(a.out) + first * a.out_stride * bytes;
    part.place = a.place + first * a.choose;
    part.weights = a.weights ? a.weights + first * a.choose : nullptr;
    ACC_TRY(launch(op, who, var->fn, ceil_div(part.tokens * pieces, 256), 256, 0, stream, part));
  }
  return ACC_OK;
} ACC_OP_CATCH("acc_exec_combine")

int acc_exec_combine_gradient(acc_op op, const acc_strided *dout, const acc_strided *y, const acc_strided *place, const acc_strided *weights,
                              const acc_strided *dy, const acc_strided *dweights, acc_stream stream)
try {
  const char *who = "acc_exec_combine_gradient";
  acc_combine_args a = {};
  ACC_TRY(begin(op, ACC_OP_COMBINE, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "dout", dout, 2));
  ACC_TRY(check_result(who, "dy", dy, 2));
  const int64_t tokens = dout->shape[0], width = dout->shape[1];
  ACC_TRY(check_slots(who, place, weights, tokens));
  ACC_TRY(check_shape(who, "dy", *dy, {dy->shape[0], width}));
  if ((dweights != nullptr) != (y != nullptr)) return fail(ACC_ERR_INVALID, "%s: y and dweights go together", who);
  if (y) {
    ACC_TRY(check_unit(who, "y", y, 2));
    ACC_TRY(check_shape(who, "y", *y, {dy->shape[0], width}));
    ACC_TRY(check_result(who, "dweights", dweights, 2));
    ACC_TRY(check_shape(who, "dweights", *dweights, {tokens, place->shape[1]}));
    if (tokens > 1 && dweights->stride[0] != dweights->shape[1]) return fail(ACC_ERR_INVALID, "%s: dweights is a dense array", who);
  }
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {dy, bytes, "dy"}, {{dout, bytes, "dout"}, {y, bytes, "y"}, {place, 4, "place"}, {weights, 4, "weights"}, {dweights, 4, "dweights"}}));
  if (dweights) ACC_TRY(check_apart(who, {dweights, 4, "dweights"}, {{dout, bytes, "dout"}, {y, bytes, "y"}, {place, 4, "place"}, {weights, 4, "weights"}}));
  if (tokens == 0 || place->shape[1] == 0) return ACC_OK;
  const bool aligned = width % 8 == 0 && aligned_rows(*dout, bytes, 1) && aligned_rows(*dy, bytes, 1) && (!y || aligned_rows(*y, bytes, 1));
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(aligned ? 1u : width < 8 ? 2u : 0u, kCombineNames, 2, combine_source_of, &var));
  a.y = device<const void>(y);
  a.dout = device<const void>(dout);
  a.out = device<void>(dy);
  a.place = device<const int32_t>(place);
  a.weights = device<const float>(weights);
  a.dweights = device<float>(dweights);
  a.tokens = tokens;
  a.y_rows = dy->shape[0];
  a.y_stride = y ? y->stride[0] : 0;
  a.out_stride = dy->stride[0];
  a.dout_stride = dout->stride[0];
  a.choose = (int32_t)place->shape[1];
  a.width = (int32_t)width;
  const int block = 64 * (int)std::max<int64_t>(1, std::min<int64_t>(4, ceil_div(width, 512)));
  const int64_t most = kThreads / block;
  for (int64_t first = 0; first < tokens; first += most) {
    acc_combine_args part = a;
    part.tokens = std::min(most, tokens - first);
    part.dout = static_cast<const char *>(a.dout) + first * a.dout_stride * bytes;
    part.place = a.place + first * a.choose;
    part.weights = a.weights ? a.weights + first * a.choose : nullptr;
    part.dweights = a.dweights ? a.dweights + first * a.choose : nullptr;
    ACC_TRY(launch(op, who, var->fn2, part.tokens, block, 0, stream, part));
  }
  return ACC_OK;
} ACC_OP_CATCH("acc_exec_combine_gradient")

// ---- 4-bit numbers --------------------------------------------------------------------

// codes and scales of `rows` rows of `k` elements (in `batches` matrices where the arrays have rank 3)
static int check_micro(const char *who, const char *what, const acc_strided *codes, const acc_strided *scales, int rank, bool result)
{
  ACC_TRY(result ? check_result(who, what, codes, rank) : check_unit(who, what, codes, rank));
  ACC_TRY(result ? check_result(who, what, scales, rank) : check_unit(who, what, scales, rank));
  for (int d = 0; d < rank - 1; ++d)
    if (codes->shape[d] != scales->shape[d]) return fail(ACC_ERR_INVALID, "%s: %s: codes of %lld rows, scales of %lld", who, what, (long long)codes->shape[d], (long long)scales->shape[d]);
  if (codes->shape[rank - 1] != 16 * scales->shape[rank - 1])
    return fail(ACC_ERR_INVALID, "%s: %s: a row of %lld bytes of codes and %lld scales (16 bytes a scale)", who, what, (long long)codes->shape[rank - 1], (long long)scales->shape[rank - 1]);
  if (!aligned_rows(*codes, 1, rank - 1)) return fail(ACC_ERR_INVALID, "%s: %s: rows of codes start on 16 bytes", who, what);
  return ACC_OK;
}

static int micro_elements(acc_op op, const char *who, bool back, const acc_strided *x, const acc_strided *codes, const acc_strided *scales, acc_stream stream, acc_micro_args a)
{
  const int bytes = type_bytes(op->spec.type), epc = 16 / bytes;
  const int64_t rows = x->shape[0], k = x->shape[1], blocks = ceil_div(k, 32);
  ACC_TRY(check_shape(who, "codes", *codes, {rows, 16 * blocks}));
  if (is_empty(*x)) return ACC_OK;
  const bool aligned = k % epc == 0 && aligned_rows(*x, bytes, 1);
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(kMicroElements | (aligned ? 1u : 0u), kMicroNames, 2, micro_source_of, &var));
  a.x = device<const void>(x);
  a.out = device<void>(x);
  a.codes = device<uint8_t>(codes);
  a.scales = device<uint8_t>(scales);
  a.rows = rows;
  a.x_stride = x->stride[0];
  a.codes_stride = codes->stride[0];
  a.scales_stride = scales->stride[0];
  a.k = (int32_t)k;
  a.blocks = (int32_t)blocks;
  set_divisor((int32_t)blocks, &a);
  // (four threads a block)
  const int64_t most = std::max<int64_t>(1, (kThreads - 255) / 4 / blocks);
  for (int64_t first = 0; first < rows; first += most) {
    acc_micro_args part = a;
    part.rows = std::min(most, rows - first);
    part.x = static_cast<const char *>(a.x) + first * a.x_stride * bytes;
    part.out = static_cast<char *>(a.out) + first * a.x_stride * bytes;
    part.codes = a.codes + first * a.codes_stride;
    part.scales = a.scales + first * a.scales_stride;
    ACC_TRY(launch(op, who, back ? var->fn2 : var->fn, ceil_div(part.rows * blocks * 4, 256), 256, 0, stream, part));
  }
  return ACC_OK;
}

int acc_exec_micro_quantise(acc_op op, const acc_strided *x, const acc_strided *codes, const acc_strided *scales, acc_stream stream)
try {
  const char *who = "acc_exec_micro_quantise";
  acc_micro_args a = {};
  ACC_TRY(begin(op, ACC_OP_MICRO, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "x", x, 2));
  ACC_TRY(check_micro(who, "the result", codes, scales, 2, true));
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {codes, 1, "codes"}, {{x, bytes, "x"}, {scales, 1, "scales"}}));
  ACC_TRY(check_apart(who, {scales, 1, "scales"}, {{x, bytes, "x"}}));
  return micro_elements(op, who, false, x, codes, scales, stream, a);
} ACC_OP_CATCH("acc_exec_micro_quantise")

int acc_exec_micro_values(acc_op op, const acc_strided *codes, const acc_strided *scales, const acc_strided *out, acc_stream stream)
try {
  const char *who = "acc_exec_micro_values";
  acc_micro_args a = {};
  ACC_TRY(begin(op, ACC_OP_MICRO, who, stream, &a.guard));
  ACC_TRY(check_result(who, "the result", out, 2));
  ACC_TRY(check_micro(who, "x", codes, scales, 2, false));
  ACC_TRY(check_apart(who, {out, type_bytes(op->spec.type), "the result"}, {{codes, 1, "codes"}, {scales, 1, "scales"}}));
  return micro_elements(op, who, true, out, codes, scales, stream, a);
} ACC_OP_CATCH("acc_exec_micro_values")

int acc_exec_micro_rows(acc_op op, const acc_strided *xcodes, const acc_strided *xscales, const acc_strided *wcodes, const acc_strided *wscales,
                        const acc_strided *offsets, const acc_strided *index, int32_t per, const acc_strided *out, acc_stream stream)
try {
  const char *who = "acc_exec_micro_rows";
  acc_product_args a = {};
  ACC_TRY(begin(op, ACC_OP_MICRO, who, stream, &a.guard));
  ACC_TRY(check_micro(who, "x", xcodes, xscales, 2, false));
  ACC_TRY(check_micro(who, "w", wcodes, wscales, 3, false));
  ACC_TRY(check_unit(who, "offsets", offsets, 1));
  ACC_TRY(check_result(who, "the result", out, 2));
  if (index) ACC_TRY(check_unit(who, "index", index, 1));
  if (per < 0) return fail(ACC_ERR_INVALID, "%s: a divisor of %d", who, per);
  const int64_t experts = wscales->shape[0], n = wscales->shape[1], blocks = wscales->shape[2], rows = out->shape[0];
  ACC_TRY(check_shape(who, "offsets", *offsets, {experts + 1}));
  ACC_TRY(check_shape(who, "the result", *out, {rows, n}));
  if (index) ACC_TRY(check_shape(who, "index", *index, {rows}));
  ACC_TRY(check_shape(who, "x", *xscales, {index ? xscales->shape[0] : rows, blocks}));
  ACC_TRY(check_extents(who, {experts, n, wcodes->shape[2], rows, xcodes->shape[0]}));
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {out, bytes, "the result"}, {{xcodes, 1, "x"}, {xscales, 1, "x's scales"}, {wcodes, 1, "w"}, {wscales, 1, "w's scales"}, {offsets, 4, "offsets"}, {index, 4, "index"}}));
  if (is_empty(*out)) return ACC_OK;
  ProductVariant v;
  // (codes lie on 16 bytes; scales are taken four at a time where every row of them starts on 4 bytes and is whole fours)
  v.fours = blocks % 4 == 0;
  v.tiny = blocks < 4;
  v.aligned = near_enough(*xcodes, 0, 16 * blocks, 1, index != nullptr) && near_enough(*wcodes, 1, 16 * blocks, 1, false) &&
              near_enough(*xscales, 0, blocks, 1, true) && near_enough(*wscales, 1, blocks, 1, true);
  for (const acc_strided *t : {xscales, wscales}) {
    v.fours = v.fours && t->ptr % 4 == 0;
    for (int d = 0; d + 1 < t->rank; ++d) v.fours = v.fours && (t->shape[d] <= 1 || t->stride[d] % 4 == 0);
  }
  v.tile = tile_of(op->spec, v, rows_tile(op->spec, v, rows, experts, n, ceil_div(blocks, 8)));
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kProductNames, v.tile >= kSkinny ? 1 : 2, micro_source_of, &var));
  a.a = device<const void>(xcodes);
  a.b = device<const void>(wcodes);
  a.a_scales = device<const uint8_t>(xscales);
  a.b_scales = device<const uint8_t>(wscales);
  a.out = device<void>(out);
  a.offsets = device<const int32_t>(offsets);
  a.index_a = device<const int32_t>(index);
  a.a_stride = xcodes->stride[0];
  a.a_scales_stride = xscales->stride[0];
  a.b_stride = wcodes->stride[1];
  a.b_expert = wcodes->stride[0];
  a.b_scales_stride = wscales->stride[1];
  a.b_scales_expert = wscales->stride[0];
  a.out_stride = out->stride[0];
  a.rows = rows;
  a.a_rows = (int32_t)xscales->shape[0];
  a.nj = (int32_t)n;
  a.k = (int32_t)(16 * blocks);
  a.experts = (int32_t)experts;
  set_divisor(per, &a);
  return launch_rows(op, who, v, var, a, stream);
} ACC_OP_CATCH("acc_exec_micro_rows")

// ---- 4-bit whole numbers in groups --------------------------------------------------------

// codes [experts, n, 16 blocks], scales and zeros [experts, groups, n] of matrices of k columns (k 0: as many as the codes have)
static int check_grouped(acc_op op, const char *who, const acc_strided *codes, const acc_strided *scales, const acc_strided *zeros, int64_t k, bool result, acc_grouped_args *a)
{
  ACC_TRY(result ? check_result(who, "codes", codes, 3) : check_unit(who, "codes", codes, 3));
  ACC_TRY(result ? check_result(who, "scales", scales, 3) : check_unit(who, "scales", scales, 3));
  if (zeros) ACC_TRY(result ? check_result(who, "zeros", zeros, 3) : check_unit(who, "zeros", zeros, 3));
  const int64_t experts = codes->shape[0], n = codes->shape[1], blocks = ceil_div(k, 32), groups = ceil_div(k, op->spec.group);
  ACC_TRY(check_shape(who, "codes", *codes, {experts, n, 16 * blocks}));
  ACC_TRY(check_shape(who, "scales", *scales, {experts, groups, n}));
  if (zeros) ACC_TRY(check_shape(who, "zeros", *zeros, {experts, groups, n}));
  if (!aligned_rows(*codes, 1, 2)) return fail(ACC_ERR_INVALID, "%s: rows of codes start on 16 bytes", who);
  ACC_TRY(check_extents(who, {experts, n, k}));
  if (k > (1 << 30)) return fail(ACC_ERR_INVALID, "%s: rows of %lld numbers", who, (long long)k);
  a->codes = device<void>(codes);
  a->scales = device<void>(scales);
  a->zeros = device<void>(zeros);
  a->codes_expert = codes->stride[0];
  a->codes_stride = codes->stride[1];
  a->scales_expert = scales->stride[0];
  a->scales_stride = scales->stride[1];
  a->zeros_expert = zeros ? zeros->stride[0] : 0;
  a->zeros_stride = zeros ? zeros->stride[1] : 0;
  a->experts = (int32_t)experts;
  a->nj = (int32_t)n;
  a->k = (int32_t)k;
  a->blocks = (int32_t)blocks;
  a->group = (int32_t)std::min<int64_t>(op->spec.group, int64_t(1) << 30);
  a->groups = (int32_t)groups;
  for (a->group_shift = 5; (1 << a->group_shift) < a->group; ++a->group_shift) {}
  return ACC_OK;
}

static int launch_elements(acc_op op, const char *who, bool back, int64_t threads, acc_grouped_args &a, acc_stream stream)
{
  GroupedVariant v;
  v.elements = true;
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kGroupedElementNames, 2, grouped_source_of, &var));
  const int64_t groups = ceil_div(threads, 256), most = kThreads / 256;
  for (int64_t first = 0; first < groups; first += most) {
    a.first = first * 256;
    ACC_TRY(launch(op, who, back ? var->fn2 : var->fn, std::min(most, groups - first), 256, 0, stream, a));
  }
  return ACC_OK;
}

int acc_exec_grouped_quantise(acc_op op, const acc_strided *w, const acc_strided *codes, const acc_strided *scales, const acc_strided *zeros, acc_stream stream)
try {
  const char *who = "acc_exec_grouped_quantise";
  acc_grouped_args a = {};
  ACC_TRY(begin(op, ACC_OP_GROUPED, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "w", w, 3));
  ACC_TRY(check_grouped(op, who, codes, scales, zeros, w->shape[2], true, &a));
  ACC_TRY(check_shape(who, "w", *w, {codes->shape[0], codes->shape[1], w->shape[2]}));
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {codes, 1, "codes"}, {{w, bytes, "w"}, {scales, bytes, "scales"}, {zeros, 1, "zeros"}}));
  ACC_TRY(check_apart(who, {scales, bytes, "scales"}, {{w, bytes, "w"}, {zeros, 1, "zeros"}}));
  if (zeros) ACC_TRY(check_apart(who, {zeros, 1, "zeros"}, {{w, bytes, "w"}}));
  if (is_empty(*w)) return ACC_OK;
  a.w = device<const void>(w);
  a.w_expert = w->stride[0];
  a.w_stride = w->stride[1];
  return launch_elements(op, who, false, (int64_t)a.experts * a.nj * a.groups * std::min(64, a.group / 8), a, stream);
} ACC_OP_CATCH("acc_exec_grouped_quantise")

int acc_exec_grouped_values(acc_op op, const acc_strided *codes, const acc_strided *scales, const acc_strided *zeros, const acc_strided *out, acc_stream stream)
try {
  const char *who = "acc_exec_grouped_values";
  acc_grouped_args a = {};
  ACC_TRY(begin(op, ACC_OP_GROUPED, who, stream, &a.guard));
  ACC_TRY(check_result(who, "the result", out, 3));
  ACC_TRY(check_grouped(op, who, codes, scales, zeros, out->shape[2], false, &a));
  ACC_TRY(check_shape(who, "the result", *out, {codes->shape[0], codes->shape[1], out->shape[2]}));
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {out, bytes, "the result"}, {{codes, 1, "codes"}, {scales, bytes, "scales"}, {zeros, 1, "zeros"}}));
  if (is_empty(*out)) return ACC_OK;
  a.out = device<void>(out);
  a.out_expert = out->stride[0];
  a.out_stride = out->stride[1];
  return launch_elements(op, who, true, (int64_t)a.experts * a.nj * a.blocks * 4, a, stream);
} ACC_OP_CATCH("acc_exec_grouped_values")

int acc_exec_grouped_rows(acc_op op, const acc_strided *x, const acc_strided *codes, const acc_strided *scales, const acc_strided *zeros,
                          const acc_strided *offsets, const acc_strided *index, int32_t per, const acc_strided *out, acc_stream stream)
try {
  const char *who = "acc_exec_grouped_rows";
  acc_grouped_args a = {};
  ACC_TRY(begin(op, ACC_OP_GROUPED, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "x", x, 2));
  ACC_TRY(check_grouped(op, who, codes, scales, zeros, x->shape[1], false, &a));
  ACC_TRY(check_unit(who, "offsets", offsets, 1));
  ACC_TRY(check_result(who, "the result", out, 2));
  if (index) ACC_TRY(check_unit(who, "index", index, 1));
  if (per < 0) return fail(ACC_ERR_INVALID, "%s: a divisor of %d", who, per);
  const int64_t experts = a.experts, n = a.nj, rows = out->shape[0], k = a.k;
  ACC_TRY(check_shape(who, "offsets", *offsets, {experts + 1}));
  ACC_TRY(check_shape(who, "the result", *out, {rows, n}));
  if (index) ACC_TRY(check_shape(who, "index", *index, {rows}));
  ACC_TRY(check_shape(who, "x", *x, {index ? x->shape[0] : rows, k}));
  ACC_TRY(check_extents(who, {rows, x->shape[0]}));
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {out, bytes, "the result"}, {{x, bytes, "x"}, {codes, 1, "codes"}, {scales, bytes, "scales"}, {zeros, 1, "zeros"}, {offsets, 4, "offsets"}, {index, 4, "index"}}));
  if (is_empty(*out)) return ACC_OK;
  const int64_t mean = ceil_div(rows, std::max<int64_t>(1, std::min(rows, experts)));
  const bool tall = grouped_tall(op->spec, rows, experts, n, k, codes->stride[1], mean);
  int64_t height = 0;
  GroupedVariant v;
  if (tall) {
    v.tall = true;
    height = op->spec.type == 0 ? 32 : 64;
  } else {
    v = grouped_variant(op->spec, rows, experts, n, k, codes->stride[1], mean, &height);
  }
  v.zeros = zeros != nullptr;
  a.x = device<const void>(x);
  a.out = device<void>(out);
  a.offsets = device<const int32_t>(offsets);
  a.index = device<const int32_t>(index);
  a.x_stride = x->stride[0];
  a.out_stride = out->stride[0];
  a.rows = rows;
  a.x_rows = (int32_t)x->shape[0];
  set_divisor(per, &a);
  a.tiles_i = (int32_t)tiles_at_most(rows, experts, height);
  a.height = (int32_t)height;
  a.run = v.fn;
  size_t lds = 0;
  if (v.tall) {
    a.run = 16;
    lds = (size_t)grouped_tall_lds(op->spec, v.zeros);
  }
  if (v.stream) {
    // a workgroup a compute unit; where it has fewer tiles of columns than waves, those share them
    const int64_t all = std::max(ceil_div(rows, height), std::min(rows, experts)) * ceil_div(n, 16);
    a.run = (int32_t)std::max<int64_t>(1, std::min(ceil_div(n, 16), ceil_div(all, v.wide == 8 ? 512 : 256)));
    a.split = 1;
    while (a.split < v.waves() && a.split * a.run < v.waves() && a.split < ceil_div(k, 128)) a.split *= 2;
    lds = (size_t)grouped_lds(op->spec, height, ceil_div(k, 128), v.waves());
    v.few = ceil_div(ceil_div(k, 128), a.split) <= 2;
  }
  a.tiles_j = (int32_t)ceil_div(n, 16 * a.run);
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kGroupedNames, 1, grouped_source_of, &var));
  return launch(op, who, var->fn, (int64_t)a.tiles_i * a.tiles_j, 64 * v.waves(), lds, stream, a);
} ACC_OP_CATCH("acc_exec_grouped_rows")

// ---- recurrence -------------------------------------------------------------------------

// states: a Float32 array of `width` columns, or none
static int check_states(const char *who, const char *what, const acc_strided *a, int64_t width, bool result)
{
  if (!a) return ACC_OK;
  ACC_TRY(result ? check_result(who, what, a, 2) : check_unit(who, what, a, 2));
  return check_shape(who, what, *a, {a->shape[0], width});
}

static bool same_array(const acc_strided &a, const acc_strided &b)
{
  return a.ptr == b.ptr && a.shape[0] == b.shape[0] && (a.shape[0] <= 1 || a.stride[0] == b.stride[0]);
}

// where sequences begin and end: states that are replaced in place are the same array
static int check_replaced(const char *who, const acc_strided *state, const acc_strided *last)
{
  if (!state || !last) return ACC_OK;
  if (state->shape[0] != last->shape[0]) return fail(ACC_ERR_INVALID, "%s: %lld states to begin with, %lld to end with", who, (long long)state->shape[0], (long long)last->shape[0]);
  return same_array(*state, *last) ? ACC_OK : check_apart(who, {last, 4, "last"}, {{state, 4, "state"}});
}

// the tiles of all rows, forward or back: a.gates ... are there, the rest is filled in
static int launch_recur(acc_op op, const char *who, bool back, acc_recur_args &a, acc_stream stream)
{
  const hipStream_t st = static_cast<hipStream_t>(stream);
  RecurVariant v;
  v.back = back;
  v.thin = op->spec.type != 0 && a.width <= 64;
  const int64_t channels = v.channels(op->spec.type);
  v.rows = recur_rows(back, a.rows, ceil_div(a.width, channels));
  const int64_t tiles = std::max<int64_t>(1, ceil_div(a.rows, (int64_t)kRecurWaves * v.rows)), strips = ceil_div(a.width, channels);
  if (tiles * strips > kThreads / (64 * kRecurWaves)) return fail(ACC_ERR_INVALID, "%s: %lld rows of %d channels are too many", who, (long long)a.rows, a.width);
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kRecurNames, 2, recur_source_of, &var));
  a.tiles = (int32_t)tiles;
  a.strips = (int32_t)strips;
  a.status = reinterpret_cast<uint32_t *>(op->ctx->status_dev);
  const int64_t words = tiles * strips * 3 * channels;
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(st, &capture) != hipSuccess) (void)hipGetLastError();
  const bool recorded = capture != hipStreamCaptureStatusNone;
  // Workgroups that wait for others are the device's alone, as with the scans; what runs beside a graph nobody knows, so there tiles
  // are drawn in the order in which workgroups start, and so they are where the last call's stream is being recorded and cannot be waited for.
  bool drawn = recorded;
  if (tiles > 1 && !recorded) ACC_TRY(acc::scan_order_before(op->ctx->device, st, &drawn));
  const bool ordered = tiles > 1 && !drawn;
  acc::ScratchRef scratch;
  int rc = op->ctx->scratch_acquire(256 + (size_t)words * 8, st, acc::SCRATCH_FLAGS, &scratch, recorded);
  if (rc == ACC_OK) {
    a.words = reinterpret_cast<uint64_t *>(static_cast<char *>(scratch.ptr) + 256);
    a.tag = scratch.epoch;
    if (drawn) {
      a.ticket = static_cast<uint32_t *>(scratch.ptr);
      rc = launch(op, who, var->fn2, ceil_div(words, 256), 256, 0, stream, a);
    }
    if (rc == ACC_OK) rc = launch(op, who, var->fn, tiles * strips, 64 * kRecurWaves, 0, stream, a);
    op->ctx->scratch_release(scratch, st);
  }
  if (ordered) acc::scan_order_after(op->ctx->device);
  return rc;
}

int acc_exec_recur(acc_op op, const acc_strided *gates, const acc_strided *values, const acc_strided *offsets, const acc_strided *index,
                   const acc_strided *state, const acc_strided *last, const acc_strided *out, acc_stream stream)
try {
  const char *who = "acc_exec_recur";
  acc_recur_args a = {};
  ACC_TRY(begin(op, ACC_OP_RECUR, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "gates", gates, 2));
  ACC_TRY(check_unit(who, "values", values, 2));
  ACC_TRY(check_unit(who, "offsets", offsets, 1));
  ACC_TRY(check_result(who, "the result", out, 2));
  if (index) ACC_TRY(check_unit(who, "index", index, 1));
  const int64_t rows = out->shape[0], width = out->shape[1], sequences = offsets->shape[0] - 1;
  if (sequences < 0) return fail(ACC_ERR_INVALID, "%s: offsets are one more than sequences", who);
  ACC_TRY(check_shape(who, "gates", *gates, {rows, width}));
  ACC_TRY(check_shape(who, "values", *values, {rows, width}));
  if (index) ACC_TRY(check_shape(who, "index", *index, {sequences}));
  ACC_TRY(check_states(who, "state", state, width, false));
  ACC_TRY(check_states(who, "last", last, width, true));
  ACC_TRY(check_extents(who, {rows, width, sequences}));
  ACC_TRY(check_replaced(who, state, last));
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {out, bytes, "the result"}, {{gates, bytes, "gates"}, {values, bytes, "values"}, {offsets, 4, "offsets"}, {index, 4, "index"}, {state, 4, "state"}, {last, 4, "last"}}));
  if (last) ACC_TRY(check_apart(who, {last, 4, "last"}, {{gates, bytes, "gates"}, {values, bytes, "values"}, {offsets, 4, "offsets"}, {index, 4, "index"}}));
  if (width == 0 || sequences == 0 || (rows == 0 && !last)) return ACC_OK;
  a.gates = device<const void>(gates);
  a.values = device<const void>(values);
  a.out = device<void>(out);
  a.offsets = device<const int32_t>(offsets);
  a.index = device<const int32_t>(index);
  a.enter = device<const float>(state);
  a.leave = device<float>(last);
  a.gates_stride = gates->stride[0];
  a.values_stride = values->stride[0];
  a.out_stride = out->stride[0];
  a.enter_stride = state ? state->stride[0] : 0;
  a.leave_stride = last ? last->stride[0] : 0;
  a.rows = rows;
  a.width = (int32_t)width;
  a.sequences = (int32_t)sequences;
  a.states = (int32_t)(state ? state->shape[0] : last ? last->shape[0] : 0);
  return launch_recur(op, who, false, a, stream);
} ACC_OP_CATCH("acc_exec_recur")

int acc_exec_recur_gradient(acc_op op, const acc_strided *gates, const acc_strided *values, const acc_strided *offsets, const acc_strided *h,
                            const acc_strided *dout, const acc_strided *state, const acc_strided *dlast, const acc_strided *dgates,
                            const acc_strided *dvalues, const acc_strided *dstate, acc_stream stream)
try {
  const char *who = "acc_exec_recur_gradient";
  acc_recur_args a = {};
  ACC_TRY(begin(op, ACC_OP_RECUR, who, stream, &a.guard));
  if (op->spec.gate == ACC_GATE_GIVEN) values = nullptr;
  ACC_TRY(check_unit(who, "gates", gates, 2));
  if (op->spec.gate != ACC_GATE_GIVEN) ACC_TRY(check_unit(who, "values", values, 2));
  ACC_TRY(check_unit(who, "offsets", offsets, 1));
  ACC_TRY(check_unit(who, "h", h, 2));
  ACC_TRY(check_unit(who, "dout", dout, 2));
  ACC_TRY(check_result(who, "dgates", dgates, 2));
  ACC_TRY(check_result(who, "dvalues", dvalues, 2));
  const int64_t rows = dout->shape[0], width = dout->shape[1], sequences = offsets->shape[0] - 1;
  if (sequences < 0) return fail(ACC_ERR_INVALID, "%s: offsets are one more than sequences", who);
  const Named arrays[] = {{gates, 0, "gates"}, {values, 0, "values"}, {h, 0, "h"}, {dgates, 0, "dgates"}, {dvalues, 0, "dvalues"}};
  for (const Named &n : arrays)
    if (n.a) ACC_TRY(check_shape(who, n.what, *n.a, {rows, width}));
  const Named states[] = {{state, 0, "state"}, {dlast, 0, "dlast"}, {dstate, 1, "dstate"}};
  for (const Named &n : states)
    if (n.a) {
      ACC_TRY(check_states(who, n.what, n.a, width, n.bytes == 1));
      ACC_TRY(check_shape(who, n.what, *n.a, {sequences, width}));
    }
  ACC_TRY(check_extents(who, {rows, width, sequences}));
  if (dlast && dstate && !same_array(*dlast, *dstate)) ACC_TRY(check_apart(who, {dstate, 4, "dstate"}, {{dlast, 4, "dlast"}}));
  const int bytes = type_bytes(op->spec.type);
  const Named results[] = {{dgates, bytes, "dgates"}, {dvalues, bytes, "dvalues"}, {dstate, 4, "dstate"}};
  for (int k = 0; k < 3; ++k) {
    if (!results[k].a) continue;
    ACC_TRY(check_apart(who, results[k], {{gates, bytes, "gates"}, {values, bytes, "values"}, {offsets, 4, "offsets"}, {h, bytes, "h"}, {dout, bytes, "dout"}, {state, 4, "state"}}));
    if (k < 2) ACC_TRY(check_apart(who, results[k], {{dlast, 4, "dlast"}}));
    for (int m = 0; m < k; ++m) ACC_TRY(check_apart(who, results[k], {results[m]}));
  }
  if (width == 0 || sequences == 0 || (rows == 0 && !dstate)) return ACC_OK;
  a.gates = device<const void>(gates);
  a.values = device<const void>(values);
  a.h = device<const void>(h);
  a.dout = device<const void>(dout);
  a.dgates = device<void>(dgates);
  a.dvalues = device<void>(dvalues);
  a.offsets = device<const int32_t>(offsets);
  a.enter = device<const float>(dlast);
  a.leave = device<float>(dstate);
  a.state = device<const float>(state);
  a.gates_stride = gates->stride[0];
  a.values_stride = values ? values->stride[0] : 0;
  a.h_stride = h->stride[0];
  a.dout_stride = dout->stride[0];
  a.dgates_stride = dgates->stride[0];
  a.dvalues_stride = dvalues->stride[0];
  a.enter_stride = dlast ? dlast->stride[0] : 0;
  a.leave_stride = dstate ? dstate->stride[0] : 0;
  a.state_stride = state ? state->stride[0] : 0;
  a.rows = rows;
  a.width = (int32_t)width;
  a.sequences = a.states = (int32_t)sequences;
  return launch_recur(op, who, true, a, stream);
} ACC_OP_CATCH("acc_exec_recur_gradient")

int acc_exec_recur_step(acc_op op, const acc_strided *gates, const acc_strided *values, const acc_strided *index, const acc_strided *state,
                        const acc_strided *last, const acc_strided *out, acc_stream stream)
try {
  const char *who = "acc_exec_recur_step";
  acc_recur_args a = {};
  ACC_TRY(begin(op, ACC_OP_RECUR, who, stream, &a.guard));
  ACC_TRY(check_unit(who, "gates", gates, 2));
  ACC_TRY(check_unit(who, "values", values, 2));
  ACC_TRY(check_result(who, "the result", out, 2));
  if (index) ACC_TRY(check_unit(who, "index", index, 1));
  const int64_t rows = out->shape[0], width = out->shape[1];
  ACC_TRY(check_shape(who, "gates", *gates, {rows, width}));
  ACC_TRY(check_shape(who, "values", *values, {rows, width}));
  if (index) ACC_TRY(check_shape(who, "index", *index, {rows}));
  if (!state || !last) return fail(ACC_ERR_INVALID, "%s: %s missing", who, state ? "last" : "state");
  ACC_TRY(check_states(who, "state", state, width, false));
  ACC_TRY(check_states(who, "last", last, width, true));
  ACC_TRY(check_extents(who, {rows, width}));
  ACC_TRY(check_replaced(who, state, last));
  const int bytes = type_bytes(op->spec.type);
  ACC_TRY(check_apart(who, {out, bytes, "the result"}, {{gates, bytes, "gates"}, {values, bytes, "values"}, {index, 4, "index"}, {state, 4, "state"}, {last, 4, "last"}}));
  ACC_TRY(check_apart(who, {last, 4, "last"}, {{gates, bytes, "gates"}, {values, bytes, "values"}, {index, 4, "index"}}));
  if (is_empty(*out)) return ACC_OK;
  RecurVariant v;
  v.step = true;
  v.thin = op->spec.type != 0 && width == 1;
  const OpVariant *var = nullptr;
  ACC_TRY(op->variant(v.key(), kRecurStepNames, 1, recur_source_of, &var));
  a.gates_stride = gates->stride[0];
  a.values_stride = values->stride[0];
  a.out_stride = out->stride[0];
  a.enter_stride = state->stride[0];
  a.leave_stride = last->stride[0];
  a.width = (int32_t)width;
  a.strips = (int32_t)ceil_div(width, 4 * v.channels(op->spec.type));
  const int64_t most = kThreads / 256 / a.strips;
  for (int64_t first = 0; first < rows; first += most) {
    // (without index the states' rows go along)
    const int64_t at = index ? 0 : first;
    a.gates = device<const char>(gates) + first * gates->stride[0] * bytes;
    a.values = device<const char>(values) + first * values->stride[0] * bytes;
    a.out = device<char>(out) + first * out->stride[0] * bytes;
    a.index = index ? device<const int32_t>(index) + first : nullptr;
    a.enter = device<const float>(state) + at * state->stride[0];
    a.leave = device<float>(last) + at * last->stride[0];
    a.states = (int32_t)std::max<int64_t>(0, state->shape[0] - at);
    a.rows = std::min(most, rows - first);
    ACC_TRY(launch(op, who, var->fn, a.rows * a.strips, 256, 0, stream, a));
  }
  return ACC_OK;
} ACC_OP_CATCH("acc_exec_recur_step")

}  // extern "C"
