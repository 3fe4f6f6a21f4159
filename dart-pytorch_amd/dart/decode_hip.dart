/// Decoding on the GPU that holds the index: a paged key-value cache with the
/// attention of one new token, and beam search, over libvs_hip.so (C ABI:
/// include/vs_hip.h, `vs_kv_*` and `vs_beam_*`) through `dart:ffi`.
///
/// The calls work on device memory: `GpuArray` here, or addresses that another
/// library on the same GPU hands over.  They run on `stream` (a hipStream_t's
/// address, 0 the default stream) and return without waiting; `GpuArray.read`
/// and `PagedKvCache.check` wait.
///
/// This file needs the Dart SDK (absent from the build container); the same
/// call sequence is exercised by the repository's Python tests through the
/// identical C ABI.
library;

import 'dart:ffi' as ffi;
import 'dart:math' as math;
import 'dart:typed_data';

import 'package:ffi/ffi.dart';

import 'gpu_index_flat_hip.dart' show vsLibraryPath;

typedef _P = ffi.Pointer<ffi.Void>;

/// Element types of device buffers (VS_DTYPE_*; the cache takes the first two).
enum GpuType {
  f32(0, 4),
  bf16(1, 2),
  i32(-1, 4),
  u8(-1, 1);

  const GpuType(this.code, this.size);
  final int code;
  final int size;
}

final class _SeqsC extends ffi.Struct {
  external _P table;
  external _P lens;
  external _P refs;
  @ffi.Int64()
  external int nseq;
  @ffi.Int64()
  external int width;
}

typedef _S = ffi.Pointer<_SeqsC>;

class _Lib {
  _Lib() : lib = ffi.DynamicLibrary.open(vsLibraryPath());
  final ffi.DynamicLibrary lib;

  late final alloc = lib.lookupFunction<ffi.Int32 Function(ffi.Int32, ffi.Int64, ffi.Pointer<_P>),
      int Function(int, int, ffi.Pointer<_P>)>('vs_dev_alloc');
  late final free = lib.lookupFunction<ffi.Int32 Function(ffi.Int32, _P), int Function(int, _P)>('vs_dev_free');
  late final upload = lib.lookupFunction<ffi.Int32 Function(ffi.Int32, _P, _P, ffi.Int64),
      int Function(int, _P, _P, int)>('vs_dev_upload');
  late final download = lib.lookupFunction<ffi.Int32 Function(ffi.Int32, _P, _P, ffi.Int64),
      int Function(int, _P, _P, int)>('vs_dev_download');
  late final lastError =
      lib.lookupFunction<ffi.Pointer<Utf8> Function(), ffi.Pointer<Utf8> Function()>('vs_last_error');

  late final kvCreate = lib.lookupFunction<
      ffi.Int32 Function(ffi.Int32, ffi.Int64, ffi.Int64, ffi.Int64, ffi.Int64, ffi.Int64, ffi.Int32, _P,
          ffi.Pointer<_P>),
      int Function(int, int, int, int, int, int, int, _P, ffi.Pointer<_P>)>('vs_kv_create');
  late final kvDestroy = lib.lookupFunction<ffi.Void Function(_P), void Function(_P)>('vs_kv_destroy');
  late final attend = lib.lookupFunction<
      ffi.Int32 Function(_P, _S, ffi.Int64, ffi.Int64, _P, ffi.Int64, ffi.Int64, _P, ffi.Int64, ffi.Int64, _P,
          ffi.Int64, ffi.Int64, _P, ffi.Int64, ffi.Int64, _P, ffi.Float, ffi.Int64, ffi.Int64, _P),
      int Function(_P, _S, int, int, _P, int, int, _P, int, int, _P, int, int, _P, int, int, _P, double, int, int,
          _P)>('vs_kv_attend');
  late final append = lib.lookupFunction<
      ffi.Int32 Function(_P, _S, ffi.Int64, _P, ffi.Int64, ffi.Int64, _P, ffi.Int64, ffi.Int64, _P, ffi.Int64, _P),
      int Function(_P, _S, int, _P, int, int, _P, int, int, _P, int, _P)>('vs_kv_append');
  late final extend = lib.lookupFunction<ffi.Int32 Function(_P, _S, ffi.Int64, _P, _P),
      int Function(_P, _S, int, _P, _P)>('vs_kv_extend');
  late final fork = lib.lookupFunction<ffi.Int32 Function(_P, _S, _P, _S, _P),
      int Function(_P, _S, _P, _S, _P)>('vs_kv_fork');
  late final freeSeqs = lib.lookupFunction<ffi.Int32 Function(_P, _S, _P, ffi.Int64, _P),
      int Function(_P, _S, _P, int, _P)>('vs_kv_free');
  late final evict = lib.lookupFunction<ffi.Int32 Function(_P, _S, ffi.Int64, ffi.Int64, _P),
      int Function(_P, _S, int, int, _P)>('vs_kv_evict');
  late final compactWith = lib.lookupFunction<
      ffi.Int32 Function(_P, _S, _S, ffi.Pointer<_S>, ffi.Int64, _P, _P),
      int Function(_P, _S, _S, ffi.Pointer<_S>, int, _P, _P)>('vs_kv_compact_with');
  late final check = lib.lookupFunction<ffi.Int32 Function(_P, _P), int Function(_P, _P)>('vs_kv_check');

  late final beamCreate = lib.lookupFunction<ffi.Int32 Function(ffi.Int32, ffi.Pointer<_P>),
      int Function(int, ffi.Pointer<_P>)>('vs_beam_create');
  late final beamDestroy = lib.lookupFunction<ffi.Void Function(_P), void Function(_P)>('vs_beam_destroy');
  late final beamSelect = lib.lookupFunction<
      ffi.Int32 Function(_P, _P, ffi.Int32, ffi.Int64, ffi.Int64, ffi.Int64, ffi.Int64, _P, _P, ffi.Int64, ffi.Int64,
          _P, _P, _P, _P, _P),
      int Function(_P, _P, int, int, int, int, int, _P, _P, int, int, _P, _P, _P, _P, _P)>('vs_beam_select');
  late final beamReorder = lib.lookupFunction<
      ffi.Int32 Function(_P, _P, ffi.Int64, _P, ffi.Int64, ffi.Int64, _P, ffi.Int64, ffi.Int64, _P, _P),
      int Function(_P, _P, int, _P, int, int, _P, int, int, _P, _P)>('vs_beam_reorder');

  void ok(int rc) {
    if (rc == 0) return;
    final msg = lastError().toDartString();
    if (rc == 1) throw ArgumentError(msg);
    if (rc == 4) throw UnsupportedError(msg);
    throw StateError('libvs_hip: $msg (status $rc)');
  }
}

final _Lib _vs = _Lib();

_P _at(int address) => _P.fromAddress(address);

/// A contiguous array in device memory.
class GpuArray {
  GpuArray(this.shape, this.type, {this.device = 0}) {
    final out = calloc<_P>();
    try {
      _vs.ok(_vs.alloc(device, math.max(1, length * type.size), out));
      _ptr = out.value;
    } finally {
      calloc.free(out);
    }
  }

  final List<int> shape;
  final GpuType type;
  final int device;
  late _P _ptr;

  int get length => shape.fold(1, (a, b) => a * b);
  _P get pointer => _ptr.address == 0 ? throw StateError('GpuArray used after dispose()') : _ptr;

  /// Host bytes of the array's own type and length.
  void write(TypedData data) {
    final bytes = data.buffer.asUint8List(data.offsetInBytes, data.lengthInBytes);
    if (bytes.length != length * type.size) throw ArgumentError('${bytes.length} bytes for $shape');
    if (bytes.isEmpty) return;
    final host = calloc<ffi.Uint8>(bytes.length);
    try {
      host.asTypedList(bytes.length).setAll(0, bytes);
      _vs.ok(_vs.upload(device, pointer, host.cast(), bytes.length));
    } finally {
      calloc.free(host);
    }
  }

  /// A host copy of the bytes (waits for the default stream).
  Uint8List read() {
    final n = length * type.size;
    if (n == 0) return Uint8List(0);
    final host = calloc<ffi.Uint8>(n);
    try {
      _vs.ok(_vs.download(device, host.cast(), pointer, n));
      return Uint8List.fromList(host.asTypedList(n));
    } finally {
      calloc.free(host);
    }
  }

  void dispose() {
    if (_ptr.address != 0) _vs.free(device, _ptr);
    _ptr = ffi.nullptr;
  }
}

void _expect(GpuArray a, String what, List<int> shape, GpuType type) {
  final same = a.shape.length == shape.length &&
      Iterable<int>.generate(shape.length).every((i) => a.shape[i] == shape[i]);
  if (!same || a.type != type) throw ArgumentError('$what: ${a.type} ${a.shape}, expected $type $shape');
}

/// Sequences on a [PagedKvCache]: table `[n, width]`, lens `[n]`, refs `[pages]`, all i32.
class KvSequences {
  KvSequences(this.table, this.lens, this.refs)
      : n = table.shape[0],
        width = table.shape[1] {
    _expect(table, 'table', [n, width], GpuType.i32);
    _expect(lens, 'lens', [n], GpuType.i32);
    _expect(refs, 'refs', [refs.shape[0]], GpuType.i32);
    _c.ref
      ..table = table.pointer
      ..lens = lens.pointer
      ..refs = refs.pointer
      ..nseq = n
      ..width = width;
  }

  final GpuArray table, lens, refs;
  final int n, width;
  final _S _c = calloc<_SeqsC>();

  /// Frees the descriptor, not the arrays.
  void dispose() => calloc.free(_c);
}

/// Keys and values of every layer, in pages that stay in HBM.
class PagedKvCache {
  PagedKvCache(this.pages, this.pageSize, this.kvHeads, this.headDim,
      {this.layers = 1, this.type = GpuType.bf16, this.device = 0}) {
    if (type.code < 0) throw ArgumentError('a cache is f32 or bf16');
    final out = calloc<_P>();
    try {
      _vs.ok(_vs.kvCreate(device, pages, pageSize, layers, kvHeads, headDim, type.code, ffi.nullptr, out));
      _h = out.value;
    } finally {
      calloc.free(out);
    }
  }

  final int pages, pageSize, kvHeads, headDim, layers, device;
  final GpuType type;
  late _P _h;

  _P get _handle => _h.address == 0 ? throw StateError('PagedKvCache used after dispose()') : _h;

  _S _seqs(KvSequences s) =>
      s.refs.shape[0] == pages ? s._c : throw ArgumentError('refs of ${s.refs.shape[0]} pages on a cache of $pages');

  KvSequences newSequences(int n, int width, {GpuArray? refs}) {
    final table = GpuArray([n, width], GpuType.i32, device: device)
      ..write(Int32List(n * width)..fillRange(0, n * width, -1));
    final lens = GpuArray([n], GpuType.i32, device: device)..write(Int32List(n));
    final counts = refs ?? (GpuArray([pages], GpuType.i32, device: device)..write(Int32List(pages)));
    return KvSequences(table, lens, counts);
  }

  /// Attention of each sequence's last position: q, out `[n, heads, headDim]`;
  /// k, v `[n, kvHeads, headDim]`, the new token's, stored in the same pass.
  void attend(KvSequences s, GpuArray q, GpuArray out,
      {GpuArray? k,
      GpuArray? v,
      GpuArray? lse,
      int layer = 0,
      double? scale,
      int window = 0,
      int sinks = 0,
      int stream = 0}) {
    final heads = q.shape[1];
    _expect(q, 'q', [s.n, heads, headDim], type);
    _expect(out, 'out', [s.n, heads, headDim], type);
    for (final a in [k, v]) {
      if (a != null) _expect(a, 'k and v', [s.n, kvHeads, headDim], type);
    }
    if (lse != null) _expect(lse, 'lse', [s.n, heads], GpuType.f32);
    final row = heads * headDim, kvRow = kvHeads * headDim;
    _vs.ok(_vs.attend(
        _handle, _seqs(s), layer, heads, q.pointer, row, headDim, k?.pointer ?? ffi.nullptr, kvRow, headDim,
        v?.pointer ?? ffi.nullptr, kvRow, headDim, out.pointer, row, headDim, lse?.pointer ?? ffi.nullptr,
        scale ?? 1 / math.sqrt(headDim), window, sinks, _at(stream)));
  }

  /// Rows `[rows, kvHeads, headDim]` to the sequences' last positions; starts `[n + 1]`: whose rows they are.
  void append(KvSequences s, GpuArray k, GpuArray v, {GpuArray? starts, int layer = 0, int stream = 0}) {
    final rows = k.shape[0], row = kvHeads * headDim;
    _expect(k, 'k', [rows, kvHeads, headDim], type);
    _expect(v, 'v', [rows, kvHeads, headDim], type);
    if (starts != null) _expect(starts, 'starts', [s.n + 1], GpuType.i32);
    _vs.ok(_vs.append(_handle, _seqs(s), layer, k.pointer, row, headDim, v.pointer, row, headDim,
        starts?.pointer ?? ffi.nullptr, rows, _at(stream)));
  }

  /// [count] more positions for every sequence, with copies of shared last pages.
  void extend(KvSequences s, int count, {int stream = 0}) =>
      _vs.ok(_vs.extend(_handle, _seqs(s), count, ffi.nullptr, _at(stream)));

  /// out's sequence i = a copy of s's parents[i] that shares its pages.
  void fork(KvSequences s, GpuArray parents, KvSequences out, {int stream = 0}) {
    if (parents.length != out.n || parents.type != GpuType.i32) throw ArgumentError('parents: ${parents.shape}');
    _vs.ok(_vs.fork(_handle, _seqs(s), parents.pointer, _seqs(out), _at(stream)));
  }

  /// Drops the listed sequences (all where [ids] is null).
  void free(KvSequences s, {GpuArray? ids, int stream = 0}) {
    if (ids != null && ids.type != GpuType.i32) throw ArgumentError('ids: ${ids.type}');
    _vs.ok(_vs.freeSeqs(_handle, _seqs(s), ids?.pointer ?? ffi.nullptr, ids?.length ?? 0, _at(stream)));
  }

  /// Gives back whole pages behind the window.
  void evict(KvSequences s, int window, {int sinks = 0, int stream = 0}) =>
      _vs.ok(_vs.evict(_handle, _seqs(s), window, sinks, _at(stream)));

  /// Moves the pages in use to the cache's front, whoever holds them: every
  /// other set of sequences on the same counts has to be in [others], whose
  /// tables follow in place; [moved] (i32 `[pages]`) receives where each page's
  /// contents are now, for holds that are in no table.
  void compact(KvSequences s,
      {KvSequences? out, List<KvSequences> others = const [], GpuArray? moved, int stream = 0}) {
    if (moved != null) _expect(moved, 'moved', [pages], GpuType.i32);
    final more = calloc<_S>(math.max(1, others.length));
    try {
      for (var i = 0; i < others.length; i++) {
        more[i] = _seqs(others[i]);
      }
      _vs.ok(_vs.compactWith(_handle, _seqs(s), _seqs(out ?? s), more, others.length,
          moved?.pointer ?? ffi.nullptr, _at(stream)));
    } finally {
      calloc.free(more);
    }
  }

  /// Waits; throws what earlier calls met on the device (too few pages, ...).
  void check({int stream = 0}) => _vs.ok(_vs.check(_handle, _at(stream)));

  void dispose() {
    if (_h.address != 0) _vs.kvDestroy(_h);
    _h = ffi.nullptr;
  }
}

/// The choice of the next beams and the reordering of their states.
class BeamSearch {
  BeamSearch({this.device = 0}) {
    final out = calloc<_P>();
    try {
      _vs.ok(_vs.beamCreate(device, out));
      _h = out.value;
    } finally {
      calloc.free(out);
    }
  }

  final int device;
  late _P _h;

  _P get _handle => _h.address == 0 ? throw StateError('BeamSearch used after dispose()') : _h;

  /// logits `[requests * beams, vocab]`, scores `[requests, beams]`; outputs `[requests, k]`.
  void select(GpuArray logits, GpuArray scores, GpuArray scoresOut, GpuArray tokensOut, GpuArray parentsOut,
      {GpuArray? finished, GpuArray? finishedOut, int eos = -1, int stream = 0}) {
    final requests = scores.shape[0], beams = scores.shape[1], vocab = logits.shape[1], k = scoresOut.shape[1];
    if (logits.type.code < 0) throw ArgumentError('logits are f32 or bf16');
    _expect(logits, 'logits', [requests * beams, vocab], logits.type);
    _expect(scores, 'scores', [requests, beams], GpuType.f32);
    _expect(scoresOut, 'scoresOut', [requests, k], GpuType.f32);
    _expect(tokensOut, 'tokensOut', [requests, k], GpuType.i32);
    _expect(parentsOut, 'parentsOut', [requests, k], GpuType.i32);
    if (finished != null) _expect(finished, 'finished', [requests, beams], GpuType.u8);
    if (finishedOut != null) _expect(finishedOut, 'finishedOut', [requests, k], GpuType.u8);
    _vs.ok(_vs.beamSelect(
        _handle, logits.pointer, logits.type.code, vocab, requests, beams, vocab, scores.pointer,
        finished?.pointer ?? ffi.nullptr, eos, k, scoresOut.pointer, tokensOut.pointer, parentsOut.pointer,
        finishedOut?.pointer ?? ffi.nullptr, _at(stream)));
  }

  /// Row i of [out] = row parents[i] of [state]; with [tail], an i32 state's last column is tail's.
  void reorder(GpuArray parents, GpuArray state, GpuArray out, {GpuArray? tail, int stream = 0}) {
    final rows = out.shape[0], wide = out.shape[1] * out.type.size;
    _expect(state, 'state', [state.shape[0], out.shape[1]], out.type);
    if (parents.length != rows || parents.type != GpuType.i32) throw ArgumentError('parents: ${parents.shape}');
    if (tail != null && (tail.length != rows || tail.type != GpuType.i32 || out.type != GpuType.i32 || wide == 0)) {
      throw ArgumentError('tail needs an i32 state of at least one column, and one value per row');
    }
    _vs.ok(_vs.beamReorder(_handle, parents.pointer, rows, state.pointer, state.shape[0], wide, out.pointer, wide,
        tail == null ? wide : wide - 4, tail?.pointer ?? ffi.nullptr, _at(stream)));
  }

  void dispose() {
    if (_h.address != 0) _vs.beamDestroy(_h);
    _h = ffi.nullptr;
  }
}
