using System.Runtime.InteropServices;

namespace Llmdot.Hip.Native;

/// <summary>
/// P/Invoke declarations of include/llmdot_hip_cache.h: the quantised KV cache,
/// attention over it and the verification of drafted tokens, over device memory
/// (same names, argument order and meaning).
/// </summary>
internal static unsafe class HipCacheNative
{
    private const string Lib = "llmdot_hip";

    /// <summary>llmdot_hip_kv_cache_desc; types are GgmlType values (Q8_0 or Q4_0).</summary>
    [StructLayout(LayoutKind.Sequential)]
    public struct KvCacheDesc
    {
        public int Slots;
        public int KvHeads;
        public int HeadDim;
        public int Capacity;
        public uint KType;
        public uint VType;
    }

    /// <summary>llmdot_hip_token_batch: device arrays of slots, first positions and counts.</summary>
    [StructLayout(LayoutKind.Sequential)]
    public struct TokenBatch
    {
        public int Batch;
        public int Tokens;
        public int* Slots;
        public int* Starts;
        public int* Counts;
    }

    /// <summary>llmdot_hip_attention.</summary>
    [StructLayout(LayoutKind.Sequential)]
    public struct Attention
    {
        public int Heads;
        public int Window;
        public float Scale;
        public nint Prefix;
        public int PrefixSlot;
        public int PrefixLen;
        public long QStride;
        public long OutStride;
    }

    [DllImport(Lib)] public static extern int llmdot_hip_stream(nint ctx, nint* stream);

    [DllImport(Lib)] public static extern int llmdot_hip_kv_cache_create(nint ctx, KvCacheDesc* desc, nint* cache);

    [DllImport(Lib)] public static extern int llmdot_hip_kv_cache_destroy(nint cache);

    [DllImport(Lib)] public static extern int llmdot_hip_kv_cache_write(nint cache, float* k, long kStride, float* v,
        long vStride, TokenBatch* rows);

    [DllImport(Lib)] public static extern int llmdot_hip_kv_cache_read(nint cache, float* k, long kStride, float* v,
        long vStride, TokenBatch* rows);

    [DllImport(Lib)] public static extern int llmdot_hip_kv_cache_attention(nint cache, float* q, float* output,
        TokenBatch* rows, Attention* options, void* workspace, nuint workspaceBytes);

    [DllImport(Lib)] public static extern int llmdot_hip_kv_cache_attention_workspace(nint cache, int heads, int batch,
        int tokens, int hasPrefix, nuint* bytes);

    [DllImport(Lib)] public static extern int llmdot_hip_verify_drafts(nint ctx, float* target, float* draft, int* drafts,
        int* counts, float* uniforms, int batch, int draftCount, int vocab, float temperature, int* tokens, int* accepted,
        void* workspace, nuint workspaceBytes);

    [DllImport(Lib)] public static extern int llmdot_hip_verify_drafts_workspace(nint ctx, int batch, int drafts, int vocab,
        nuint* bytes);
}
